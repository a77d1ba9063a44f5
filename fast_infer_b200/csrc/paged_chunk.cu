// Attention of a chunk of new tokens over the paged KV cache (chunked prefill, verification
// of drafted tokens, single tokens, and batches that mix them), on sm_100a tensor cores.
//
//   o_i = sum_j exp(s_ij - lse_i) v_j,  lse_i = log sum_j exp(s_ij)   (j over visible keys;
//   the batch, visibility and score are described in chunk_common.cuh; a token that sees
//   nothing gives o = 0, lse = -inf).
//
// Design:
// * A unit is 2 x (128 / group) consecutive tokens of one sequence for one KV head: two
//   128-row tiles (rows = token x head of the group) that share every K/V tile.
// * The work of a launch is one line of (KV head, unit, key tile) steps, cut into equal
//   contiguous parts, one per CTA. A long prefill, many single tokens over long contexts and
//   any mixture balance alike, without knowing the lengths on the host: every CTA derives
//   the line from cu / ctx in shared memory first. A unit cut between CTAs leaves fp32
//   partial rows in the workspace, joined by chunk_combine_kernel in CTA order (the same bits
//   on every run).
// * Roles (384 threads), tensor memory (S0 | S1 | O0 | O1), the lazily rescaled online
//   softmax and the MMA order are those of the causal prefill kernel (prefill_sm100.cu). K
//   and V tiles are two pages each, gathered by TMA through the block table.
// * Sequences of at most 32 rows (single tokens, drafted tokens) have a kernel of their own, of
//   the same roles, in which a unit runs transposed: S^T = K Q^T with the 128 keys of a tile as
//   tensor-memory lanes and N = its rows, then O^T += V^T P^T with P through shared memory, so
//   no lane idles and a tile costs a softmax thread its rows, not 128 columns. The warpgroups
//   take alternate key tiles as two running softmaxes and merge them at the end. A row's max
//   moves only when some score passes it by 2^8, found by one vote per tile. (One kernel for
//   both forms was tried: its registers spilled and its code, 150 KB, missed the instruction
//   caches; long prefills lost 10 %, single tokens 40 %.) A batch that may hold both kinds
//   launches both kernels, the second beginning on each SM as the first leaves it. (Sharing the
//   SMs out between them by cost was no faster: a step of 24 rows costs as much as a wide one.)
// * What bounds it: a wide step of 256 rows x 128 keys takes 3850 cycles, of which (by count, not by
//   counters) its products need 2040 of the tensor core and its exponentials 1800 of the special
//   function units; issue slots and the chain through tensor memory are the rest. 4096 tokens over
//   61003: 3.18 ms, 999 TFLOP/s, in a burst of 15 ms; repeated for seconds 3.71 ms, 856 TFLOP/s, at
//   the 1.39 GHz that the power cap leaves. 4225 over 2000: 215 us, 992 TFLOP/s (for seconds 250, at
//   1.69 GHz). Single tokens are bound by HBM: 64 over 4000 each, 178 us, 5.9 TB/s; one over 512 by
//   its two launches, 12.3 us.
// * Slots behind a sequence's last token may hold anything: their scores are replaced by
//   -inf, and their V rows are zeroed in shared memory before the product (0 * NaN is NaN).
#include <float.h>

#include "chunk_common.cuh"

namespace fi {

constexpr int kCkThreads = 384;
constexpr int kCkRegsSoftmax = 184;  // 2 x 128 x 184 + 128 x 136 = 384 x 168
constexpr int kCkRegsOther = 136;
constexpr int kCkStages = 2;
constexpr int kCkTeardownBar = 15;
constexpr int kCkMaxBatch = 2048;    // sequences per launch
constexpr int kCkMaxUnits = 4608;    // token units per launch (per KV head)
constexpr int kCkNarrow = 32;        // rows up to which a unit runs transposed
constexpr float kCkRescale = 8.0f;   // log2 units of growth of the max before O is rescaled
constexpr int kCkEmuPairs = 1;       // of 8 column pairs, exp2 on the FMA pipe
// Steps that a unit's start and end are worth: with 0 and 0 / 1 and 2 / 3 and 2 / 4 and 3, 64 single
// tokens over 1000 beside 2048 new over 2000 take 177 / 170 / 168 / 171 us, and 64 over 4000 beside
// 512 new (units of the narrow kernel, all in a few CTAs' parts) 294 / 252 / 200 / 201.
constexpr int kCkPadNarrow = 3, kCkPadWide = 2;
constexpr int kCkManyNew = 500;      // new tokens past one each for which both kernels run
constexpr int kCkSlots = 4;          // units that the scheduler is ahead

// A CTA's part of a unit: key steps [j0, j1) of its n.
struct alignas(16) CkUnit {
  int b, hk;
  int token, pos;      // first packed row, its position
  int rows[2];         // live rows of the two tiles
  int keys, prefix;
  int np, lo;          // step j is key tile j < np ? j : lo + j - np
  int j0, j1, n;
  int pages_ok;        // no block-table entry of its keys is invalid
  int last_cta;        // the CTA with the unit's last step
  int valid;           // 0: no unit is left
};
static_assert(sizeof(CkUnit) == 64, "read as four 16-byte words");

// The unit whose first part a CTA holds when the rest lies in the next CTAs.
struct CkJoin {
  int valid, last_cta, token, hk, rows[2], pad[2];
};

struct CkBarriers {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kCkStages], k_empty[kCkStages];
  uint64_t v_full[kCkStages], v_empty[kCkStages];
  uint64_t s_full[2], p_full[2], o_full[2], o_empty[2];
  uint64_t mma_done;
  uint64_t unit_full[kCkSlots], unit_empty[kCkSlots];
  uint64_t merge;  // both softmax warpgroups, in a transposed unit
  uint32_t tmem_base;
  // transposed units, per warpgroup: rows' max, partial maxima / sums, scale, slope, token
  float n_max[2][kCkNarrow], n_red[2][4][kCkNarrow], n_alpha[2][kCkNarrow];
  alignas(16) float n_neg[2][kCkNarrow];  // -max; FLT_MAX: no score yet, -inf: no such row
  float n_slope[2][kCkNarrow], n_pos[2][kCkNarrow];
  int64_t n_off[kCkNarrow];  // where a row's output goes
  CkUnit units[kCkSlots];
  uint8_t row_token[kChunkTile], row_head[kChunkTile];  // of a tile's rows
  uint32_t warp_sums[kCkThreads / 32];
  uint32_t unit_off[kCkMaxBatch + 1];  // first unit of each sequence
  uint32_t work[kCkMaxUnits + 1];      // steps before each unit
};
constexpr int kCkSmemBytes = 1024 + (2 + 2 * kCkStages) * kChunkTileBytes + (int)sizeof(CkBarriers);
static_assert(kCkSmemBytes <= 227 * 1024, "shared memory");

constexpr int kCkPBytes = kCkNarrow * 256;  // P^T of a transposed unit: 32 rows x 128 keys
static_assert(kCkNarrow == 32, "a column per lane where rows are summed");
static_assert(2 * kCkPBytes <= kChunkTileBytes, "P of both warpgroups in one query tile");

struct ChunkParams {
  ChunkBatch b;
  ScoreForm f;
  void* o;
  int64_t os[2];
  float* lse;  // [total, hq] or null
  // [cta][first, last unit], then rows_cap rows of 128: as they are (narrow), or 32 rows' 4 values
  // side by side (wide, whose threads have a row each)
  float* ws_o;
  float* ws_lse;  // [cta][first, last unit][rows_cap], log2 domain
  CkJoin* join;   // [cta]
  int rows_cap;
  int unit_tokens;  // tokens of a unit: two tiles, or those of kCkNarrow rows
  int split_rows;   // sequences of at most so many rows are the narrow kernel's, others the wide's
  int o_wide;       // rows of o are 32-byte aligned
  int late_wait;    // the kernel before on the stream is the other one of this call
  int* err;
};

__device__ __forceinline__ int ck_tile(const CkUnit& u, int j) {
  return j < u.np ? j : u.lo + (j - u.np);
}

// Key tiles that the unit of tokens [t0, t1) of a sequence visits: [0, np) for the prefix and
// [lo, lo + n - np). A unit that sees nothing visits one (all of it masked).
__device__ __forceinline__ void ck_tiles(const ChunkBatch& p, const ChunkSeq& s, int t0, int t1,
                                         int& np, int& lo, int& n) {
  const int p0 = s.pos0 + t0, p1 = s.pos0 + t1 - 1;
  const int end = min(s.keys, max(p1 + 1, s.prefix));
  const int hi = end > 0 ? (end - 1) / kChunkTile : 0;
  lo = p.window ? min(max(p0 - p.window + 1, 0) / kChunkTile, hi) : 0;
  np = min((s.prefix + kChunkTile - 1) / kChunkTile, lo);
  n = np + hi - lo + 1;
}

// The scheduler (one warp): walks the CTA's part of the line and hands its units to the other
// roles through a ring in shared memory. Its lanes look the units' pages over, so that no one
// else has to unless an entry is invalid. On the line a unit is `pad` steps longer than its key
// tiles, which stand for what it costs to begin and end one; its step j is at pad + j.
__device__ __forceinline__ void ck_schedule(const ChunkBatch& p, int unit_tokens, int pad,
                                            CkBarriers* s, uint32_t units, CkJoin* join_out,
                                            int* err) {
  const int G = gridDim.x, cta = blockIdx.x, lane = threadIdx.x & 31;
  const uint32_t per_head = s->work[units];
  const int64_t total = (int64_t)per_head * p.hk;
  const int active = (int)(total < G ? total : G);  // CTAs with work
  int64_t w = cta < active ? total * cta / active : 0;
  const int64_t end = cta < active ? total * (cta + 1) / active : 0;
  int hk = 0, e = 0, b = 0, at = 0;  // `at`: where in the unit this CTA begins
  if (w < end) {
    hk = (int)(w / per_head);
    const uint32_t r = (uint32_t)(w - (int64_t)hk * per_head);
    e = last_le(s->work, (int)units, r);
    b = last_le(s->unit_off, p.batch, (uint32_t)e);
    at = (int)(r - s->work[e]);
  }
  ChunkSeq q = chunk_seq(p, b);
  const int tt = p.tile_tokens;
  CkJoin join = {};
#pragma unroll 1
  for (int i = 0;; ++i) {
    const int slot = i % kCkSlots;
    if (i >= kCkSlots &&
        !__all_sync(0xffffffffu, mbar_wait(&s->unit_empty[slot], ((i / kCkSlots) - 1) & 1, err)))
      break;
    CkUnit u;
    const int len = w < end ? (int)(s->work[e + 1] - s->work[e]) : 0;
    const int stop = len - at <= end - w ? len : at + (int)(end - w);
    u.valid = stop > pad;  // (not so: no unit, or one whose steps are all in the next CTA)
    bool pages_ok = true;
    if (u.valid) {
      const int t0 = (e - (int)s->unit_off[b]) * unit_tokens, t1 = min(t0 + unit_tokens, q.n);
      int tiles;
      ck_tiles(p, q, t0, t1, u.np, u.lo, tiles);
      u.n = len - pad;  // the line's own count: the walk always ends
      u.b = b;
      u.hk = hk;
      u.token = q.start + t0;
      u.pos = q.pos0 + t0;
      u.keys = q.keys;
      u.prefix = q.prefix;
      u.rows[0] = min(t1 - t0, tt) * p.group;
      u.rows[1] = max(t1 - t0 - tt, 0) * p.group;
      u.j0 = max(at - pad, 0);
      u.j1 = stop - pad;
      // the unit's last step, w - at + len - 1, is the last CTA's that starts at or before it
      u.last_cta = stop == len ? cta : (int)(((w - at + len) * active - 1) / total);
      for (int j = u.j0 + (lane >> 1); j < u.j1; j += 16) {
        const int tile = ck_tile(u, j), half = lane & 1;
        if ((tile * 2 + half) * kChunkPage < u.keys &&
            chunk_page(p, b, u.keys, tile, half) == p.num_blocks)
          pages_ok = false;
      }
      w += stop - at;
      at = 0;
      if (++e == (int)units) {
        e = 0;
        ++hk;
      }
      if (w < end && (e < (int)s->unit_off[b] || e >= (int)s->unit_off[b + 1])) {
        if (e == 0) b = -1;
        do ++b; while ((int)s->unit_off[b + 1] <= e);
        q = chunk_seq(p, b);
      }
    }
    u.pages_ok = __all_sync(0xffffffffu, pages_ok);
    if (lane == 0) {
      s->units[slot] = u;
      mbar_arrive(&s->unit_full[slot]);  // released to the waits that read it
    }
    if (u.valid && u.j0 == 0 && u.j1 < u.n) {  // begins here and goes on: it is the last one
      join.valid = 1;
      join.last_cta = u.last_cta;
      join.token = u.token;
      join.hk = u.hk;
      join.rows[0] = u.rows[0];
      join.rows[1] = u.rows[1];
    }
    if (!u.valid) break;
  }
  if (lane == 0) *join_out = join;
}

// The next unit of the ring, null when none is left; it stays in shared memory, read there by
// whole warps (or one thread, kWarp = false), until ck_done gives the slot back.
template <bool kWarp>
__device__ __forceinline__ const CkUnit* ck_next(CkBarriers* s, int i, int* err) {
  const int slot = i % kCkSlots;
  bool ok = mbar_wait(&s->unit_full[slot], (i / kCkSlots) & 1, err);
  if (kWarp) ok = __all_sync(0xffffffffu, ok);
  return ok && s->units[slot].valid ? &s->units[slot] : nullptr;
}
template <bool kWarp>
__device__ __forceinline__ void ck_done(CkBarriers* s, int& i) {
  if (kWarp) __syncwarp();
  if (!kWarp || (threadIdx.x & 31) == 0) mbar_arrive(&s->unit_empty[i % kCkSlots]);
  ++i;
}

// 32 scores of one row in log2 units, in place: the cap and the distance bias (without either,
// they stay unscaled). `off` = position of the first column's key minus the row's position; a row
// that is not `live` has no say in which form of tanh runs. The short form for small scores: 374 us
// for 4225 tokens of 24 sequences and a cap of 50, 532 without it (scores past it pay 5 % for the
// test). Where a thread has one key (score_form8) its code costs more than it saves: 48 against 45 us.
template <bool kCap, bool kAlibi>
__device__ __forceinline__ void score_form(uint32_t* sr, const ScoreForm& f, float slope2,
                                           float off, bool live) {
  if constexpr (kCap) {
    const uint64_t cin = f32x2(f.cap_in, f.cap_in), cout = f32x2(f.cap_log2, f.cap_log2);
    float big = 0.f;
#pragma unroll
    for (int c = 0; c < 32; c += 2)
      big = fmax3f(big, fabsf(__uint_as_float(sr[c])), fabsf(__uint_as_float(sr[c + 1])));
    const bool small = __all_sync(0xffffffffu, !live || big * f.cap_in <= 1.f);
    const bool tiny = __all_sync(0xffffffffu, !live || big <= f.tiny_max);
    if (tiny) {
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const uint64_t x = f32x2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
        float a, b;
        f32x2_split(mul_f32x2(cap_tiny_x2(f, x), x), a, b);
        sr[c] = __float_as_uint(a);
        sr[c + 1] = __float_as_uint(b);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const uint64_t u =
            mul_f32x2(f32x2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), cin);
        uint64_t y = tanh_poly_x2(u);
        if (!small) {
          float u0, u1, y0, y1;
          f32x2_split(u, u0, u1);
          f32x2_split(y, y0, y1);
          y = f32x2(fabsf(u0) <= 1.f ? y0 : tanh_any(u0), fabsf(u1) <= 1.f ? y1 : tanh_any(u1));
        }
        float a, b;
        f32x2_split(mul_f32x2(y, cout), a, b);
        sr[c] = __float_as_uint(a);
        sr[c + 1] = __float_as_uint(b);
      }
    }
  }
  if constexpr (kAlibi) {
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      const float s = __uint_as_float(sr[c]);
      const float d = fabsf(off + (float)c) * slope2;
      sr[c] = __float_as_uint(kCap ? s - d : fmaf(s, f.scale_log2, -d));
    }
  }
}

// 8 scores of one key in log2 units, one per row of a transposed unit. `pos` and `key` count from
// the unit's first token, so that distances are exact at any position.
template <bool kCap, bool kAlibi>
__device__ __forceinline__ void score_form8(const uint32_t* raw, float* s, const ScoreForm& f,
                                             const float* slope2, const float* pos, float key) {
  bool small = true;
  if constexpr (kCap) {
    float big = 0.f;
#pragma unroll
    for (int c = 0; c < 8; c += 2)
      big = fmax3f(big, fabsf(__uint_as_float(raw[c])), fabsf(__uint_as_float(raw[c + 1])));
    small = __all_sync(0xffffffffu, big * f.cap_in <= 1.f);
  }
#pragma unroll
  for (int c = 0; c < 8; c += 2) {
    uint64_t x = f32x2(__uint_as_float(raw[c]), __uint_as_float(raw[c + 1]));
    if constexpr (kCap) {
      const uint64_t v = mul_f32x2(x, f32x2(f.cap_in, f.cap_in));
      uint64_t y = tanh_poly_x2(v);
      if (!small) {
        float v0, v1, y0, y1;
        f32x2_split(v, v0, v1);
        f32x2_split(y, y0, y1);
        y = f32x2(fabsf(v0) <= 1.f ? y0 : tanh_any(v0), fabsf(v1) <= 1.f ? y1 : tanh_any(v1));
      }
      x = mul_f32x2(y, f32x2(f.cap_log2, f.cap_log2));
    } else {
      x = mul_f32x2(x, f32x2(f.scale_log2, f.scale_log2));
    }
    f32x2_split(x, s[c], s[c + 1]);
    if constexpr (kAlibi) {
      s[c] -= slope2[c] * fabsf(pos[c] - key);
      s[c + 1] -= slope2[c + 1] * fabsf(pos[c + 1] - key);
    }
  }
}

// p = 2^(s * sl2 - mref) of a row, its sum, and p packed in place. 1 of 8 pairs takes exp2 on the
// FMA pipe (0: 4772 us for a chunk of 4096 tokens over 61003, 1: 3587, 2: 3746, 3: 3802), to 2.2e-7:
// lse is an output, which a rougher polynomial would show in.
// The sum takes p in 32 bits; the product with V takes it in V's type, as kind::f16 asks of both
// operands: half a step (2^-12 .. 2^-11, bf16 2^-9 .. 2^-8) of each p, which adds to the output's own
// rounding: 3.0e-4 in place of 2.1e-4 (root mean square, relative; bf16 2.3e-3 and 1.7e-3). P as the
// sum of two such values would take the product twice.
template <typename T>
__device__ __forceinline__ float ck_exp(uint32_t* sr, float sl2, float mref) {
  const uint64_t sc2 = f32x2(sl2, sl2), nm2 = f32x2(-mref, -mref);
  uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int c = 0; c < kChunkTile; c += 2) {
    const uint64_t xp =
        fma_f32x2(f32x2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), sc2, nm2);
    float p0, p1;
    if (((c >> 1) & 7) < kCkEmuPairs) {
      f32x2_split(exp2_poly5_x2(xp), p0, p1);
    } else {
      float x0, x1;
      f32x2_split(xp, x0, x1);
      p0 = fast_exp2(x0);
      p1 = fast_exp2(x1);
    }
    sum2[(c >> 1) & 3] = add_f32x2(sum2[(c >> 1) & 3], f32x2(p0, p1));
    sr[c >> 1] = Half16<T>::pack(p0, p1);
  }
  float lo, hi;
  f32x2_split(add_f32x2(add_f32x2(sum2[0], sum2[1]), add_f32x2(sum2[2], sum2[3])), lo, hi);
  return lo + hi;
}

// Zero rows [from, 128) of a V tile (both 64-value columns) with one warpgroup.
__device__ __forceinline__ void zero_v_rows(uint8_t* v, int from, int tid) {
  const int chunks = (kChunkTile - from) * 8;
#pragma unroll 1
  for (int i = tid; i < 2 * chunks; i += 128) {
    const int half = i >= chunks, k = half ? i - chunks : i;
    *reinterpret_cast<uint4*>(v + half * kChunkHalf + from * 128 + k * 16) = make_uint4(0, 0, 0, 0);
  }
}

// A transposed unit, softmax side: warpgroup t takes key tiles j0 + t, j0 + t + 2, ... A thread is
// one key of the tile (and, for O^T, one dim). `ok` turns false when a wait runs out; a warp that
// saw it goes on without waiting, so that every barrier here gets all of its threads.
template <typename T, bool kCap, bool kAlibi>
__device__ __forceinline__ void narrow_unit(const ChunkParams& p, CkBarriers* bars, const CkUnit& u,
                                            uint8_t* sP, uint8_t* sV, uint32_t tmem, int t,
                                            int quarter, int lane, int& sc, int& g,
                                            int& uc, int& merges, int cta, bool& ok) {
  const ChunkBatch& pb = p.b;
  const int rows = u.rows[0], n = u.j1 - u.j0, tid = quarter * 32 + lane;
  const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
  const uint32_t tS = tmem + lane_off + t * 128, tO = tmem + lane_off + 256;
  const bool mine = t < n;  // this warpgroup has a key tile
  float l[kCkNarrow];
#pragma unroll
  for (int c = 0; c < kCkNarrow; ++c) l[c] = 0.f;
  float* n_max = bars->n_max[t];
  constexpr float kTop = 256.f;  // 2^kCkRescale
  if (tid < kCkNarrow) {
    n_max[tid] = -INFINITY;
    bars->n_neg[t][tid] = tid < rows ? FLT_MAX : -INFINITY;
    bars->n_alpha[t][tid] = 0.f;
    if (kAlibi) {
      const bool live = tid < rows;
      bars->n_slope[t][tid] = live ? p.f.slopes[u.hk * pb.group + bars->row_head[tid]] * kLog2e : 0.f;
      bars->n_pos[t][tid] = (float)bars->row_token[tid];
    }
  }
  __syncwarp();
  named_bar_sync(1 + t, 128);
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err));
  };
  auto meet = [&]() {  // both warpgroups
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->merge);
    wait(&bars->merge, merges++ & 1);
  };
  // P^T is [rows][128 keys], K-major with the 128-byte swizzle: this thread's column of it
  uint8_t* pcol = sP + t * kCkPBytes + (tid >> 6) * (kCkPBytes / 2);
  const uint32_t kbyte = (uint32_t)(tid & 63) * 2;
#pragma unroll 1
  for (int j = t; j < n; j += 2, ++sc) {
    const int tile = ck_tile(u, u.j0 + j), k0 = tile * kChunkTile, key = k0 + tid;
    const int stage = (g + j) % kCkStages;
    const bool page_ok =
        u.pages_ok || chunk_page(pb, u.b, u.keys, tile, tid >> 6) != pb.num_blocks;
    wait(&bars->s_full[t], sc & 1);
    if (k0 + kChunkTile > u.keys) {
      wait(&bars->v_full[stage], ((g + j) / kCkStages) & 1);
      zero_v_rows(sV + stage * kChunkTileBytes, max(u.keys - k0, 0), tid);
    }
    tc_fence_after();
    // columns [c_lo, c_hi) see this key
    int c_lo = 0, c_hi = rows;
    if (key >= u.prefix) {
      c_lo = min(max(key - u.pos, 0), kCkNarrow) * pb.group;
      if (pb.window) c_hi = min(rows, min(max(key + pb.window - u.pos, 0), kCkNarrow) * pb.group);
    }
    if (!page_ok || key >= u.keys) c_hi = 0;
    const bool mask = !__all_sync(0xffffffffu, c_lo <= 0 && c_hi >= rows);
    const uint32_t vis = low_bits(c_hi, 0) & ~low_bits(c_lo, 0);
    float s[kCkNarrow];  // scores in log2 units, then 2^(score - max)
    // the first tile sets the rows' max; later ones keep it unless some score passes it by 2^8
#pragma unroll 1
    for (bool move = j == t;; move = true) {
      uint32_t raw[kCkNarrow];
#pragma unroll
      for (int cc = 0; cc < kCkNarrow; cc += 8)
        if (cc < rows) tmem_ld8(tS + cc, raw + cc);
      tmem_wait_ld();
      reg_fence<kCkNarrow>(raw);
#pragma unroll
      for (int cc = 0; cc < kCkNarrow; cc += 8)
        if (cc < rows) {
          score_form8<kCap, kAlibi>(raw + cc, s + cc, p.f, bars->n_slope[t] + cc, bars->n_pos[t] + cc,
                                     (float)(key - u.pos));
          if (mask) {
#pragma unroll
            for (int c = cc; c < cc + 8; ++c)
              if (!((vis >> c) & 1u)) s[c] = -INFINITY;
          }
        }
      if (move) {
#pragma unroll
        for (int cc = 0; cc < kCkNarrow; cc += 8)
          if (cc < rows) {
            // over the lanes: columns trade places until four lanes have one
            float mx[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) mx[c] = s[cc + c];
#pragma unroll
            for (int half = 4; half > 0; half >>= 1) {
              const bool up = lane & (half * 4);
#pragma unroll
              for (int c = 0; c < half; ++c) {
                const float give = up ? mx[c] : mx[c + half], keep = up ? mx[c + half] : mx[c];
                mx[c] = fmax_nan(keep, __shfl_xor_sync(0xffffffffu, give, half * 4));
              }
            }
            mx[0] = fmax_nan(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], 2));
            mx[0] = fmax_nan(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], 1));
            if ((lane & 3) == 0) bars->n_red[t][quarter][cc + (lane >> 2)] = mx[0];
          }
        __syncwarp();
        named_bar_sync(1 + t, 128);
        if (tid < rows) {
          const float was = n_max[tid];
          const float now = fmax3_nan(
              was, fmax_nan(bars->n_red[t][0][tid], bars->n_red[t][1][tid]),
              fmax_nan(bars->n_red[t][2][tid], bars->n_red[t][3][tid]));
          bars->n_alpha[t][tid] = was == -INFINITY ? 0.f : fast_exp2(was - now);
          n_max[tid] = now;
          bars->n_neg[t][tid] = now == -INFINITY ? FLT_MAX : -now;
        }
        __syncwarp();
        named_bar_sync(1 + t, 128);
        if (j >= 2) {
          // the product of this warpgroup's last tile is complete: S here was committed after it
#pragma unroll
          for (int cc = 0; cc < kCkNarrow; cc += 8)
            if (cc < rows) {
              uint32_t ov[8];
              tmem_ld8(tO + t * 128 + cc, ov);
              tmem_wait_ld();
              reg_fence<8>(ov);
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const float a = bars->n_alpha[t][cc + c];
                ov[c] = __float_as_uint(__uint_as_float(ov[c]) * a);
                l[cc + c] *= a;
              }
              tmem_st8(tO + t * 128 + cc, ov);
            }
          tmem_wait_st();
        }
      }
      // A row whose max is still -inf (it has seen nothing, or keys that score -inf alone) adds
      // FLT_MAX: a finite score gives 2^FLT_MAX, past any bound, and one of -inf the weight 0. A
      // score that is NaN makes NaN of its weight and, where the max moves, of the max: -inf is left
      // to rows that no score of theirs counts in. A column without a row adds -inf: p = 0.
      float top = 0.f;
#pragma unroll
      for (int cc = 0; cc < kCkNarrow; cc += 8)
        if (cc < rows) {
#pragma unroll
          for (int c = cc; c < cc + 8; c += 4) {
            const float4 nm = *reinterpret_cast<const float4*>(&bars->n_neg[t][c]);
            s[c] = fast_exp2(s[c] + nm.x);
            s[c + 1] = fast_exp2(s[c + 1] + nm.y);
            s[c + 2] = fast_exp2(s[c + 2] + nm.z);
            s[c + 3] = fast_exp2(s[c + 3] + nm.w);
            top = fmax3f(fmax3f(top, s[c], s[c + 1]), s[c + 2], s[c + 3]);
          }
          if (mask) {
#pragma unroll
            for (int c = cc; c < cc + 8; ++c)
              if (!((vis >> c) & 1u)) s[c] = 0.f;
          }
        }
      if (move || wg_bar_and(1 + t, top <= kTop)) break;
    }
#pragma unroll
    for (int cc = 0; cc < kCkNarrow; cc += 8)
      if (cc < rows) {
#pragma unroll
        for (int c = cc; c < cc + 8; c += 2) {
          l[c] += s[c];  // in 32 bits; P is rounded to V's type for the product (see ck_exp)
          l[c + 1] += s[c + 1];
          const uint32_t pk = Half16<T>::pack(s[c], s[c + 1]);
          *reinterpret_cast<uint16_t*>(pcol + c * 128 + (kbyte ^ ((c & 7) << 4))) = (uint16_t)pk;
          *reinterpret_cast<uint16_t*>(pcol + (c + 1) * 128 + (kbyte ^ (((c + 1) & 7) << 4))) =
              (uint16_t)(pk >> 16);
        }
      }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->p_full[t]);
  }
  if (mine) wait(&bars->o_full[t], uc & 1);
  // sums over the lanes: halves of the columns trade places until lane i has column i
#pragma unroll
  for (int half = kCkNarrow / 2; half > 0; half >>= 1) {
#pragma unroll
    for (int c = 0; c < half; ++c) {
      const bool up = lane & half;
      const float give = up ? l[c] : l[c + half], keep = up ? l[c + half] : l[c];
      l[c] = keep + __shfl_xor_sync(0xffffffffu, give, half);
    }
  }
  bars->n_red[t][quarter][lane] = l[0];
  tc_fence_before();
  meet();
  tc_fence_after();
  const bool whole = u.j0 == 0 && u.j1 == u.n;
  if (t == 0 && tid < rows) {
    const float m0 = bars->n_max[0][tid], m1 = bars->n_max[1][tid], mx = fmax_nan(m0, m1);
    float l0 = 0.f, l1 = 0.f;
    for (int i = 0; i < 4; ++i) {
      l0 += bars->n_red[0][i][tid];
      l1 += bars->n_red[1][i][tid];
    }
    const float w0 = m0 == -INFINITY ? 0.f : exp2f(m0 - mx), w1 = m1 == -INFINITY ? 0.f : exp2f(m1 - mx);
    const float sum = w0 * l0 + w1 * l1;
    const bool none = mx == -INFINITY;
    bars->n_alpha[0][tid] = none ? 0.f : w0 / sum;
    bars->n_alpha[1][tid] = none ? 0.f : w1 / sum;
    const float lse2 = none ? -INFINITY : mx + log2f(sum);
    const int64_t token = u.token + bars->row_token[tid];
    const int head = u.hk * pb.group + bars->row_head[tid];
    if (whole) {
      bars->n_off[tid] = token * p.os[0] + head * p.os[1];
      if (p.lse) p.lse[token * pb.hq + head] = lse2 * kLn2;
    } else {
      const int64_t part = (int64_t)(cta * 2 + (u.j0 == 0 ? 1 : 0)) * p.rows_cap + tid;
      bars->n_off[tid] = part * 128;
      p.ws_lse[part] = lse2;
    }
  }
  meet();
#pragma unroll 1
  for (int cc = t * 8; cc < rows; cc += 16) {
    uint32_t a0[8], a1[8];
    tmem_ld8(tO + cc, a0);
    if (n > 1) tmem_ld8(tO + 128 + cc, a1);
    tmem_wait_ld();
    reg_fence<8>(a0);
    if (n > 1) reg_fence<8>(a1);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int r = cc + c;
      if (r < rows) {
        const float f0 = bars->n_alpha[0][r], f1 = bars->n_alpha[1][r];
        // a factor of 0 is no tile or nothing seen: the accumulator does not count
        float v = f0 != 0.f ? f0 * __uint_as_float(a0[c]) : 0.f;
        if (n > 1 && f1 != 0.f) v = fmaf(f1, __uint_as_float(a1[c]), v);
        if (whole)
          static_cast<uint16_t*>(p.o)[bars->n_off[r] + tid] = (uint16_t)Half16<T>::pack(v, 0.f);
        else
          p.ws_o[bars->n_off[r] + tid] = v;
      }
    }
  }
  tc_fence_before();
  meet();
  if (mine) {
    if (lane == 0) mbar_arrive(&bars->o_empty[t]);
    ++uc;
  }
  g += n;
}

template <typename T, bool kCap, bool kAlibi, bool kNarrow>
__global__ void __launch_bounds__(kCkThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tm_q,
                       const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const ChunkParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align1024(smem_raw);
  uint8_t* sQ = smem;
  uint8_t* sK = smem + 2 * kChunkTileBytes;
  uint8_t* sV = sK + kCkStages * kChunkTileBytes;
  CkBarriers* bars = reinterpret_cast<CkBarriers*>(sV + kCkStages * kChunkTileBytes);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;

  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 32) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->q_full[t], 1);
      mbar_init(&bars->q_empty[t], 1);
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->p_full[t], 4);
      mbar_init(&bars->o_full[t], 1);
      mbar_init(&bars->o_empty[t], 4);
    }
    for (int s = 0; s < kCkStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    mbar_init(&bars->mma_done, 1);
    mbar_init(&bars->merge, 8);
    for (int s = 0; s < kCkSlots; ++s) {
      mbar_init(&bars->unit_full[s], 1);
      mbar_init(&bars->unit_empty[s], 10);  // TMA, UMMA, the 8 softmax warps
    }
    fence_barrier_init();
  }

  // The line of work: units of each sequence, then key tiles of each unit, both as sums.
  if (!p.late_wait) grid_dep_wait();
  grid_dep_launch();
  const ChunkBatch& pb = p.b;
  if (threadIdx.x == 0) bars->unit_off[0] = bars->work[0] = 0;
  if (threadIdx.x < kChunkTile) {
    bars->row_token[threadIdx.x] = (uint8_t)(threadIdx.x / pb.group);
    bars->row_head[threadIdx.x] = (uint8_t)(threadIdx.x % pb.group);
  }
  constexpr int kPad = kNarrow ? kCkPadNarrow : kCkPadWide;
  bool single = true;  // at most one unit in each of this thread's sequences
#pragma unroll 1
  for (int b = threadIdx.x; b < pb.batch; b += kCkThreads) {
    const ChunkSeq q = chunk_seq(pb, b);
    if (q.bad && cta == 0) set_error(p.err, FI_DEVERR_CONTEXT_LEN);
    const bool here = (q.n * pb.group <= p.split_rows) == kNarrow;
    const int n = here ? (q.n + p.unit_tokens - 1) / p.unit_tokens : 0;
    bars->unit_off[b + 1] = (uint32_t)n;
    single &= n == 1;
    if (n == 1) {
      int np, lo, tiles;
      ck_tiles(pb, q, 0, q.n, np, lo, tiles);
      bars->work[b + 1] = (uint32_t)(tiles + kPad);
    }
  }
  uint32_t units;
  if (__syncthreads_and(single)) {  // unit b is sequence b
    units = (uint32_t)pb.batch;
    for (int b = threadIdx.x; b < pb.batch; b += kCkThreads) bars->unit_off[b + 1] = b + 1;
  } else {
    block_scan(bars->unit_off, pb.batch, bars->warp_sums);
    // cu that is not ascending could name more units than the host counted: those are dropped
    units = min(bars->unit_off[pb.batch], (uint32_t)kCkMaxUnits);
    if (units != bars->unit_off[pb.batch] && threadIdx.x == 0)
      set_error(p.err, FI_DEVERR_CONTEXT_LEN);
#pragma unroll 1
    for (int e = threadIdx.x; e < (int)units; e += kCkThreads) {
      const int b = last_le(bars->unit_off, pb.batch, (uint32_t)e);
      const ChunkSeq q = chunk_seq(pb, b);
      const int t0 = (e - (int)bars->unit_off[b]) * p.unit_tokens;
      int np, lo, n;
      ck_tiles(pb, q, t0, min(t0 + p.unit_tokens, q.n), np, lo, n);
      bars->work[e + 1] = (uint32_t)(n + kPad);
    }
    __syncthreads();
  }
  block_scan(bars->work, (int)units, bars->warp_sums);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp >= 8) {
    if constexpr (!kNarrow) setmaxnreg_dec<kCkRegsOther>();
    if (warp == 8 && lane == 0) {
      // ---------------------------------------------------------- TMA producer
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      const uint32_t q_bytes = (uint32_t)(pb.group * pb.tile_tokens * 256);
      int qc[2] = {0, 0};
      int g = 0, next_unit = 0;
      bool ok = true;
#pragma unroll 1
      for (const CkUnit* up; ok && (up = ck_next<false>(bars, next_unit, p.err)) != nullptr;
           ck_done<false>(bars, next_unit)) {
        const CkUnit& u = *up;
        auto load_q = [&]() {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || u.rows[t] == 0) continue;
            if (qc[t] > 0) ok = mbar_wait(&bars->q_empty[t], (qc[t] - 1) & 1, p.err);
            if (!ok) continue;
            const int token = u.token + t * pb.tile_tokens;
            uint8_t* dst = sQ + t * kChunkTileBytes;
            mbar_arrive_expect_tx(&bars->q_full[t], q_bytes);
            tma_load_4d(dst, &tm_q, &bars->q_full[t], 0, 0, u.hk, token);
            tma_load_4d(dst + kChunkHalf, &tm_q, &bars->q_full[t], 64, 0, u.hk, token);
            ++qc[t];
          }
        };
        int ph[2];
        for (int i = 0; i < 2; ++i) ph[i] = chunk_page(pb, u.b, u.keys, ck_tile(u, u.j0), i);
#pragma unroll 1
        for (int j = u.j0; ok && j < u.j1; ++j, ++g) {
          const int s = g % kCkStages;
          const uint32_t par = ((g / kCkStages) - 1) & 1;
          int next[2] = {0, 0};  // the next tile's pages, read while this one waits
          if (j + 1 < u.j1)
            for (int i = 0; i < 2; ++i) next[i] = chunk_page(pb, u.b, u.keys, ck_tile(u, j + 1), i);
          for (int i = 0; i < 2; ++i)
            if (ph[i] == pb.num_blocks && ck_tile(u, j) * kChunkTile + i * kChunkPage < u.keys)
              set_error(p.err, FI_DEVERR_BAD_BLOCK);
          if (g >= kCkStages && !(ok = mbar_wait(&bars->k_empty[s], par, p.err))) break;
          uint8_t* dk = sK + s * kChunkTileBytes;
          mbar_arrive_expect_tx(&bars->k_full[s], kChunkTileBytes);
          for (int i = 0; i < 2; ++i) {
            tma_load_4d(dk + i * kChunkHalf / 2, &tm_k, &bars->k_full[s], 0, u.hk, 0, ph[i]);
            tma_load_4d(dk + kChunkHalf + i * kChunkHalf / 2, &tm_k, &bars->k_full[s], 64, u.hk, 0,
                        ph[i]);
          }
          if (j == u.j0) load_q();
          if (!ok) break;
          if (g >= kCkStages && !(ok = mbar_wait(&bars->v_empty[s], par, p.err))) break;
          uint8_t* dv = sV + s * kChunkTileBytes;
          mbar_arrive_expect_tx(&bars->v_full[s], kChunkTileBytes);
          for (int i = 0; i < 2; ++i) {
            tma_load_4d(dv + i * kChunkHalf / 2, &tm_v, &bars->v_full[s], 0, u.hk, 0, ph[i]);
            tma_load_4d(dv + kChunkHalf + i * kChunkHalf / 2, &tm_v, &bars->v_full[s], 64, u.hk, 0,
                        ph[i]);
          }
          ph[0] = next[0];
          ph[1] = next[1];
        }
      }
    } else if (warp == 10) {
      ck_schedule(pb, p.unit_tokens, kPad, bars, units, p.join + cta, p.err);
    } else if (warp == 9 && lane == 0) {
      // ---------------------------------------------------------- UMMA issuer
      constexpr uint32_t idesc_qk = umma_idesc<T>(128, 128, 0, 0);
      constexpr uint32_t idesc_pv = umma_idesc<T>(128, 128, 0, 1);
      const uint32_t q_addr = smem_u32(sQ), k_addr = smem_u32(sK), v_addr = smem_u32(sV);
      int qc[2] = {0, 0};  // uses of a query tile
      int oc[2] = {0, 0};  // uses of an O accumulator
      int sc[2] = {0, 0};  // S tiles issued per tile
      int g = 0;
      bool ok = true;
      auto issue_s = [&](int t, int kstage) {
        const uint64_t da = umma_desc_sw128(q_addr + t * kChunkTileBytes, 16, 1024);
        const uint64_t db = umma_desc_sw128(k_addr + kstage * kChunkTileBytes, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t off = ((kk >> 2) * kChunkHalf + (kk & 3) * 32) >> 4;
          umma_ss(tmem + t * 128, da + off, db + off, idesc_qk, kk > 0);
        }
        umma_commit(&bars->s_full[t]);
      };
      auto issue_pv = [&](int t, int vstage, bool first) {
        const uint64_t db = umma_desc_sw128(v_addr + vstage * kChunkTileBytes, kChunkHalf, 1024);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, db + (uint32_t)(kk * 128),
                  idesc_pv, (!first || kk > 0) ? 1u : 0u);
      };
      int next_unit = 0;
#pragma unroll 1
      for (const CkUnit* up; ok && (up = ck_next<false>(bars, next_unit, p.err)) != nullptr;
           ck_done<false>(bars, next_unit)) {
        const CkUnit& u = *up;
        const int n = u.j1 - u.j0;
        if constexpr (kNarrow) {
          const uint32_t cols = (uint32_t)(u.rows[0] + 15) / 16 * 16;
          const uint32_t idesc_s = umma_idesc<T>(128, cols, 0, 0);
          const uint32_t idesc_o = umma_idesc<T>(128, cols, 1, 0);
          ok = mbar_wait(&bars->q_full[0], qc[0] & 1, p.err);
          // tile j's warpgroup is t = j & 1; its S count grows by one each, PV waits for the last
          const int sc0 = sc[0], sc1 = sc[1];
          auto step_s = [&](int j) {
            const int st = (g + j) % kCkStages, t = j & 1;
            if (!(ok = mbar_wait(&bars->k_full[st], ((g + j) / kCkStages) & 1, p.err))) return;
            tc_fence_after();
            const uint64_t da = umma_desc_sw128(k_addr + st * kChunkTileBytes, 16, 1024);
            const uint64_t db = umma_desc_sw128(q_addr, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t off = ((kk >> 2) * kChunkHalf + (kk & 3) * 32) >> 4;
              umma_ss(tmem + t * 128, da + off, db + off, idesc_s, kk > 0);
            }
            umma_commit(&bars->s_full[t]);
            umma_commit(&bars->k_empty[st]);
            if (j == n - 1) umma_commit(&bars->q_empty[0]);
          };
#pragma unroll 1
          for (int j = -2; ok && j < n; ++j) {
            if (j < 0) {
              if (j + 2 < n) step_s(j + 2);
              continue;
            }
            const int st = (g + j) % kCkStages, t = j & 1;
            ok = mbar_wait(&bars->v_full[st], ((g + j) / kCkStages) & 1, p.err) &&
                 mbar_wait(&bars->p_full[t], ((t ? sc1 : sc0) + (j >> 1)) & 1, p.err);
            const int uses = t ? oc[1] : oc[0];
            if (ok && j < 2 && uses > 0) ok = mbar_wait(&bars->o_empty[t], (uses - 1) & 1, p.err);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = umma_desc_sw128(v_addr + st * kChunkTileBytes, kChunkHalf, 1024);
            const uint64_t db = umma_desc_sw128(q_addr + kChunkTileBytes + t * kCkPBytes, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              umma_ss(tmem + 256 + t * 128, da + (uint32_t)(kk * 128),
                      db + (uint32_t)(((kk >> 2) * (kCkPBytes / 2) + (kk & 3) * 32) >> 4), idesc_o,
                      (j >= 2 || kk > 0) ? 1u : 0u);
            umma_commit(&bars->v_empty[st]);
            if (j + 2 >= n) umma_commit(&bars->o_full[t]);
            else step_s(j + 2);  // its scores overwrite those that P was made of
          }
          g += n;
          sc[0] += (n + 1) >> 1;
          sc[1] += n >> 1;
          ++qc[0];
          ++oc[0];
          if (n > 1) ++oc[1];
        } else {
        ok = mbar_wait(&bars->k_full[g % kCkStages], (g / kCkStages) & 1, p.err);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || u.rows[t] == 0) continue;
          ok = mbar_wait(&bars->q_full[t], qc[t] & 1, p.err);
          if (!ok) continue;
          tc_fence_after();
          issue_s(t, g % kCkStages);
          ++sc[t];
          if (n == 1) umma_commit(&bars->q_empty[t]);
        }
        if (ok) umma_commit(&bars->k_empty[g % kCkStages]);
#pragma unroll 1
        for (int j = 0; ok && j < n; ++j, ++g) {
          const bool has_next = j + 1 < n;
          if (has_next) {
            ok = mbar_wait(&bars->k_full[(g + 1) % kCkStages], ((g + 1) / kCkStages) & 1, p.err);
            if (!ok) break;
          }
          ok = mbar_wait(&bars->v_full[g % kCkStages], (g / kCkStages) & 1, p.err);
          if (!ok) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || u.rows[t] == 0) continue;
            ok = mbar_wait(&bars->p_full[t], (sc[t] - 1) & 1, p.err);
            // the first product of a unit overwrites O: the last unit's epilogue has read it
            if (ok && j == 0 && oc[t] > 0)
              ok = mbar_wait(&bars->o_empty[t], (oc[t] - 1) & 1, p.err);
            if (!ok) continue;
            tc_fence_after();
            issue_pv(t, g % kCkStages, j == 0);
            if (!has_next) {
              umma_commit(&bars->o_full[t]);
            } else {
              issue_s(t, (g + 1) % kCkStages);
              ++sc[t];
              if (j + 2 == n) umma_commit(&bars->q_empty[t]);
            }
          }
          if (!ok) break;
          umma_commit(&bars->v_empty[g % kCkStages]);
          if (has_next) umma_commit(&bars->k_empty[(g + 1) % kCkStages]);
        }
        for (int t = 0; t < 2; ++t)
          if (u.rows[t] > 0) ++qc[t], ++oc[t];
        }
      }
      umma_commit(&bars->mma_done);
      mbar_wait(&bars->mma_done, 0, p.err);
    }
    __syncwarp();
    named_bar_arrive(kCkTeardownBar, kCkThreads);
    return;
  }

  // ------------------------------------------- softmax + epilogue, warps 0-7
  if constexpr (!kNarrow) setmaxnreg_inc<kCkRegsSoftmax>();
  {
    const int t = warp >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_off + t * 128;
    const uint32_t tO = tmem + lane_off + 256 + t * 128;
    const float sl2 = kCap || kAlibi ? 1.f : p.f.scale_log2;
    int sc = 0;  // S tiles consumed of this tile
    int g = 0;   // K/V tiles streamed (all units)
    int uc = 0;  // units finished
    int merges = 0;
    // false once a wait ran out; the warp then goes on without waiting (see narrow_unit)
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err));
    };
    int next_unit = 0;
#pragma unroll 1
    for (const CkUnit* up; (up = ck_next<true>(bars, next_unit, p.err)) != nullptr;
         ck_done<true>(bars, next_unit)) {
      const CkUnit& u = *up;
      const int rows = t ? u.rows[1] : u.rows[0];
      const bool begins = u.j0 == 0, ends = u.j1 == u.n;
      if constexpr (kNarrow) {
        narrow_unit<T, kCap, kAlibi>(p, bars, u, sQ + kChunkTileBytes, sV, tmem, t, quarter, lane, sc,
                                     g, uc, merges, cta, ok);
      } else {
      if (rows == 0) {
        g += u.j1 - u.j0;
        continue;
      }
      const bool live = row < rows;             // this row is stored
      const bool warp_live = quarter * 32 < rows;
      const int tok = bars->row_token[row], head = u.hk * pb.group + bars->row_head[row];
      const int pos = u.pos + t * pb.tile_tokens + tok;
      float slope2 = 0.f;
      if (kAlibi && live) slope2 = p.f.slopes[head] * kLog2e;
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = u.j0; j < u.j1; ++j, ++sc, ++g) {
        const int tile = ck_tile(u, j);
        const int k0 = tile * kChunkTile;
        // (keys past the context are masked by their number)
        const bool page0 = u.pages_ok || chunk_page(pb, u.b, u.keys, tile, 0) != pb.num_blocks;
        const bool page1 = u.pages_ok || chunk_page(pb, u.b, u.keys, tile, 1) != pb.num_blocks;
        wait(&bars->s_full[t], sc & 1);
        if (t == 0 && k0 + kChunkTile > u.keys) {
          wait(&bars->v_full[g % kCkStages], (g / kCkStages) & 1);
          zero_v_rows(sV + (g % kCkStages) * kChunkTileBytes, max(u.keys - k0, 0), threadIdx.x);
          fence_proxy_async_smem();
        }
        if (warp_live) {
          tc_fence_after();
          // columns [c_lo, c_hi) and [0, c_pre) are visible
          const int c_hi = min(pos + 1, u.keys) - k0, c_pre = u.prefix - k0;
          const int c_lo = pb.window ? pos - pb.window + 1 - k0 : 0;
          const bool all = !live || ((c_hi >= kChunkTile && c_lo <= 0) || c_pre >= kChunkTile);
          const bool mask = !__all_sync(0xffffffffu, all && page0 && page1);
          if (kCap || kAlibi || mask) {
            // the score's form and the mask, 32 columns at a time, back into tensor memory
#pragma unroll 1
            for (int cc = 0; cc < kChunkTile; cc += 32) {
              uint32_t sr[32];
              tmem_ld32(tS + cc, sr);
              tmem_wait_ld();
              reg_fence<32>(sr);
              score_form<kCap, kAlibi>(sr, p.f, slope2, (float)(k0 + cc - pos), live);
              if (mask) {
                uint32_t vis = (low_bits(c_hi - cc, 0) & ~low_bits(c_lo - cc, 0)) |
                               low_bits(c_pre - cc, 0);
                if (!(cc < 64 ? page0 : page1)) vis = 0;
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  if (!((vis >> c) & 1u)) sr[c] = __float_as_uint(-INFINITY);
              }
              tmem_st32(tS + cc, sr);
            }
            tmem_wait_st();
          }
          uint32_t sr[kChunkTile];
          tmem_ld32(tS + 0, sr + 0);
          tmem_ld32(tS + 32, sr + 32);
          tmem_ld32(tS + 64, sr + 64);
          tmem_ld32(tS + 96, sr + 96);
          tmem_wait_ld();
          reg_fence<kChunkTile>(sr);
          float mx8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float a = __uint_as_float(sr[i]);
#pragma unroll
            for (int kk = 1; kk < 15; kk += 2)
              a = fmax3_nan(a, __uint_as_float(sr[i + 8 * kk]),
                            __uint_as_float(sr[i + 8 * (kk + 1)]));
            mx8[i] = fmax_nan(a, __uint_as_float(sr[i + 120]));
          }
          // NaN where any score is: the whole row is NaN then, whichever columns hold it
          const float mx = fmax_nan(fmax3_nan(mx8[0], mx8[1], mx8[2]),
                                    fmax3_nan(fmax3_nan(mx8[3], mx8[4], mx8[5]), mx8[6], mx8[7]));
          const float m_new = fmax_nan(m, mx * sl2);
          bool rescale = false;
          float alpha = 1.f;
          if (j == u.j0) {
            m = m_new;
          } else {
            const bool need = !(m_new <= m + kCkRescale) && m == m;  // (once to NaN; it stays)
            rescale = __any_sync(0xffffffffu, need);
            if (need) {
              alpha = fast_exp2(m - m_new);
              m = m_new;
              l *= alpha;
            }
          }
          l += ck_exp<T>(sr, sl2, m == -INFINITY ? 0.f : m);
          tmem_st32(tS + 0, sr);
          tmem_st32(tS + 32, sr + 32);
          if (rescale) {
            // the previous step's product is complete: S of this step was committed after it
#pragma unroll
            for (int cc = 0; cc < 128; cc += 32) {
              uint32_t ov[32];
              tmem_ld32(tO + cc, ov);
              tmem_wait_ld();
              reg_fence<32>(ov);
#pragma unroll
              for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
              tmem_st32(tO + cc, ov);
            }
          }
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[t]);
      }
      // ----------------------------------------------------------- epilogue
      wait(&bars->o_full[t], uc & 1);
      tc_fence_after();
      const bool none = m == -INFINITY;
      const float inv = none ? 0.f : 1.f / l;
      const float lse2 = none ? -INFINITY : m + log2f(l);
      const int64_t out_row = u.token + t * pb.tile_tokens + tok;
      const int64_t part = (int64_t)(cta * 2 + (begins ? 1 : 0)) * p.rows_cap + t * 128 + row;
      T* orow = static_cast<T*>(p.o) + out_row * p.os[0] + head * p.os[1];
      float* prow = p.ws_o + (part & ~31) * 128 + (part & 31) * 4;
      if (warp_live) {
#pragma unroll 1
        for (int cc = 0; cc < 128; cc += 32) {
          uint32_t ov[32];
          tmem_ld32(tO + cc, ov);
          tmem_wait_ld();
          reg_fence<32>(ov);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            ov[e] = none ? 0u : __float_as_uint(__uint_as_float(ov[e]) * inv);
          if (live && begins && ends) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              uint32_t pk[8];
#pragma unroll
              for (int i = 0; i < 8; ++i)
                pk[i] = Half16<T>::pack(__uint_as_float(ov[e + 2 * i]), __uint_as_float(ov[e + 2 * i + 1]));
              if (p.o_wide) {
                st_global_v8(orow + cc + e, pk);
              } else {
                *reinterpret_cast<uint4*>(orow + cc + e) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                *reinterpret_cast<uint4*>(orow + cc + e + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
              }
            }
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(prow + (cc + e) * 32) =
                  make_uint4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
          }
        }
        if (live) {
          if (begins && ends) {
            if (p.lse) p.lse[out_row * pb.hq + head] = lse2 * kLn2;
          } else {
            p.ws_lse[part] = lse2;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->o_empty[t]);
      ++uc;
      }
    }
  }

  if (p.late_wait && threadIdx.x == 0) grid_dep_wait();
  __syncwarp();
  tc_fence_before();
  named_bar_sync(kCkTeardownBar, kCkThreads);
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a unit that several CTAs hold: weights 2^(lse_part - max), the max running.
// A block joins kCkJoinRows rows of one CTA's unit: `p`'s first, then `p2`'s. A thread has 8 values
// of a row: a warp those of two rows, or of 16 rows where 32 rows lie side by side. Bound by issue
// slots, not by memory (512 new tokens over 2000: 34.4 us in all; 4 values a thread 35.8).
constexpr int kCkJoinRows = 16;
template <typename T>
__global__ void __launch_bounds__(256, 5) chunk_combine_kernel(const ChunkParams p,
                                                               const ChunkParams p2) {
  grid_dep_wait();
  grid_dep_launch();
  const bool second = (int)blockIdx.y >= p.rows_cap / kCkJoinRows;
  const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = ((int)blockIdx.y - (second ? p.rows_cap / kCkJoinRows : 0)) * kCkJoinRows;
  const CkJoin jn = second ? p2.join[cta] : p.join[cta];
  if (!jn.valid) return;
  const int rows_cap = second ? p2.rows_cap : p.rows_cap;
  const bool by_row = rows_cap == kCkNarrow;
  const float* ws_lse = second ? p2.ws_lse : p.ws_lse;
  const float* ws_o = second ? p2.ws_o : p.ws_o;
  const int r = r0 + (by_row ? warp * 2 + (lane >> 4) : lane & 15), t = r >> 7, row = r & 127;
  const int col = (by_row ? lane & 15 : warp * 2 + (lane >> 4)) * 8;
  if (row >= (t ? jn.rows[1] : jn.rows[0])) return;
  const int off = by_row ? r * 128 + col : (r & ~31) * 128 + col * 32 + (r & 31) * 4;
  const int far = by_row ? 4 : 128;  // from the first 4 values to the others
  float mx = -INFINITY, sum = 0.f, acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int c = cta; c <= jn.last_cta; ++c) {
    const int at = (c * 2 + (c == cta ? 1 : 0)) * rows_cap;
    const float l = ws_lse[at + r];
    const float* src = ws_o + at * 128 + off;
    const float4 v = *reinterpret_cast<const float4*>(src);
    const float4 w = *reinterpret_cast<const float4*>(src + far);
    const float x[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
    if (l > mx) {
      const float a = fast_exp2(mx - l);
      mx = l;
      sum *= a;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= a;
    }
    const float wgt = l == -INFINITY ? 0.f : fast_exp2(l - mx);
    sum += wgt;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(wgt, x[i], acc[i]);
  }
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  const int64_t token = jn.token + t * p.b.tile_tokens + row / p.b.group;
  const int head = jn.hk * p.b.group + row % p.b.group;
  uint4 pk;
  pk.x = Half16<T>::pack(acc[0] * inv, acc[1] * inv);
  pk.y = Half16<T>::pack(acc[2] * inv, acc[3] * inv);
  pk.z = Half16<T>::pack(acc[4] * inv, acc[5] * inv);
  pk.w = Half16<T>::pack(acc[6] * inv, acc[7] * inv);
  *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + token * p.os[0] + head * p.os[1] + col) = pk;
  if (col == 0 && p.lse) p.lse[token * p.b.hq + head] = none ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

template <typename T, bool kCap, bool kAlibi, bool kNarrow>
static int launch_main(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                       const ChunkParams& p, cudaStream_t st) {
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    // the register split must fit what the block is launched with, or setmaxnreg would wait
    cudaFuncAttributes a;
    const cudaError_t e = cudaFuncGetAttributes(&a, paged_chunk_kernel<T, kCap, kAlibi, kNarrow>);
    if (e != cudaSuccess) return e;
    if (!kNarrow && a.numRegs * kCkThreads < 2 * 128 * kCkRegsSoftmax + 128 * kCkRegsOther)
      return cudaErrorInvalidConfiguration;
    return cudaFuncSetAttribute(paged_chunk_kernel<T, kCap, kAlibi, kNarrow>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, kCkSmemBytes);
  });
  if (e != cudaSuccess) return cuda_fail(e, "fi_paged_chunk: kernel set-up");
  e = launch_pdl(paged_chunk_kernel<T, kCap, kAlibi, kNarrow>, dim3((unsigned)sm_count()),
                 dim3(kCkThreads), kCkSmemBytes, st, tq, tk, tv, p);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_paged_chunk: launch");
}

template <typename T, bool kNarrow>
static int launch_form(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                       const ChunkParams& p, cudaStream_t st) {
  if (p.f.cap_log2 > 0.f)
    return p.f.slopes ? launch_main<T, true, true, kNarrow>(tq, tk, tv, p, st)
                      : launch_main<T, true, false, kNarrow>(tq, tk, tv, p, st);
  return p.f.slopes ? launch_main<T, false, true, kNarrow>(tq, tk, tv, p, st)
                    : launch_main<T, false, false, kNarrow>(tq, tk, tv, p, st);
}

// The narrow kernel, the wide one or both (whichever `narrow` and `wide` name), and the join.
template <typename T>
static int launch_chunk(const CUtensorMap& tq_n, const CUtensorMap& tq_w, const CUtensorMap& tk,
                        const CUtensorMap& tv, const ChunkParams* narrow, const ChunkParams* wide,
                        cudaStream_t st) {
  int r = narrow ? launch_form<T, true>(tq_n, tk, tv, *narrow, st) : FI_OK;
  if (r == FI_OK && wide) r = launch_form<T, false>(tq_w, tk, tv, *wide, st);
  if (r != FI_OK) return r;
  const ChunkParams& first = wide ? *wide : *narrow;
  const int parts = (first.rows_cap + (narrow && wide ? narrow->rows_cap : 0)) / kCkJoinRows;
  const cudaError_t e =
      launch_pdl(chunk_combine_kernel<T>, dim3((unsigned)sm_count(), (unsigned)parts), dim3(256), 0,
                 st, first, narrow ? *narrow : first);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_paged_chunk: combine launch");
}

static size_t ck_align(size_t n) { return (n + 255) / 256 * 256; }

// One kernel's part of the workspace; `p` null: its size alone.
static size_t ck_workspace(ChunkParams* p, uint8_t* ws, int rows_cap) {
  const size_t slots = (size_t)sm_count() * 2 * rows_cap;
  const size_t o = ck_align(slots * 128 * 4), lse = ck_align(slots * 4);
  if (p) {
    p->ws_o = reinterpret_cast<float*>(ws);
    p->ws_lse = reinterpret_cast<float*>(ws + o);
    p->join = reinterpret_cast<CkJoin*>(ws + o + lse);
    p->rows_cap = rows_cap;
  }
  return o + lse + ck_align(sm_count() * sizeof(CkJoin));
}

// Whether every sequence can only have so few rows that the narrow kernel serves the batch.
static bool ck_all_narrow(int64_t total, int64_t group) { return total * group <= kCkNarrow; }

}  // namespace fi

extern "C" size_t fi_paged_chunk_workspace_size(int64_t total_tokens, int64_t num_q_heads,
                                                int64_t num_kv_heads) {
  using namespace fi;
  if (total_tokens <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads ||
      num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 64 ||
      total_tokens > (1 << 28))
    return 0;
  const size_t narrow = ck_workspace(nullptr, nullptr, kCkNarrow);
  if (ck_all_narrow(total_tokens, num_q_heads / num_kv_heads)) return narrow;
  return narrow + ck_workspace(nullptr, nullptr, 2 * kChunkTile);
}

extern "C" int fi_paged_chunk(const void* q, const void* k_cache, const void* v_cache, void* o,
                              float* lse, const int32_t* block_table, const int32_t* cu_seqlens,
                              const int32_t* context_lens, const int32_t* prefix_lens,
                              const float* alibi_slopes, int64_t batch, int64_t total_tokens,
                              int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                              int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq,
                              const int64_t* q_strides, const int64_t* kc_strides,
                              const int64_t* vc_strides, const int64_t* o_strides,
                              const int64_t* bt_strides, float sm_scale, float softcap,
                              int64_t window, int64_t dtype, void* workspace,
                              size_t workspace_bytes, int32_t* error_flag, void* stream) {
  using namespace fi;
  clear_error();
  const char* what = "fi_paged_chunk";
  ChunkParams p = {};
  int r = chunk_batch_args(p.b, what, cu_seqlens, context_lens, prefix_lens, block_table, batch,
                           total_tokens, num_q_heads, num_kv_heads, head_dim, num_blocks,
                           block_size, max_blocks_per_seq, bt_strides, window, dtype);
  if (r != FI_OK) return r;
  r = chunk_score_args(p.f, what, sm_scale, softcap, alibi_slopes);
  if (r != FI_OK) return r;
  if (batch == 0 || total_tokens == 0) return FI_OK;
  if (!q || !k_cache || !v_cache || !o || !block_table || !cu_seqlens || !context_lens ||
      !q_strides || !kc_strides || !vc_strides || !o_strides || !bt_strides)
    return fail(FI_ERR_INVALID_ARG, "fi_paged_chunk: null pointer argument");
  // Batches of few tokens per sequence (on average at most kCkNarrow rows) are the narrow
  // kernel's alone: a sequence with more tokens is several units there, which read its keys once
  // each (from L2), unless there are many new tokens: 512 of one sequence over 2000 beside 64
  // single ones over 4000 take 238 us there and 219 in both kernels, but the wide one costs 11 us
  // when it has nothing to do. One sequence with more is the wide kernel's. Other batches may hold
  // both.
  const int64_t per_unit = p.b.group <= kCkNarrow ? kCkNarrow / p.b.group : 0;
  const bool use_narrow = per_unit > 0 && (batch > 1 || total_tokens <= per_unit);
  const bool use_wide =
      per_unit == 0 || total_tokens > batch * per_unit || total_tokens - batch >= kCkManyNew;
  const int64_t unit_tokens = use_wide ? 2 * p.b.tile_tokens : per_unit;
  if (batch > kCkMaxBatch ||
      (total_tokens + unit_tokens - 1) / unit_tokens + batch > kCkMaxUnits)
    return fail(FI_ERR_UNSUPPORTED,
                "fi_paged_chunk: at most %d sequences and %lld tokens with %d query heads per KV "
                "head; split the batch",
                kCkMaxBatch, (long long)((kCkMaxUnits - batch) * unit_tokens), p.b.group);
  if (o_strides[2] != 1 || !aligned16(o) || !stride_ok(total_tokens, o_strides[0]) ||
      !stride_ok(num_q_heads, o_strides[1]))
    return fail(FI_ERR_ALIGNMENT,
                "fi_paged_chunk o: needs a 16-byte aligned base, unit innermost stride and other "
                "strides multiple of 8");
  const size_t need = fi_paged_chunk_workspace_size(total_tokens, num_q_heads, num_kv_heads);
  if (!workspace || workspace_bytes < need)
    return fail(FI_ERR_WORKSPACE, "fi_paged_chunk: workspace of %zu bytes, needs %zu",
                workspace ? workspace_bytes : (size_t)0, need);
  if (!aligned16(workspace))
    return fail(FI_ERR_ALIGNMENT, "fi_paged_chunk: workspace not 16-byte aligned");
  const CUtensorMapDataType type = dtype == FI_DTYPE_F16 ? Half16<__half>::kTmap
                                                         : Half16<__nv_bfloat16>::kTmap;
  ChunkParams n = p;  // the narrow kernel's
  n.b.tile_tokens = per_unit > 0 ? (int)per_unit : 1;
  CUtensorMap tq_n = {}, tq_w = {}, tk, tv;
  if (use_narrow && (r = chunk_q_map(&tq_n, type, q, n.b, q_strides, "fi_paged_chunk q")) != FI_OK)
    return r;
  if (use_wide && (r = chunk_q_map(&tq_w, type, q, p.b, q_strides, "fi_paged_chunk q")) != FI_OK)
    return r;
  if ((r = chunk_kv_map(&tk, type, k_cache, p.b, kc_strides, "fi_paged_chunk k_cache")) != FI_OK)
    return r;
  if ((r = chunk_kv_map(&tv, type, v_cache, p.b, vc_strides, "fi_paged_chunk v_cache")) != FI_OK)
    return r;
  p.o = o;
  p.os[0] = o_strides[0];
  p.os[1] = o_strides[1];
  p.o_wide = reinterpret_cast<uintptr_t>(o) % 32 == 0 &&
             (total_tokens == 1 || o_strides[0] % 16 == 0) &&
             (num_q_heads == 1 || o_strides[1] % 16 == 0);
  p.lse = lse;
  p.err = error_flag;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  {
    const ChunkBatch nb = n.b;
    n = p;
    n.b = nb;
  }
  ws += ck_workspace(&n, ws, kCkNarrow);
  if (use_wide) ck_workspace(&p, ws, 2 * kChunkTile);
  n.unit_tokens = (int)per_unit;
  n.split_rows = use_wide ? kCkNarrow : 0x7fffffff;
  p.unit_tokens = 2 * p.b.tile_tokens;
  p.split_rows = use_narrow ? kCkNarrow : 0;
  p.late_wait = use_narrow;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const ChunkParams* np = use_narrow ? &n : nullptr;
  const ChunkParams* wp = use_wide ? &p : nullptr;
  return dtype == FI_DTYPE_F16 ? launch_chunk<__half>(tq_n, tq_w, tk, tv, np, wp, st)
                               : launch_chunk<__nv_bfloat16>(tq_n, tq_w, tk, tv, np, wp, st);
}
