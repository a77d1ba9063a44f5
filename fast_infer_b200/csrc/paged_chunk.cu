// Attention of new tokens over the paged KV cache (chunked prefill, verification of drafted tokens and
// trees of them, single tokens, and batches that mix them), on sm_100a tensor cores.
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
// * Trees (kTree): a token sees the cached tokens before the new ones and, of the new ones, those of its bit mask; only
//   tiles that hold new tokens read masks. New tokens of at most two row tiles are split evenly over both, and a unit
//   with rows for one tile only is taken by both warpgroups, alternate key tiles each, merged through tensor
//   memory at its end (one warpgroup idle instead: 16 trees of 9 to 33 tokens over 500 to 4000, scores capped, 15 us
//   more; uneven tiles: 8 of 50 to 85 tokens over 20000 to 32000, 17 us more). The 16 take 59 us (178 MB, 27 at a copy's
//   rate), bound by the chain of a step and a start of 15 us; the 8 over codes take 340 us (fp16 334).
// * Pages of 8-bit codes (Code): TMA brings a tile's codes into the half of its place that they fill, and the softmax
//   warpgroups spread them to 16 bits in place while they would wait for the first product (in warps of their
//   own, two or four, 40 to 60 us more for the 8 trees above; with 16-bit pages they take 212). K's scales multiply scores
//   in fp32, V's go onto P in fp32; for fp16, which lacks fp32's range, the softmax then runs relative to a maximum of
//   score + log2 of V's scale (ck_reference). Spreading and softmax, 6600 cycles a tile, bound it.
// * Slots behind a sequence's last token may hold anything: their scores are replaced by
//   -inf, and their V rows are zeroed in shared memory before the product (0 * NaN is NaN).
#include <float.h>

#include <type_traits>

#include "paged_chunk.cuh"
#include "quant8.cuh"

namespace fi {

constexpr int kCkThreads = 384;
constexpr int kCkRegsSoftmax = 184;  // 2 x 128 x 184 + 128 x 136 = 384 x 168
constexpr int kCkRegsOther = 136;
// Scales of a key tile are read after its product is done, that is after its stage may be filled again. The place of tile j
// is written for tile j + 4 once K of that has arrived, so once S of tile j + 2 is complete. S of tile j + 2 is issued
// after the product with V of tile j (where the warpgroups alternate key tiles; else of tile j + 1), which waits
// for the weights of tile j, and S of a unit's first tiles after all products of the unit before.
constexpr int kCkScaleSlots = 4;
constexpr int kCkStages = 2;
constexpr int kCkTeardownBar = 15;
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
  int keys, prefix;    // with a tree, `prefix` is the sequence's first new slot instead
  int np, lo;          // step j is key tile j < np ? j : lo + j - np
  int j0, j1, n;
  int pages_ok;        // no block-table entry of its keys is invalid
  int last_cta;        // the CTA with the unit's last step
  int valid;           // 0: no unit is left
};
static_assert(sizeof(CkUnit) == 64, "read as four 16-byte words");

struct CkBarriers {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kCkStages], k_empty[kCkStages];
  uint64_t v_full[kCkStages], v_empty[kCkStages];
  uint64_t s_full[2], p_full[2], o_full[2], o_empty[2];
  uint64_t mma_done;
  uint64_t unit_full[kCkSlots], unit_empty[kCkSlots];
  uint64_t kc_full[kCkStages], vc_full[kCkStages];  // codes have arrived
  alignas(16) float k_scale[kCkScaleSlots][kChunkTile];
  alignas(16) float v_scale[kCkScaleSlots][kChunkTile];
  alignas(16) float v_top[kCkScaleSlots][4];  // log2 of the greatest, of 32 each
  uint64_t merge;  // both softmax warpgroups, in a transposed unit
  uint32_t tmem_base;
  // transposed units, per warpgroup: rows' max, partial maxima / sums, scale, slope, token
  float n_max[2][kCkNarrow], n_red[2][4][kCkNarrow], n_alpha[2][kCkNarrow];
  alignas(16) float n_neg[2][kCkNarrow];  // -max; FLT_MAX: no score yet, -inf: no such row
  float n_slope[2][kCkNarrow], n_pos[2][kCkNarrow];
  int64_t n_off[kCkNarrow];  // where a row's output goes
  float twin_mv[4][32];      // m' of the second warpgroup's rows, where both have them
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

__device__ __forceinline__ int ck_tile(const CkUnit& u, int j) {
  return j < u.np ? j : u.lo + (j - u.np);
}

// The scheduler (one warp): walks the CTA's part of the line and hands its units to the other
// roles through a ring in shared memory. Its lanes look the units' pages over, so that no one
// else has to unless an entry is invalid. On the line a unit is `pad` steps longer than its key
// tiles, which stand for what it costs to begin and end one; its step j is at pad + j.
struct CkScheduler {
  const ChunkBatch& p;
  CkBarriers* s;
  CkJoin* join_out;
  int* err;
  int64_t total, w, end;
  uint32_t units;
  int unit_tokens, pad, active;
  int hk, e, b, at;  // `at`: where in the unit this CTA begins
  int i;             // units handed out
  bool open;         // some may be left
  bool even;         // tokens for two tiles are split evenly over them, not the first one filled
  ChunkSeq q;
  CkJoin join;

  __device__ __forceinline__ CkScheduler(const ChunkBatch& p, int unit_tokens, int pad,
                                         CkBarriers* s, uint32_t units, CkJoin* join_out, int* err,
                                         bool even)
      : p(p), s(s), join_out(join_out), err(err), units(units), unit_tokens(unit_tokens), pad(pad),
        even(even) {
    const int G = gridDim.x, cta = blockIdx.x;
    const uint32_t per_head = s->work[units];
    total = (int64_t)per_head * p.hk;
    active = (int)(total < G ? total : G);  // CTAs with work
    w = cta < active ? total * cta / active : 0;
    end = cta < active ? total * (cta + 1) / active : 0;
    hk = e = b = at = 0;
    if (w < end) {
      hk = (int)(w / per_head);
      const uint32_t r = (uint32_t)(w - (int64_t)hk * per_head);
      e = last_le(s->work, (int)units, r);
      b = last_le(s->unit_off, p.batch, (uint32_t)e);
      at = (int)(r - s->work[e]);
    }
    q = chunk_seq(p, b);
    join = {};
    i = 0;
    open = true;
  }

  // The next unit into the ring, an invalid one after the last.
  __device__ __forceinline__ void next() {
    const int cta = blockIdx.x, lane = threadIdx.x & 31, slot = i % kCkSlots;
    if (i >= kCkSlots &&
        !__all_sync(0xffffffffu, mbar_wait(&s->unit_empty[slot], ((i / kCkSlots) - 1) & 1, err))) {
      open = false;
      return;
    }
    ++i;
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
      u.prefix = p.tree ? q.pos0 : q.prefix;
      // (where two tiles are needed: 8 trees of 50 to 85 tokens over 20 to 32 k, 366 us, split evenly 349;
      // with rows for one tile only, a second one would be work for nothing: 99 us, and 109)
      const int tt = even && t1 - t0 > p.tile_tokens ? (t1 - t0 + 1) / 2 : p.tile_tokens;
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
    open = u.valid;
  }
  __device__ __forceinline__ void finish() {
    if ((threadIdx.x & 31) == 0) *join_out = join;
  }
};

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
// rounding: 3.0e-4 in place of the 2.1e-4 of P in 32 bits (root mean square, relative; bf16 2.3e-3 and
// 1.7e-3). P as the sum of two such values would take the product twice; P and V's codes in fp16 under
// bf16, 5 to 13 % of the time over codes.
// Over codes P takes the scales of V's rows (and the sum does not), and with kRun the row's `factor` (see ck_reference).
template <typename T, bool kCode, bool kRun>
__device__ __forceinline__ float ck_exp(uint32_t* sr, float sl2, float mref, const float* v_scale, float factor) {
  const uint64_t sc2 = f32x2(sl2, sl2), nm2 = f32x2(-mref, -mref);
  uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
  // (over codes the special function units wait for the issue slots as it is)
  constexpr int kEmu = kCode ? 0 : kCkEmuPairs;
#pragma unroll
  for (int c = 0; c < kChunkTile; c += 4) {
    ulonglong2 f = make_ulonglong2(0, 0);
    if constexpr (kCode) f = *reinterpret_cast<const ulonglong2*>(v_scale + c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = c + 2 * i;
      const uint64_t xp =
          fma_f32x2(f32x2(__uint_as_float(sr[d]), __uint_as_float(sr[d + 1])), sc2, nm2);
      float p0, p1;
      if (((d >> 1) & 7) < kEmu) {
        f32x2_split(exp2_poly5_x2(xp), p0, p1);
      } else {
        float x0, x1;
        f32x2_split(xp, x0, x1);
        p0 = fast_exp2(x0);
        p1 = fast_exp2(x1);
      }
      uint64_t pp = f32x2(p0, p1);
      sum2[(d >> 1) & 3] = add_f32x2(sum2[(d >> 1) & 3], pp);
      if constexpr (kRun) pp = mul_f32x2(pp, f32x2(factor, factor));
      if constexpr (kCode) f32x2_split(mul_f32x2(pp, i ? f.y : f.x), p0, p1);
      sr[d >> 1] = Half16<T>::pack(p0, p1);
    }
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
template <typename T, bool kCap, bool kAlibi, bool kTree>
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
    uint32_t tree_vis = 0xffffffffu;
    if constexpr (kTree) {
      // a new token's key: the bits of the unit's tokens; one before them: by the tokens' depths
      if (key >= u.prefix || pb.window) {
        tree_vis = 0;
#pragma unroll 4
        for (int i = 0; i * pb.group < rows; ++i) {
          const bool see = key >= u.prefix
                               ? (tree_bits(pb, u.token + i, key - u.prefix) & 1u) != 0
                               : key > u.prefix + pb.depths[u.token + i] - pb.window;
          if (see) tree_vis |= low_bits((i + 1) * pb.group, 0) & ~low_bits(i * pb.group, 0);
        }
      }
    } else if (key >= u.prefix) {
      c_lo = min(max(key - u.pos, 0), kCkNarrow) * pb.group;
      if (pb.window) c_hi = min(rows, min(max(key + pb.window - u.pos, 0), kCkNarrow) * pb.group);
    }
    if (!page_ok || key >= u.keys) c_hi = 0;
    const uint32_t vis = low_bits(c_hi, 0) & ~low_bits(c_lo, 0) & tree_vis;
    const bool mask = !__all_sync(
        0xffffffffu, kTree ? (vis & low_bits(rows, 0)) == low_bits(rows, 0) : c_lo <= 0 && c_hi >= rows);
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

// Scores of one row times the scales of their keys.
template <int N>
__device__ __forceinline__ void scale_columns(uint32_t* sr, const float* scale) {
#pragma unroll
  for (int c = 0; c < N; c += 4) {
    const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(scale + c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float a, b;
      f32x2_split(mul_f32x2(f32x2(__uint_as_float(sr[c + 2 * i]), __uint_as_float(sr[c + 2 * i + 1])),
                            i ? f.y : f.x),
                  a, b);
      sr[c + 2 * i] = __float_as_uint(a);
      sr[c + 2 * i + 1] = __float_as_uint(b);
    }
  }
}

// Codes under fp16: P times V's scales does not go into 16 bits as it is (a scale may be 1e-30 or 1e30), nor do V's codes
// times them. So P' = p vs 2^(m - m') does, with m' a running maximum of s + log2(vs), less 5; O goes with m', the sum of p
// with m (m' for both would cost lse two bits). m' moves where a bound of s + log2(vs), the row's greatest score with the
// tile's greatest scale, is past m' + 15: P' is below 2^15, and what is 2^-19 of a row's greatest and more is rounded by half
// a step of its own (from 2^0 on, P' of 2^-14 would lose bits: with scales far apart a good part of the keys). m' is
// at least m - 100, where the factor is finite, for rows of zeros may hold all the weight; what a scale of 2^-100 leaves is
// 2^-76 of fp16's least value.
// Here: m' for a tile of scores in tensor memory (times `k_scale`, if they are not yet), from `m` so far, in two passes over
// it, for a unit's first tile and the few where m' may move. 8 scores at a time keep its code short: it is seldom in the
// instruction caches (8 trees of 50 to 85 tokens over 20 to 32 k, int8 under fp16, in an earlier form: with 32 at a time
// 491 us, with 8 407, and 361 where m' lies 5 rather than 8 below the maximum, so that it moves less often).
template <typename T>
constexpr bool kCkRunScale = std::is_same_v<T, __half>;
constexpr float kCkRunTop = 15.f, kCkRunRoom = 5.f, kCkRunGap = 100.f;
__device__ __forceinline__ float ck_reference(uint32_t tS, float sl2, const float* k_scale, const float* v_scale,
                                              float m) {
  float mx = -INFINITY, top = 0.f;
#pragma unroll 1
  for (int i = 0; i < 2 * kChunkTile; i += 8) {
    const int cc = i % kChunkTile;
    const float ref = mx == -INFINITY ? 0.f : mx;
    uint32_t sr[8];
    tmem_ld8(tS + cc, sr);
    tmem_wait_ld();
    reg_fence<8>(sr);
    if (k_scale) scale_columns<8>(sr, k_scale + cc);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float s = __uint_as_float(sr[c]) * sl2;
      if (i < kChunkTile) mx = fmaxf(mx, s);
      else top = fmaxf(top, fast_exp2(s - ref) * v_scale[cc + c]);
    }
  }
  return fmax3f(m, mx + (__log2f(top) - kCkRunRoom), mx - kCkRunGap);
}

// 16 codes as 16-bit values of type T (exact).
template <typename T, typename Code>
__device__ __forceinline__ void spread16(const uint4& raw, uint32_t* out) {
  const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h[2];
    if constexpr (std::is_same_v<T, __nv_bfloat16> && std::is_same_v<Code, CodeI8>) {
      CodeI8::decode4_bf16(r[i], out[2 * i], out[2 * i + 1]);
      continue;
    }
    Code::decode4(r[i], h[0], h[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (std::is_same_v<T, __half>) {
        out[2 * i + j] = h[j];
      } else {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[j]));
        out[2 * i + j] = Half16<T>::pack(f.x, f.y);
      }
    }
  }
}

// Between TMA and the tensor core: a warpgroup spreads the codes of a tile (128 keys x 128 bytes, 128-byte swizzle),
// which lie in the first half of the tile's 16-bit place, a row where its first 64 values will be, so that the 8
// lanes of a row read it and then write over it. Lanes are given rows r and r ^ 5 such that neither the reads
// nor the writes of 8 lanes meet a bank twice.
template <typename T, typename Code>
__device__ __forceinline__ void spread_tile(uint8_t* tile, int live, int quarter) {
  const int lane = threadIdx.x & 31;
  const int q = lane & 3, flip = (lane >> 2) & 1 ? 5 : 0, column = (lane >> 3) & 1, pair = lane >> 4;
  const int piece = column * 4 + q;
#pragma unroll 1
  for (int i0 = 0; i0 < 8; i0 += 4) {  // 16 rows' reads before their writes
    uint4 raw[4];
    int row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      row[i] = 32 * quarter + 4 * i0 + 8 * (i >> 1) + (((i & 1) * 2 + pair) ^ flip);
      raw[i] = *reinterpret_cast<const uint4*>(tile + row[i] * 128 + ((piece ^ (row[i] & 7)) << 4));
      if (row[i] >= live) raw[i] = make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t v[8];
      spread16<T, Code>(raw[i], v);
      uint8_t* to = tile + column * kChunkHalf + row[i] * 128;
      *reinterpret_cast<uint4*>(to + (((2 * q) ^ (row[i] & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<uint4*>(to + (((2 * q + 1) ^ (row[i] & 7)) << 4)) =
          make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// The softmax warpgroups spread codes where they would wait: after the weights of tile j, the first one K of
// tile j + 2 (its stage is free since S of tile j), the second one V of tile j + 1, and both the first tiles of
// the next unit before a unit's end. (Warps of their own for it: four cost the softmax its registers,
// two were slower than the tensor core, 408 us for 8 trees over 20 to 32 k keys.)
// K and V keep their codes, which are exact in T. A thread of the first one looks up the scales of one row. Rows of keys past
// the context are zero, like those without a page.
template <typename T, typename Code>
struct CodeSpreader {
  const ChunkParams& p;
  CkBarriers* bars;
  uint8_t* tiles;  // K's or V's
  int t, quarter, row;
  int g;           // tiles spread so far
  float k, v;      // scales of `row` of the next one

  __device__ __forceinline__ CodeSpreader(const ChunkParams& p, CkBarriers* bars, uint8_t* sK,
                                          uint8_t* sV, int t, int quarter)
      : p(p), bars(bars), tiles(t ? sV : sK), t(t), quarter(quarter),
        row(quarter * 32 + (threadIdx.x & 31)), g(0), k(0.f), v(0.f) {}

  __device__ __forceinline__ int page(const CkUnit& u, int j) const {
    return chunk_page(p.b, u.b, u.keys, ck_tile(u, j), row >> 6);
  }
  __device__ __forceinline__ void look_up(const CkUnit& u, int j, int page) {
    const bool held = page != p.b.num_blocks && ck_tile(u, j) * kChunkTile + row < u.keys;
    const int64_t slot = row & (kChunkPage - 1);
    k = v = 0.f;
    if (held && t == 0) {
      k = p.scale[0][page * p.ss[0][0] + u.hk * p.ss[0][1] + slot * p.ss[0][2]];
      v = p.scale[1][page * p.ss[1][0] + u.hk * p.ss[1][1] + slot * p.ss[1][2]];
    }
  }
  // Tile j of the unit, whose scales have been looked up.
  template <typename Wait>
  __device__ __forceinline__ void spread(const CkUnit& u, int j, Wait&& wait) {
    const int s = g % kCkStages;
    wait(t ? &bars->vc_full[s] : &bars->kc_full[s], (g / kCkStages) & 1);
    if (t == 0) {
      bars->k_scale[g % kCkScaleSlots][row] = k;
      bars->v_scale[g % kCkScaleSlots][row] = v;
      if constexpr (kCkRunScale<T>) {  // (not negative, so in the order of their bits)
        const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
        if ((threadIdx.x & 31) == 0) bars->v_top[g % kCkScaleSlots][quarter] = __log2f(top);
      }
    }
    const int live = u.keys - ck_tile(u, j) * kChunkTile;
    spread_tile<T, Code>(tiles + s * kChunkTileBytes, live, quarter);
    if ((threadIdx.x & 31) == 0) mbar_arrive(t ? &bars->v_full[s] : &bars->k_full[s]);
    ++g;
  }
  // Tiles [from, to) of the unit.
  template <typename Wait>
  __device__ __forceinline__ void run(const CkUnit& u, int from, int to, Wait&& wait) {
#pragma unroll 1
    for (int j = from; j < min(to, u.j1); ++j) {
      look_up(u, j, page(u, j));
      spread(u, j, wait);
    }
  }
  // The tiles that a unit begins with (see `twin` for those of one row tile).
  template <typename Wait>
  __device__ __forceinline__ void begin(const CkUnit& u, Wait&& wait) {
    run(u, u.j0, u.j0 + (t && u.rows[1] > 0 ? 1 : 2), wait);
  }
};

// Code: the type of 8-bit pages (void: 16-bit pages of type T).
template <typename T, bool kCap, bool kAlibi, bool kNarrow, bool kTree, typename Code>
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

  constexpr bool kCode = !std::is_void_v<Code>;
  [[maybe_unused]] constexpr bool kRun = kCode && kCkRunScale<T>;
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
      mbar_init(&bars->k_full[s], kCode ? 4 : 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], kCode ? 4 : 1);
      mbar_init(&bars->v_empty[s], 1);
      mbar_init(&bars->kc_full[s], 1);
      mbar_init(&bars->vc_full[s], 1);
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
            const int token = u.token + t * (kTree ? u.rows[0] / pb.group : pb.tile_tokens);
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
          if constexpr (kCode) {  // codes into the tile's first half; the softmax warpgroups spread them out
            mbar_arrive_expect_tx(&bars->kc_full[s], kChunkHalf);
            for (int i = 0; i < 2; ++i)
              tma_load_4d(dk + i * kChunkHalf / 2, &tm_k, &bars->kc_full[s], 0, u.hk, 0, ph[i]);
          } else {
            mbar_arrive_expect_tx(&bars->k_full[s], kChunkTileBytes);
            for (int i = 0; i < 2; ++i) {
              tma_load_4d(dk + i * kChunkHalf / 2, &tm_k, &bars->k_full[s], 0, u.hk, 0, ph[i]);
              tma_load_4d(dk + kChunkHalf + i * kChunkHalf / 2, &tm_k, &bars->k_full[s], 64, u.hk, 0,
                          ph[i]);
            }
          }
          if (j == u.j0) load_q();
          if (!ok) break;
          if (g >= kCkStages && !(ok = mbar_wait(&bars->v_empty[s], par, p.err))) break;
          uint8_t* dv = sV + s * kChunkTileBytes;
          if constexpr (kCode) {
            mbar_arrive_expect_tx(&bars->vc_full[s], kChunkHalf);
            for (int i = 0; i < 2; ++i)
              tma_load_4d(dv + i * kChunkHalf / 2, &tm_v, &bars->vc_full[s], 0, u.hk, 0, ph[i]);
          } else {
            mbar_arrive_expect_tx(&bars->v_full[s], kChunkTileBytes);
            for (int i = 0; i < 2; ++i) {
              tma_load_4d(dv + i * kChunkHalf / 2, &tm_v, &bars->v_full[s], 0, u.hk, 0, ph[i]);
              tma_load_4d(dv + kChunkHalf + i * kChunkHalf / 2, &tm_v, &bars->v_full[s], 64, u.hk, 0,
                          ph[i]);
            }
          }
          ph[0] = next[0];
          ph[1] = next[1];
        }
      }
    } else if (warp == 10) {
      CkScheduler sched(pb, p.unit_tokens, kPad, bars, units, p.join + cta, p.err, kTree && !kNarrow);
      while (sched.open) sched.next();
      sched.finish();
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
      auto issue_s = [&](int t, int kstage, int qtile) {
        const uint64_t da = umma_desc_sw128(q_addr + qtile * kChunkTileBytes, 16, 1024);
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
        } else if (kTree && u.rows[1] == 0) {
          // rows for one tile: both warpgroups have it, and alternate key tiles (tile j is that of j & 1)
          ok = mbar_wait(&bars->q_full[0], qc[0] & 1, p.err);
          const int sc0 = sc[0], sc1 = sc[1];
          auto step_s = [&](int j) {
            const int st = (g + j) % kCkStages, t = j & 1;
            if (!(ok = mbar_wait(&bars->k_full[st], ((g + j) / kCkStages) & 1, p.err))) return;
            tc_fence_after();
            issue_s(t, st, 0);
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
            issue_pv(t, st, j < 2);
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
            issue_s(t, g % kCkStages, t);
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
                issue_s(t, (g + 1) % kCkStages, t);
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
    using Spreader =
        std::conditional_t<kCode, CodeSpreader<T, std::conditional_t<kCode, Code, CodeI8>>, int>;
    [[maybe_unused]] auto spreader = [&] {
      if constexpr (kCode) return Spreader(p, bars, sK, sV, t, quarter);
      else return 0;
    }();
    [[maybe_unused]] bool begun = false;  // the next unit's first tiles are spread
    int next_unit = 0;
#pragma unroll 1
    for (const CkUnit* up; (up = ck_next<true>(bars, next_unit, p.err)) != nullptr;
         ck_done<true>(bars, next_unit)) {
      const CkUnit& u = *up;
      // Rows for one tile only: the warpgroups take them both, and alternate key tiles, as two running
      // softmaxes that the first one merges at the end (16 trees of 9 to 33 tokens over 500 to 4000, scores
      // capped: 84 us, with the second one idle 99).
      const bool twin = kTree && !kNarrow && u.rows[1] == 0;
      const int rows = t && !twin ? u.rows[1] : u.rows[0];
      const bool begins = u.j0 == 0, ends = u.j1 == u.n;
      if constexpr (kCode) {
        if (!begun) spreader.begin(u, wait);
      }
      if constexpr (kNarrow) {
        narrow_unit<T, kCap, kAlibi, kTree>(p, bars, u, sQ + kChunkTileBytes, sV, tmem, t, quarter, lane, sc,
                                     g, uc, merges, cta, ok);
      } else {
      if (rows == 0) {
        g += u.j1 - u.j0;
        continue;
      }
      const bool live = row < rows;             // this row is stored
      const bool warp_live = quarter * 32 < rows;
      const int tok = bars->row_token[row], head = u.hk * pb.group + bars->row_head[row];
      // the tile's first token of the unit
      const int tile0 = twin ? 0 : t * (kTree ? u.rows[0] / pb.group : pb.tile_tokens);
      const int first = twin ? u.j0 + t : u.j0, g0 = g - u.j0;
      const int pos = u.pos + tile0 + tok;
      float slope2 = 0.f;
      if (kAlibi && live) slope2 = p.f.slopes[head] * kLog2e;
      float m = -INFINITY, l = 0.f;
      [[maybe_unused]] float mv = -INFINITY;  // m' of ck_reference
#pragma unroll 1
      for (int j = first; j < u.j1; j += twin ? 2 : 1, ++sc) {
        g = g0 + j;
        const int tile = ck_tile(u, j);
        const int k0 = tile * kChunkTile;
        // (keys past the context are masked by their number)
        const bool page0 = u.pages_ok || chunk_page(pb, u.b, u.keys, tile, 0) != pb.num_blocks;
        const bool page1 = u.pages_ok || chunk_page(pb, u.b, u.keys, tile, 1) != pb.num_blocks;
        [[maybe_unused]] const int ahead = j + 2 - t;  // the tile that is spread after this one's weights
        [[maybe_unused]] int ahead_page = pb.num_blocks;
        if constexpr (kCode)
          if (ahead < u.j1) ahead_page = spreader.page(u, ahead);
        wait(&bars->s_full[t], sc & 1);
        if constexpr (kCode)
          if (ahead < u.j1) spreader.look_up(u, ahead, ahead_page);
        if (!kCode && (twin || t == 0) && k0 + kChunkTile > u.keys) {
          wait(&bars->v_full[g % kCkStages], (g / kCkStages) & 1);
          zero_v_rows(sV + (g % kCkStages) * kChunkTileBytes, max(u.keys - k0, 0), threadIdx.x & 127);
          fence_proxy_async_smem();
        }
        if (warp_live) {
          tc_fence_after();
          // columns [c_lo, c_hi) and [0, c_pre) are visible
          int c_hi = min(pos + 1, u.keys) - k0, c_pre = u.prefix - k0;
          int c_lo = pb.window ? pos - pb.window + 1 - k0 : 0;
          int c_tree = kChunkTile;  // columns from here on go by the tree's bits
          if (kTree && pb.tree) {
            c_tree = u.prefix - k0;
            c_hi = min(c_tree, u.keys - k0);
            c_pre = 0;
            if (pb.window && live)
              c_lo = u.prefix + pb.depths[u.token + tile0 + tok] - pb.window + 1 - k0;
          }
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
              if constexpr (kCode) scale_columns<32>(sr, bars->k_scale[g % kCkScaleSlots] + cc);
              score_form<kCap, kAlibi>(sr, p.f, slope2, (float)(k0 + cc - pos), live);
              if (mask) {
                uint32_t vis = (low_bits(c_hi - cc, 0) & ~low_bits(c_lo - cc, 0)) |
                               low_bits(c_pre - cc, 0);
                if (kTree && pb.tree && live && cc + 32 > c_tree)
                  vis |= tree_bits(pb, u.token + tile0 + tok, cc - c_tree) &
                         low_bits(u.keys - k0 - cc, 0);
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
          auto load = [&]() {
            tmem_ld32(tS + 0, sr + 0);
            tmem_ld32(tS + 32, sr + 32);
            tmem_ld32(tS + 64, sr + 64);
            tmem_ld32(tS + 96, sr + 96);
            tmem_wait_ld();
            reg_fence<kChunkTile>(sr);
            if constexpr (kCode) {
              if (!(kCap || mask)) scale_columns<kChunkTile>(sr, bars->k_scale[g % kCkScaleSlots]);
            }
          };
          load();
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
          if (j == first) {
            m = m_new;
          } else {
            const bool need = !(m_new <= m + kCkRescale) && m == m;  // (once to NaN; it stays)
            if constexpr (!kRun) rescale = __any_sync(0xffffffffu, need);
            if (need) {
              alpha = fast_exp2(m - m_new);
              m = m_new;
              l *= alpha;
            }
          }
          [[maybe_unused]] float factor = 0.f;
          if constexpr (kRun) {
            alpha = 1.f;
            const float4 v4 = *reinterpret_cast<const float4*>(bars->v_top[g % kCkScaleSlots]);
            const float bound = mx * sl2 + fmaxf(fmax3f(v4.x, v4.y, v4.z) - kCkRunTop, v4.w - kCkRunTop);
            if (__any_sync(0xffffffffu, live && (bound > mv || m > mv + kCkRunGap + kCkRescale))) {
              const float to = ck_reference(tS, sl2, kCap || mask ? nullptr : bars->k_scale[g % kCkScaleSlots],
                                            bars->v_scale[g % kCkScaleSlots], mv);
              alpha = to == mv ? 1.f : fast_exp2(mv - to);
              mv = to;
              rescale = j != first;
              load();
            }
            factor = mv == -INFINITY ? 0.f : fast_exp2(m - mv);
          }
          l += ck_exp<T, kCode, kRun>(sr, sl2, m == -INFINITY ? 0.f : m, bars->v_scale[g % kCkScaleSlots],
                                      factor);
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
        if constexpr (kCode) {
          if (ahead < u.j1) spreader.spread(u, ahead, wait);
          if (twin) spreader.run(u, ahead + 1, ahead + 2, wait);
        }
      }
      g = g0 + u.j1;
      if constexpr (kCode) {
        const CkUnit* un = ck_next<true>(bars, next_unit + 1, p.err);
        begun = un != nullptr;
        if (begun) spreader.begin(*un, wait);
      }
      // ----------------------------------------------------------- epilogue
      const bool mine = first < u.j1;
      if (mine) wait(&bars->o_full[t], uc & 1);
      tc_fence_after();
      bool none = m == -INFINITY;
      float inv = none ? 0.f : (kRun ? exp2f(mv - m) : 1.f) / l, inv1 = 0.f;
      float lse2 = none ? -INFINITY : m + log2f(l);
      const bool two = twin && u.j1 - u.j0 > 1;  // the second warpgroup has a sum as well
      auto meet = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->merge);
        wait(&bars->merge, merges++ & 1);
      };
      if (two) {
        if (t == 1) {
          bars->n_red[0][quarter][lane] = m;
          bars->n_red[1][quarter][lane] = l;
          if constexpr (kRun) bars->twin_mv[quarter][lane] = mv;
        }
        tc_fence_before();
        meet();
        tc_fence_after();
        if (t == 0) {
          const float m1 = bars->n_red[0][quarter][lane], l1 = bars->n_red[1][quarter][lane];
          const float mx = fmax_nan(m, m1);
          const float w0 = m == -INFINITY ? 0.f : exp2f(m - mx);
          const float w1 = m1 == -INFINITY ? 0.f : exp2f(m1 - mx);
          const float sum = w0 * l + w1 * l1;
          none = mx == -INFINITY;
          inv = none ? 0.f : (kRun ? exp2f(mv - mx) : w0) / sum;
          inv1 = none ? 0.f : (kRun ? exp2f(bars->twin_mv[quarter][lane] - mx) : w1) / sum;
          lse2 = none ? -INFINITY : mx + log2f(sum);
        }
      }
      const int64_t out_row = u.token + tile0 + tok;
      const int64_t part = (int64_t)(cta * 2 + (begins ? 1 : 0)) * p.rows_cap + (twin ? 0 : t * 128) + row;
      T* orow = static_cast<T*>(p.o) + out_row * p.os[0] + head * p.os[1];
      float* prow = p.ws_o + (part & ~31) * 128 + (part & 31) * 4;
      if (warp_live && !(twin && t == 1)) {
#pragma unroll 1
        for (int cc = 0; cc < 128; cc += 32) {
          uint32_t ov[32];
          tmem_ld32(tO + cc, ov);
          tmem_wait_ld();
          reg_fence<32>(ov);
          // (a factor of 0 is nothing seen: the accumulator does not count)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            ov[e] = none || (kTree && inv == 0.f) ? 0u : __float_as_uint(__uint_as_float(ov[e]) * inv);
          if (two) {
            uint32_t o1[32];
            tmem_ld32(tO + 128 + cc, o1);
            tmem_wait_ld();
            reg_fence<32>(o1);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (inv1 != 0.f)
                ov[e] = __float_as_uint(fmaf(__uint_as_float(o1[e]), inv1, __uint_as_float(ov[e])));
          }
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
      if (two) meet();  // (the first has read the second's sums and O)
      __syncwarp();
      if (mine) {
        if (lane == 0) mbar_arrive(&bars->o_empty[t]);
        ++uc;
      }
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
  const int64_t token = jn.token + (t ? jn.rows[0] / p.b.group : 0) + row / p.b.group;
  const int head = jn.hk * p.b.group + row % p.b.group;
  uint4 pk;
  pk.x = Half16<T>::pack(acc[0] * inv, acc[1] * inv);
  pk.y = Half16<T>::pack(acc[2] * inv, acc[3] * inv);
  pk.z = Half16<T>::pack(acc[4] * inv, acc[5] * inv);
  pk.w = Half16<T>::pack(acc[6] * inv, acc[7] * inv);
  *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + token * p.os[0] + head * p.os[1] + col) = pk;
  if (col == 0 && p.lse) p.lse[token * p.b.hq + head] = none ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

template <typename T, bool kCap, bool kAlibi, bool kNarrow, bool kTree, typename Code>
static int launch_main(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                       const ChunkParams& p, cudaStream_t st) {
  constexpr auto kernel = paged_chunk_kernel<T, kCap, kAlibi, kNarrow, kTree, Code>;
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    // the register split must fit what the block is launched with, or setmaxnreg would wait
    cudaFuncAttributes a;
    const cudaError_t e = cudaFuncGetAttributes(&a, kernel);
    if (e != cudaSuccess) return e;
    if (!kNarrow && a.numRegs * kCkThreads < 2 * 128 * kCkRegsSoftmax + 128 * kCkRegsOther)
      return cudaErrorInvalidConfiguration;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCkSmemBytes);
  });
  if (e != cudaSuccess) return cuda_fail(e, "paged attention: kernel set-up");
  e = launch_pdl(kernel, dim3((unsigned)sm_count()), dim3(kCkThreads), kCkSmemBytes, st, tq,
                 tk, tv, p);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "paged attention: launch");
}

template <typename T, bool kNarrow>
static int launch_form(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                       const ChunkParams& p, cudaStream_t st) {
  const bool cap = p.f.cap_log2 > 0.f;
  if (p.b.tree)  // (without a distance bias)
    return cap ? launch_main<T, true, false, kNarrow, true, void>(tq, tk, tv, p, st)
               : launch_main<T, false, false, kNarrow, true, void>(tq, tk, tv, p, st);
  if (cap)
    return p.f.slopes ? launch_main<T, true, true, kNarrow, false, void>(tq, tk, tv, p, st)
                      : launch_main<T, true, false, kNarrow, false, void>(tq, tk, tv, p, st);
  return p.f.slopes ? launch_main<T, false, true, kNarrow, false, void>(tq, tk, tv, p, st)
                    : launch_main<T, false, false, kNarrow, false, void>(tq, tk, tv, p, st);
}

// The wide kernel over 8-bit pages.
template <typename T, typename Code>
static int launch_codes(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                        const ChunkParams& p, cudaStream_t st) {
  return p.f.cap_log2 > 0.f ? launch_main<T, true, false, false, true, Code>(tq, tk, tv, p, st)
                            : launch_main<T, false, false, false, true, Code>(tq, tk, tv, p, st);
}

// The narrow kernel, the wide one or both (whichever `narrow` and `wide` name), and the join. `codes`: the
// type of the pages, or that of q.
template <typename T>
static int launch_chunk(const CUtensorMap& tq_n, const CUtensorMap& tq_w, const CUtensorMap& tk,
                        const CUtensorMap& tv, const ChunkParams* narrow, const ChunkParams* wide,
                        const CodePages& pages, int code_rows, int64_t codes, cudaStream_t st) {
  int r = FI_OK;
  if (codes == FI_DTYPE_I8 || codes == FI_DTYPE_E4M3) {
    const int64_t dtype = std::is_same_v<T, __half> ? FI_DTYPE_F16 : FI_DTYPE_BF16;
    if (narrow) r = launch_narrow_codes(*narrow, pages, dtype, codes, code_rows, st);
    if (r == FI_OK && wide)
      r = codes == FI_DTYPE_I8 ? launch_codes<T, CodeI8>(tq_w, tk, tv, *wide, st)
                               : launch_codes<T, CodeE4M3>(tq_w, tk, tv, *wide, st);
  } else {
    if (narrow) r = launch_form<T, true>(tq_n, tk, tv, *narrow, st);
    if (r == FI_OK && wide) r = launch_form<T, false>(tq_w, tk, tv, *wide, st);
  }
  if (r != FI_OK) return r;
  const ChunkParams& first = wide ? *wide : *narrow;
  const int parts = (first.rows_cap + (narrow && wide ? narrow->rows_cap : 0)) / kCkJoinRows;
  const cudaError_t e =
      launch_pdl(chunk_combine_kernel<T>, dim3((unsigned)sm_count(), (unsigned)parts), dim3(256), 0,
                 st, first, narrow ? *narrow : first);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "paged attention: combine launch");
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

// Workspace of a call: a part for each kernel that it may launch.
static size_t ck_workspace_size(int64_t total_tokens, int64_t num_q_heads, int64_t num_kv_heads) {
  if (total_tokens <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads ||
      num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 64 ||
      total_tokens > (1 << 28))
    return 0;
  const size_t narrow = ck_workspace(nullptr, nullptr, kCkNarrow);
  if (ck_all_narrow(total_tokens, num_q_heads / num_kv_heads)) return narrow;
  return narrow + ck_workspace(nullptr, nullptr, 2 * kChunkTile);
}

// What fi_paged_tree has beside fi_paged_chunk's arguments.
struct ChunkExtra {
  const int32_t* tree;
  const int32_t* depths;
  int64_t words;
  const float* scale[2];
  const int64_t* ss[2];
  int64_t cache_dtype;
};

static int paged_chunk(const char* what, const void* q, const void* k_cache, const void* v_cache,
                       void* o, float* lse, const int32_t* block_table, const int32_t* cu_seqlens,
                       const int32_t* context_lens, const int32_t* prefix_lens,
                       const float* alibi_slopes, int64_t batch, int64_t total_tokens,
                       int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                       int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq,
                       const int64_t* q_strides, const int64_t* kc_strides,
                       const int64_t* vc_strides, const int64_t* o_strides,
                       const int64_t* bt_strides, float sm_scale, float softcap, int64_t window,
                       int64_t dtype, const ChunkExtra& extra, void* workspace,
                       size_t workspace_bytes, int32_t* error_flag, void* stream) {
  clear_error();
  ChunkParams p = {};
  int r = chunk_batch_args(p.b, what, cu_seqlens, context_lens, prefix_lens, block_table, batch,
                           total_tokens, num_q_heads, num_kv_heads, head_dim, num_blocks,
                           block_size, max_blocks_per_seq, bt_strides, window, dtype);
  if (r != FI_OK) return r;
  p.b.tree = extra.tree;
  p.b.depths = extra.depths;
  p.b.words = (int)extra.words;
  r = chunk_score_args(p.f, what, sm_scale, softcap, alibi_slopes);
  if (r != FI_OK) return r;
  if (batch == 0 || total_tokens == 0) return FI_OK;
  if (!q || !k_cache || !v_cache || !o || !block_table || !cu_seqlens || !context_lens ||
      !q_strides || !kc_strides || !vc_strides || !o_strides || !bt_strides)
    return fail(FI_ERR_INVALID_ARG, "%s: null pointer argument", what);
  // Batches of few tokens per sequence (on average at most kCkNarrow rows) are the narrow
  // kernel's alone: a sequence with more tokens is several units there, which read its keys once
  // each (from L2), unless there are many new tokens: 512 of one sequence over 2000 beside 64
  // single ones over 4000 take 238 us there and 219 in both kernels, but the wide one costs 11 us
  // when it has nothing to do. One sequence with more is the wide kernel's. Other batches may hold
  // both.
  const bool codes = extra.cache_dtype != dtype;
  // Over codes a narrow unit has 8 or 16 rows where that is enough for the average sequence, else 32.
  int unit_rows = kCkNarrow;
  if (codes)
    for (int rows = 16; rows >= 8; rows /= 2)
      if (total_tokens <= batch * (rows / p.b.group)) unit_rows = rows;
  const int64_t per_unit = unit_rows / p.b.group;
  const bool use_wide =
      per_unit == 0 || total_tokens > batch * per_unit || total_tokens - batch >= kCkManyNew;
  // Trees of like sizes (the mask's words bound the largest) are the wide kernel's with the few small ones among
  // them, as a second kernel costs some 20 us however little it has to do: 16 trees of 9 to 33 tokens over 500 to 4000, one
  // of few rows, 84 us with both kernels and 58 with one (int8 pages 138 and 115), 16 of 4 and 16 of 40 over 4000, 132
  // and 111 (240 and 262); but 32 single tokens and 8 trees of 80 over 3000, 136 and 158 (237 and 350).
  const bool alike = extra.tree && extra.words * 32 * batch <= 5 * total_tokens;
  const bool use_narrow = per_unit > 0 && (batch > 1 || total_tokens <= per_unit) && !(use_wide && alike);
  const int64_t unit_tokens = use_wide ? 2 * p.b.tile_tokens : per_unit;
  if (batch > kCkMaxBatch ||
      (total_tokens + unit_tokens - 1) / unit_tokens + batch > kCkMaxUnits)
    return fail(FI_ERR_UNSUPPORTED,
                "%s: at most %d sequences and %lld tokens with %d query heads per KV "
                "head; split the batch",
                what, kCkMaxBatch, (long long)((kCkMaxUnits - batch) * unit_tokens), p.b.group);
  if (o_strides[2] != 1 || !aligned16(o) || !stride_ok(total_tokens, o_strides[0]) ||
      !stride_ok(num_q_heads, o_strides[1]))
    return fail(FI_ERR_ALIGNMENT,
                "%s o: needs a 16-byte aligned base, unit innermost stride and other "
                "strides multiple of 8",
                what);
  const size_t need = ck_workspace_size(total_tokens, num_q_heads, num_kv_heads);
  if (!workspace || workspace_bytes < need)
    return fail(FI_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", what,
                workspace ? workspace_bytes : (size_t)0, need);
  if (!aligned16(workspace))
    return fail(FI_ERR_ALIGNMENT, "%s: workspace not 16-byte aligned", what);
  CodePages pages = {};
  if (codes) {
    pages.q = q;
    pages.pool[0] = static_cast<const uint8_t*>(k_cache);
    pages.pool[1] = static_cast<const uint8_t*>(v_cache);
    for (int i = 0; i < 2; ++i) pages.qs[i] = q_strides[i];
    const int64_t sizes[3] = {num_blocks, block_size, num_kv_heads};
    bool ok = q_strides[2] == 1 && aligned16(q) && stride_ok(total_tokens, q_strides[0]) &&
              stride_ok(num_q_heads, q_strides[1]) && aligned16(k_cache) && aligned16(v_cache) &&
              kc_strides[3] == 1 && vc_strides[3] == 1;
    for (int i = 0; i < 3; ++i) {
      pages.st[0][i] = kc_strides[i];
      pages.st[1][i] = vc_strides[i];
      ok = ok && (sizes[i] == 1 || (kc_strides[i] % 16 == 0 && vc_strides[i] % 16 == 0));
    }
    if (!ok)
      return fail(FI_ERR_ALIGNMENT,
                  "%s: q and pages of codes need 16-byte aligned bases, unit innermost strides and other "
                  "strides that are multiples of 16 bytes",
                  what);
  }
  const CUtensorMapDataType type = dtype == FI_DTYPE_F16 ? Half16<__half>::kTmap
                                                         : Half16<__nv_bfloat16>::kTmap;
  ChunkParams n = p;  // the narrow kernel's
  n.b.tile_tokens = per_unit > 0 ? (int)per_unit : 1;
  CUtensorMap tq_n = {}, tq_w = {}, tk = {}, tv = {};
  if (use_narrow && !codes && (r = chunk_q_map(&tq_n, type, q, n.b, q_strides, what)) != FI_OK)
    return r;
  if (use_wide && (r = chunk_q_map(&tq_w, type, q, p.b, q_strides, what)) != FI_OK)
    return r;
  if (codes) {
    if (use_wide && (r = chunk_code_map(&tk, k_cache, p.b, kc_strides, what)) != FI_OK) return r;
    if (use_wide && (r = chunk_code_map(&tv, v_cache, p.b, vc_strides, what)) != FI_OK) return r;
    for (int kv = 0; kv < 2; ++kv) {
      p.scale[kv] = extra.scale[kv];
      for (int i = 0; i < 3; ++i) p.ss[kv][i] = extra.ss[kv][i];
    }
  } else {
    if ((r = chunk_kv_map(&tk, type, k_cache, p.b, kc_strides, what)) != FI_OK) return r;
    if ((r = chunk_kv_map(&tv, type, v_cache, p.b, vc_strides, what)) != FI_OK) return r;
  }
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
  return dtype == FI_DTYPE_F16
             ? launch_chunk<__half>(tq_n, tq_w, tk, tv, np, wp, pages, unit_rows,
                                    extra.cache_dtype, st)
             : launch_chunk<__nv_bfloat16>(tq_n, tq_w, tk, tv, np, wp, pages, unit_rows,
                                           extra.cache_dtype, st);
}

}  // namespace fi

extern "C" size_t fi_paged_chunk_workspace_size(int64_t total_tokens, int64_t num_q_heads,
                                                int64_t num_kv_heads) {
  return fi::ck_workspace_size(total_tokens, num_q_heads, num_kv_heads);
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
  fi::ChunkExtra extra = {};
  extra.cache_dtype = dtype;
  return fi::paged_chunk("fi_paged_chunk", q, k_cache, v_cache, o, lse, block_table, cu_seqlens,
                         context_lens, prefix_lens, alibi_slopes, batch, total_tokens, num_q_heads,
                         num_kv_heads, head_dim, num_blocks, block_size, max_blocks_per_seq,
                         q_strides, kc_strides, vc_strides, o_strides, bt_strides, sm_scale,
                         softcap, window, dtype, extra, workspace, workspace_bytes, error_flag,
                         stream);
}

extern "C" size_t fi_paged_tree_workspace_size(int64_t total_tokens, int64_t num_q_heads,
                                               int64_t num_kv_heads) {
  return fi::ck_workspace_size(total_tokens, num_q_heads, num_kv_heads);
}

extern "C" int fi_paged_tree(const void* q, const void* k_cache, const void* v_cache,
                             const float* k_scale, const float* v_scale, void* o, float* lse,
                             const int32_t* block_table, const int32_t* cu_seqlens,
                             const int32_t* context_lens, const int32_t* tree_mask,
                             const int32_t* depths, int64_t mask_words, int64_t batch,
                             int64_t total_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                             int64_t head_dim, int64_t num_blocks, int64_t block_size,
                             int64_t max_blocks_per_seq, const int64_t* q_strides,
                             const int64_t* kc_strides, const int64_t* vc_strides,
                             const int64_t* ks_strides, const int64_t* vs_strides,
                             const int64_t* o_strides, const int64_t* bt_strides, float sm_scale,
                             float softcap, int64_t window, int64_t dtype, int64_t cache_dtype,
                             void* workspace, size_t workspace_bytes, int32_t* error_flag,
                             void* stream) {
  using namespace fi;
  clear_error();
  const bool codes = cache_dtype == FI_DTYPE_I8 || cache_dtype == FI_DTYPE_E4M3;
  if (!codes && cache_dtype != dtype)
    return fail(FI_ERR_INVALID_ARG, "fi_paged_tree: unknown cache_dtype %lld",
                (long long)cache_dtype);
  if (tree_mask && (mask_words <= 0 || mask_words > (1 << 16)))
    return fail(FI_ERR_INVALID_ARG, "fi_paged_tree: mask_words must be 1 to 65536");
  if (tree_mask && window > 0 && !depths)
    return fail(FI_ERR_INVALID_ARG, "fi_paged_tree: a window over a tree needs depths");
  if (codes && batch > 0 && total_tokens > 0 && (!k_scale || !v_scale || !ks_strides || !vs_strides))
    return fail(FI_ERR_INVALID_ARG, "fi_paged_tree: 8-bit pages need their scales");
  ChunkExtra extra = {};
  extra.tree = tree_mask;
  extra.depths = depths;
  extra.words = mask_words;
  extra.cache_dtype = cache_dtype;
  if (codes) {
    extra.scale[0] = k_scale;
    extra.scale[1] = v_scale;
    extra.ss[0] = ks_strides;
    extra.ss[1] = vs_strides;
  }
  return paged_chunk("fi_paged_tree", q, k_cache, v_cache, o, lse, block_table, cu_seqlens,
                     context_lens, nullptr, nullptr, batch, total_tokens, num_q_heads,
                     num_kv_heads, head_dim, num_blocks, block_size, max_blocks_per_seq, q_strides,
                     kc_strides, vc_strides, o_strides, bt_strides, sm_scale, softcap, window,
                     dtype, extra, workspace, workspace_bytes, error_flag, stream);
}
