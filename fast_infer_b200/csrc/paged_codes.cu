// Attention of few rows per sequence (single tokens, small draft trees) over a paged cache of 8-bit codes.
//
//   s_ij = f((q_i . kc_j) ks_j * scale),  o_i = sum_j p_ij vs_j vc_j / sum_j p_ij,  p_ij = exp(s_ij - m_i)
// (kc, vc codes, ks, vs their rows' scales; the batch and visibility as in chunk_common.cuh).
//
// * Bound by HBM: 264 bytes a key and head. At 6.5 TB/s an SM has 1446 cycles for 128 keys, in which their
//   32768 codes have to become operands. Spreading them to 16-bit tiles in shared memory, as the wide kernel
//   does, would move 96 KB there each way; so here the codes go from shared memory to registers as they are
//   and become fragments of m16n8k16 products (fp16, which holds every code of either type exactly): 16 bytes
//   of a key, and of a value row, are a lane's own, for dims and keys may be permuted alike on both sides of
//   a product. Both products are transposed (S^T = K Q^T, O^T = V^T P^T), so that keys and dims fill the 16
//   rows of a product and the unit's rows its 8 columns: 1, 2 or 4 such groups of rows.
// * A warp is on its own: it takes 16 of a tile's 128 keys, has a ring of stages filled by cp.async ahead of
//   it (across units too), and a running softmax of its own. The warps meet once a unit. Work is cut into equal
//   parts of one line as in paged_chunk.cu, and units that several CTAs hold are joined likewise.
// * Scales stay out of the products: ks multiplies scores in fp32. vs_j cannot multiply codes (fp16) nor
//   P alone (vs may be 1e-6 or 1e30), so P' = p vs 2^(m - m') carries it, with m' a running maximum
//   of s + log2(vs), less 5: a row's greatest P' lies between 2^5 and 2^15, so that what is 2^-19 of it and more keeps all
//   of fp16's bits. But m' is at least m - 126, as 2^(m - m') has to be finite: a row of zeros (vs = 0) that holds all the
//   weight, or subnormal ones, leave P' below, and o below what 16 bits hold. A sum of p in 32 bits goes with m, the sum of P' vc with m'.
// * q of bf16 is brought to fp16 by a power of two per row, exactly but for values 2^-15 and less of
//   the row's greatest (then to 2^-25 of that). P' is rounded to fp16, half a step of 2^-12 to 2^-11.
// * 64 single tokens over 3000 to 9000 cached ones, 24 heads over 8 of codes, 811 MB: 154 us, 5.3 TB/s where a copy
//   reaches 6.5. Issue slots are what is left: 81 million warp instructions, a good part of them the codes' way into
//   fragments. One token over 517: 12.6 us, two launches and one chain of loads.
#include <float.h>

#include <type_traits>

#include "paged_chunk.cuh"
#include "quant8.cuh"

namespace fi {

constexpr int kPcKeys = 16;                     // keys of a tile that a warp takes: 8 warps have one
constexpr int kPcPad = 3;                       // steps that a unit's start and end are worth on the line
constexpr int kPcStageBytes = 2 * kPcKeys * 128 + 2 * kPcKeys * 4;
constexpr float kPcTopP = 256.f, kPcTop = 32768.f;  // p and P' up to which maxima stay as they are
constexpr float kPcRoom = 5.f;                  // log2 of what a row's greatest P' is then
constexpr float kPcGap = 126.f;                 // most that m' lies below m: 2^126 is finite, 2^-126 normal
static_assert(kPcStageBytes % 16 == 0, "16-byte copies");

// With 8 rows a warp has the registers for 16 of them an SM, whose halves take alternate tiles.
template <int kNT>
struct PcShape {
  static constexpr int kWarps = kNT == 1 ? 16 : 8;
  static constexpr int kThreads = kWarps * 32;
};
constexpr int kPcMaxStages = 5;
constexpr int kPcMaxShared = 227 * 1024;

// Then the ring, [warp][stage], and the line: unit_off [batch + 1], work [units + 1].
template <int kNT>
struct PcShared {
  static constexpr int kWarps = PcShape<kNT>::kWarps;
  float part[4][8][128];  // O of 4 warps, 8 rows at a time
  float m[kWarps][8 * kNT], mv[kWarps][8 * kNT], l[kWarps][8 * kNT];
  float inv[8 * kNT];
  uint32_t warp_sums[kWarps];
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A place on the CTA's part of the line, and the unit that it lies in.
struct PcCursor {
  int64_t left;      // steps of the CTA's part from this unit's start here on
  int e, hk, b;      // unit, KV head, sequence
  int t0;            // first token of the unit in its sequence
  ChunkSeq q;
  int lo, n;         // its key tiles: n from lo on
  int j0, j1;        // those of this CTA
  int last_cta;
  bool valid;
};

// Fills in the cursor's unit, whose steps from `at` on are this CTA's; skips units of which it has no key
// tile. `w`: place of the unit's step `at` on the line.
__device__ __forceinline__ void pc_enter(const ChunkParams& p, const uint32_t* unit_off,
                                         const uint32_t* work, uint32_t units,
                                         int64_t total, int active, int64_t end, int64_t& w, int at,
                                         PcCursor& c) {
  while (true) {
    c.valid = w < end;
    if (!c.valid) return;
    if (c.e < (int)unit_off[c.b] || c.e >= (int)unit_off[c.b + 1]) {
      if (c.e == 0) c.b = -1;
      do ++c.b; while ((int)unit_off[c.b + 1] <= c.e);
    }
    c.q = chunk_seq(p.b, c.b);
    const int len = (int)(work[c.e + 1] - work[c.e]);
    const int stop = len - at <= end - w ? len : at + (int)(end - w);
    c.last_cta = stop == len ? (int)blockIdx.x : (int)(((w - at + len) * active - 1) / total);
    const int64_t next = w + stop - at;
    if (stop > kPcPad) {
      c.t0 = (c.e - (int)unit_off[c.b]) * p.unit_tokens;
      int tiles, np;  // (np is 0: there is no prefix)
      ck_tiles(p.b, c.q, c.t0, min(c.t0 + p.unit_tokens, c.q.n), np, c.lo, tiles);
      c.n = len - kPcPad;
      c.j0 = max(at - kPcPad, 0);
      c.j1 = stop - kPcPad;
      w = next;
      return;
    }
    w = next;
    at = 0;
    if (++c.e == (int)units) c.e = 0, ++c.hk;
  }
}
__device__ __forceinline__ void pc_next(const ChunkParams& p, const uint32_t* unit_off,
                                         const uint32_t* work, uint32_t units,
                                        int64_t total, int active, int64_t end, int64_t& w, PcCursor& c) {
  if (++c.e == (int)units) c.e = 0, ++c.hk;
  pc_enter(p, unit_off, work, units, total, active, end, w, 0, c);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

template <typename T, typename Code, bool kCap, int kNT>
__global__ void __launch_bounds__(PcShape<kNT>::kThreads, 1)
    paged_codes_kernel(const ChunkParams p, const CodePages pages) {
  constexpr int kWarps = PcShape<kNT>::kWarps, kThreads = PcShape<kNT>::kThreads;
  constexpr int kTiles = kWarps / 8;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  PcShared<kNT>* s = reinterpret_cast<PcShared<kNT>*>(smem_raw);
  const int stages = pages.stages;
  uint8_t* rings = smem_raw + sizeof(PcShared<kNT>);
  uint32_t* unit_off = reinterpret_cast<uint32_t*>(rings + kWarps * stages * kPcStageBytes);
  uint32_t* work = unit_off + p.b.batch + 1;
  const ChunkBatch& pb = p.b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slice = warp & 7, half = warp >> 3;  // keys of a tile; which tiles
  const int cta = blockIdx.x;

  // the line of work: units of each sequence, then key tiles of each unit, both as sums
  grid_dep_wait();
  grid_dep_launch();
  if (tid == 0) unit_off[0] = work[0] = 0;
#pragma unroll 1
  for (int b = tid; b < pb.batch; b += kThreads) {
    const ChunkSeq q = chunk_seq(pb, b);
    if (q.bad && cta == 0) set_error(p.err, FI_DEVERR_CONTEXT_LEN);
    unit_off[b + 1] = q.n * pb.group <= p.split_rows
                             ? (uint32_t)((q.n + p.unit_tokens - 1) / p.unit_tokens)
                             : 0u;
  }
  __syncthreads();
  block_scan(unit_off, pb.batch, s->warp_sums);
  // cu that is not ascending could name more units than the host counted: those are dropped
  const uint32_t units = min(unit_off[pb.batch], (uint32_t)pages.max_units);
  if (units != unit_off[pb.batch] && tid == 0) set_error(p.err, FI_DEVERR_CONTEXT_LEN);
#pragma unroll 1
  for (int e = tid; e < (int)units; e += kThreads) {
    const int b = last_le(unit_off, pb.batch, (uint32_t)e);
    const ChunkSeq q = chunk_seq(pb, b);
    const int t0 = (e - (int)unit_off[b]) * p.unit_tokens;
    int np, lo, n;
    ck_tiles(pb, q, t0, min(t0 + p.unit_tokens, q.n), np, lo, n);
    work[e + 1] = (uint32_t)(n + kPcPad);
  }
  __syncthreads();
  block_scan(work, (int)units, s->warp_sums);

  const uint32_t per_head = work[units];
  const int64_t total = (int64_t)per_head * pb.hk;
  const int active = (int)(total < (int64_t)gridDim.x ? total : gridDim.x);
  const int64_t begin = cta < active ? total * cta / active : 0;
  const int64_t end = cta < active ? total * (cta + 1) / active : 0;
  PcCursor c = {};
  int64_t w_use = begin, w_load = begin;
  if (begin < end) {
    c.hk = (int)(begin / per_head);
    const uint32_t r = (uint32_t)(begin - (int64_t)c.hk * per_head);
    c.e = last_le(work, (int)units, r);
    c.b = last_le(unit_off, pb.batch, (uint32_t)c.e);
    pc_enter(p, unit_off, work, units, total, active, end, w_use, (int)(r - work[c.e]), c);
    w_load = w_use;
  }
  // Where the loads are: the warp's 16 keys of one tile, K, V and their scales, a lane copying 16 bytes of
  // rows lane / 8 + 4 i. Pieces of 16 bytes are placed so that the reads below meet no bank twice (K by the
  // row's low bit, V by its low three). What a unit fixes is kept as addresses: the copies are a fifth of
  // the instructions as it is.
  PcCursor ld = c;
  const int row0 = lane >> 3, piece = lane & 7;
  const uint8_t *src_k, *src_v;  // of this lane in page 0
  const float* src_s;
  const int32_t* src_page;  // the next tile's block-table entry
  int ld_key, ld_left;      // its first key, tiles left in the unit
  int ld_page;              // its page, looked up one step ahead (and not looked at before)
  const int slot0 = (slice & 3) * kPcKeys;
  const int64_t page_step = (int64_t)2 * kTiles * pb.bts[1];
  auto look_up = [&]() {
    ld_page = ld.valid && ld_key - slot0 < ld.q.keys ? *src_page : -1;
  };
  auto begin_unit = [&]() {  // units of one tile have none for the second half
    while (ld.valid && (ld_left = (ld.j1 - ld.j0 - half + kTiles - 1) / kTiles) <= 0)
      pc_next(p, unit_off, work, units, total, active, end, w_load, ld);
    if (ld.valid) {
      const int tile = ld.lo + ld.j0 + half;
      ld_key = tile * kChunkTile + slice * kPcKeys;
      src_k = pages.pool[0] + (slot0 + row0) * pages.st[0][1] + ld.hk * pages.st[0][2] + piece * 16;
      src_v = pages.pool[1] + (slot0 + row0) * pages.st[1][1] + ld.hk * pages.st[1][2] + piece * 16;
      const int kv = lane >> 4;
      src_s = p.scale[kv] + ld.hk * p.ss[kv][1] + (slot0 + (lane & 15)) * p.ss[kv][2];
      src_page = pb.bt + ld.b * pb.bts[0] + (int64_t)(tile * 2 + (slice >> 2)) * pb.bts[1];
    }
    look_up();
  };
  begin_unit();
  const uint8_t* my_ring = rings + warp * stages * kPcStageBytes;
  const uint32_t ring = smem_u32(my_ring);
  const uint32_t dst_k = ring + row0 * 128 + ((piece ^ ((row0 & 1) << 2)) << 4);
  const uint32_t dst_v = ring + kPcKeys * 128 + row0 * 128;
  const uint32_t even_v = (uint32_t)(piece ^ row0) << 4, odd_v = (uint32_t)(piece ^ (row0 + 4)) << 4;
  const uint32_t dst_s = ring + 2 * kPcKeys * 128 + lane * 4;
  const int64_t step_k = 4 * pages.st[0][1], step_v = 4 * pages.st[1][1];
  uint32_t held_bits = 0;  // of the stages: whether their page exists
  auto load = [&](int stage) {
    if (ld.valid) {
      const uint32_t at = stage * kPcStageBytes;
      const bool held = (uint32_t)ld_page < (uint32_t)pb.num_blocks;
      held_bits = (held_bits & ~(1u << stage)) | ((uint32_t)held << stage);
      const uint8_t *k = src_k, *v = src_v;
      const float* sc = src_s;
      if (held) {
        k += ld_page * pages.st[0][0];
        v += ld_page * pages.st[1][0];
        sc += ld_page * p.ss[lane >> 4][0];
      }
      if (held && ld_key + kPcKeys <= ld.q.keys) {
#pragma unroll
        for (int i = 0; i < 4; ++i, k += step_k) cp_async16(dst_k + at + i * 512, k, true);
#pragma unroll
        for (int i = 0; i < 4; ++i, v += step_v)
          cp_async16(dst_v + at + i * 512 + (i & 1 ? odd_v : even_v), v, true);
        cp_async4(dst_s + at, sc, true);
      } else {  // zeros past the context and where there is no page
        const int n = held ? ld.q.keys - ld_key : 0;
        if (!held && ld_key < ld.q.keys && lane == 0) set_error(p.err, FI_DEVERR_BAD_BLOCK);
#pragma unroll 1
        for (int i = 0; i < 4; ++i, k += step_k, v += step_v) {
          const bool in = row0 + 4 * i < n;
          cp_async16(dst_k + at + i * 512, in ? k : pages.pool[0], in);
          cp_async16(dst_v + at + i * 512 + (i & 1 ? odd_v : even_v), in ? v : pages.pool[1], in);
        }
        const bool in = (lane & 15) < n;
        cp_async4(dst_s + at, in ? sc : p.scale[0], in);
      }
      ld_key += kTiles * kChunkTile;
      src_page += page_step;
      if (--ld_left > 0) {
        look_up();
      } else {
        pc_next(p, unit_off, work, units, total, active, end, w_load, ld);
        begin_unit();
      }
    }
    cp_async_commit();
  };
#pragma unroll 1
  for (int i = 0; i < stages - 1; ++i) load(i);

  CkJoin join = {};
  int stage = 0;
#pragma unroll 1
  for (; c.valid; pc_next(p, unit_off, work, units, total, active, end, w_use, c)) {
    const int tokens = min(c.q.n - c.t0, p.unit_tokens), rows = tokens * pb.group;
    const int token0 = c.q.start + c.t0;
    // Q as fragments: the four dims of step i are those of word i of a lane's 32 codes of a key; this lane's
    // row of group n is 8 n + g
    uint32_t qb[kNT][8][2];
    float rs[kNT][2];  // what the products of rows 8 n + 2 t (+ 1) are multiplied with
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int row = n * 8 + g;
      const bool live = row < rows;
      const int64_t token = token0 + (live ? row / pb.group : 0);
      const int head = c.hk * pb.group + (live ? row % pb.group : 0);
      const T* src = static_cast<const T*>(pages.q) + token * pages.qs[0] + head * pages.qs[1] + t * 16;
      uint4 raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        raw[i] = live ? *reinterpret_cast<const uint4*>(src + (i >> 1) * 64 + (i & 1) * 8)
                      : make_uint4(0, 0, 0, 0);
      float unit = 1.f;
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<T>(x[j]);
            top = fmax3f(top, fabsf(f.x), fabsf(f.y));
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e of the greatest, e in [-125, 125]: its inverse is normal too
        const int e = min(max((int)(__float_as_uint(top) >> 23), 2), 252);
        unit = __uint_as_float((uint32_t)e << 23);
        const float to = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t* x = reinterpret_cast<uint32_t*>(&raw[i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<T>(x[j]);
            x[j] = pack_half2(f.x * to, f.y * to);
          }
        }
      }
      unit *= kCap ? p.f.cap_in : p.f.scale_log2;
#pragma unroll
      for (int h = 0; h < 2; ++h) rs[n][h] = __shfl_sync(0xffffffffu, unit, (2 * t + h) * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // word i: 4 dims, 8 bytes of `raw`
        const uint4& r = raw[i >> 1];
        qb[n][i][0] = i & 1 ? r.z : r.x;
        qb[n][i][1] = i & 1 ? r.w : r.y;
      }
    }
    float o[kNT][8][4], l[kNT][2], mx[kNT][2], mv[kNT][2], neg[kNT][2], fv[kNT][2];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // no score yet: any finite one gives 2^FLT_MAX, past every bound, and so does any weight of V
        l[n][h] = 0.f;
        mx[n][h] = mv[n][h] = -INFINITY;
        neg[n][h] = fv[n][h] = FLT_MAX;
      }
    }
    const int past = c.q.pos0;  // the sequence's first new slot
    int key0 = (c.lo + c.j0 + half) * kChunkTile + slice * kPcKeys;
    const int plain = pb.window ? 0 : min(past, c.q.keys);  // keys before it are seen by every row
#pragma unroll 1
    for (int j = c.j0 + half; j < c.j1; j += kTiles, key0 += kTiles * kChunkTile) {
      if (stages == 2) cp_async_wait<0>();
      else if (stages == 3) cp_async_wait<1>();
      else if (stages == 4) cp_async_wait<2>();
      else cp_async_wait<kPcMaxStages - 2>();
      __syncwarp();  // all lanes' copies are there, and all have left the stage that is filled next
      const bool page_ok = (held_bits >> stage) & 1u;
      const uint8_t* st = my_ring + stage * kPcStageBytes;
      load(stage == 0 ? stages - 1 : stage - 1);
      stage = stage == stages - 1 ? 0 : stage + 1;
      // ------------------------------------------------ scores of keys g, g + 8 and rows 2 t, 2 t + 1
      float sc[kNT][4];
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int at = ((t + 4 * hf) ^ ((g & 1) << 2)) << 4;
        const uint4 ka = *reinterpret_cast<const uint4*>(st + g * 128 + at);
        const uint4 kb = *reinterpret_cast<const uint4*>(st + (g + 8) * 128 + at);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a0, a1, a2, a3;
          Code::decode4(wa[i], a0, a2);
          Code::decode4(wb[i], a1, a3);
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma_16816(sc[n], a0, a1, a2, a3, qb[n][hf * 4 + i][0], qb[n][hf * 4 + i][1]);
        }
      }
      const float* scales = reinterpret_cast<const float*>(st + 2 * kPcKeys * 128);
      const float ks[2] = {scales[g], scales[g + 8]};
      const float vs[2] = {scales[kPcKeys + g], scales[kPcKeys + g + 8]};
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] *= ks[e >> 1] * rs[n][e & 1];
      if constexpr (kCap) {
        float big = 0.f;
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(sc[n][e]));
        const bool small = __all_sync(0xffffffffu, big <= 1.f);
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = sc[n][e];
            sc[n][e] = p.f.cap_log2 * (small || fabsf(x) <= 1.f ? tanh_poly(x) : tanh_any(x));
          }
      }
      // hidden keys: new tokens' (by position, or the tree's bits), those a window leaves behind, those past
      // the context or without a page (whose copies are zeros)
      if (!page_ok || key0 + kPcKeys > plain) {
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = min(n * 8 + 2 * t + h, rows - 1), tok = row / pb.group, token = token0 + tok;
            uint32_t see = page_ok ? low_bits(c.q.keys - key0, 0) : 0u;
            if (pb.tree) {
              uint32_t before = low_bits(past - key0, 0), inner = 0;
              if (pb.window)
                before &= ~low_bits(past + pb.depths[token] - pb.window + 1 - key0, 0);
              if (key0 + kPcKeys > past) inner = tree_bits(pb, token, key0 - past);
              if (key0 < past) inner &= ~low_bits(past - key0, 0);
              see &= before | inner;
            } else {
              const int pos = past + c.t0 + tok;
              see &= low_bits(pos + 1 - key0, 0);
              if (pb.window) see &= ~low_bits(pos - pb.window + 1 - key0, 0);
            }
            if (!((see >> g) & 1u)) sc[n][h] = -INFINITY;
            if (!((see >> (g + 8)) & 1u)) sc[n][2 + h] = -INFINITY;
          }
      }
      // ------------------------------------------------- weights; maxima move where p passes 2^8 or P' 2^15
      uint32_t pb0[kNT], pb1[kNT];
      float ps[kNT][2];
#pragma unroll 1
      for (bool moved = false;; moved = true) {
        float top_p = 0.f, top = 0.f;
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          float w[4], v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = fast_exp2(sc[n][e] + neg[n][e & 1]);
            v[e] = w[e] * vs[e >> 1] * fv[n][e & 1];
          }
          top_p = fmax3f(fmax3f(top_p, w[0], w[1]), w[2], w[3]);
          top = fmax3f(fmax3f(top, v[0], v[1]), v[2], v[3]);
          ps[n][0] = w[0] + w[2];
          ps[n][1] = w[1] + w[3];
          pb0[n] = pack_half2(v[0], v[1]);
          pb1[n] = pack_half2(v[2], v[3]);
        }
        if (moved || __all_sync(0xffffffffu, top_p <= kPcTopP && top <= kPcTop)) break;
        const float lv[2] = {__log2f(vs[0]), __log2f(vs[1])};
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float a = fmaxf(sc[n][h], sc[n][2 + h]);
            float b = fmaxf(sc[n][h] + lv[0], sc[n][2 + h] + lv[1]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
              b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, off));
            }
            a = fmaxf(a, mx[n][h]);
            b = fmax3f(b - kPcRoom, mv[n][h], a - kPcGap);
            const float fl = mx[n][h] == -INFINITY ? 0.f : fast_exp2(mx[n][h] - a);
            const float fo = mv[n][h] == -INFINITY ? 0.f : fast_exp2(mv[n][h] - b);
            mx[n][h] = a;
            mv[n][h] = b;
            neg[n][h] = a == -INFINITY ? FLT_MAX : -a;
            fv[n][h] = b == -INFINITY ? FLT_MAX : fast_exp2(a - b);
            l[n][h] *= fl;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[n][i][h] *= fo;
              o[n][i][2 + h] *= fo;
            }
          }
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        l[n][0] += ps[n][0];
        l[n][1] += ps[n][1];
        pb0[n] = movmatrix_t(pb0[n]);  // rows by keys, as the second product takes P
        pb1[n] = movmatrix_t(pb1[n]);
      }
      // ------------------------------------------------------------ V^T P': dims 16 g + 2 i (+ 1) of step i
      const uint8_t* vrow = st + kPcKeys * 128;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {  // (two of the four words of each row's 16 codes at a time)
        uint2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 2 * t + (i & 1) + (i >> 1) * 8;
          v[i] = *reinterpret_cast<const uint2*>(vrow + row * 128 + ((g ^ (row & 7)) << 4) + hf * 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a = i ? v[0].y : v[0].x, b = i ? v[1].y : v[1].x;
          const uint32_t x = i ? v[2].y : v[2].x, y = i ? v[3].y : v[3].x;
          uint32_t lo[4], hi[4];  // pairs of keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9 for the word's 4 dims
          Code::decode4(__byte_perm(a, b, 0x5140), lo[0], lo[1]);
          Code::decode4(__byte_perm(a, b, 0x7362), lo[2], lo[3]);
          Code::decode4(__byte_perm(x, y, 0x5140), hi[0], hi[1]);
          Code::decode4(__byte_perm(x, y, 0x7362), hi[2], hi[3]);
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int n = 0; n < kNT; ++n)
              mma_16816(o[n][hf * 4 + i * 2 + d], lo[2 * d], lo[2 * d + 1], hi[2 * d], hi[2 * d + 1],
                        pb0[n], pb1[n]);
        }
      }
    }
    // ---------------------------------------------------------------- the warps meet
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], off);
        if (g == 0) {
          const int row = n * 8 + 2 * t + h;
          s->m[warp][row] = mx[n][h];
          s->mv[warp][row] = mv[n][h];
          s->l[warp][row] = l[n][h];
        }
      }
    __syncthreads();
    const bool whole = c.j0 == 0 && c.j1 == c.n;
    const int64_t part0 = (int64_t)(cta * 2 + (c.j0 == 0 ? 1 : 0)) * p.rows_cap;
    if (tid < rows) {  // a thread per row: its sum, and what O is multiplied with
      float a = -INFINITY, b = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        a = fmaxf(a, s->m[w][tid]);
        b = fmaxf(b, s->mv[w][tid]);
      }
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float lw = s->l[w][tid], mw = s->m[w][tid];
        sum += mw == -INFINITY ? lw : lw * exp2f(mw - a);  // (lw is 0 there, or NaN)
      }
      const bool none = sum == 0.f;
      s->inv[tid] = none || b == -INFINITY ? (sum != sum ? sum : 0.f) : exp2f(b - a) / sum;
      const float lse2 = none ? -INFINITY : a + log2f(sum);
      if (whole) {
        const int64_t token = token0 + tid / pb.group;
        if (p.lse) p.lse[token * pb.hq + c.hk * pb.group + tid % pb.group] = lse2 * kLn2;
      } else {
        p.ws_lse[part0 + tid] = lse2;
      }
    }
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      if (n * 8 >= rows) break;
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float b = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) b = fmaxf(b, s->mv[w][n * 8 + 2 * t + h]);
        f[h] = mv[n][h] == -INFINITY ? 0.f : fast_exp2(mv[n][h] - b);
      }
      // a lane has dims [16 g, 16 g + 16) of rows 2 t and 2 t + 1, 4 at a time in an order that spreads the
      // banks; the last 4 warps go first, and the others add theirs
#pragma unroll 1
      for (int turn = 0; turn < kWarps / 4; ++turn) {
        if (warp >> 2 == kWarps / 4 - 1 - turn) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int q4 = i ^ t;
              float x[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                x[e] = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k)  // (a select over the registers: q4 is the lane's own)
                  x[e] = q4 == k ? o[n][2 * k + (e >> 1)][2 * (e & 1) + h] * f[h] : x[e];
              }
              float4* to = reinterpret_cast<float4*>(&s->part[warp & 3][2 * t + h][16 * g + q4 * 4]);
              if (turn > 0) {
                const float4 was = *to;
                x[0] += was.x;
                x[1] += was.y;
                x[2] += was.z;
                x[3] += was.w;
              }
              *to = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
        __syncthreads();
      }
      if (tid < 256) {
        const int row = tid >> 5, col = (tid & 31) * 4, r = n * 8 + row;
        if (r < rows) {
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(&s->part[w][row][col]);
            sum.x += x.x;
            sum.y += x.y;
            sum.z += x.z;
            sum.w += x.w;
          }
          const float f1 = s->inv[r];
          sum.x *= f1;
          sum.y *= f1;
          sum.z *= f1;
          sum.w *= f1;
          if (whole) {
            const int64_t token = token0 + r / pb.group;
            const int head = c.hk * pb.group + r % pb.group;
            uint2 pk;
            pk.x = Half16<T>::pack(sum.x, sum.y);
            pk.y = Half16<T>::pack(sum.z, sum.w);
            *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + token * p.os[0] + head * p.os[1] + col) = pk;
          } else {
            *reinterpret_cast<float4*>(p.ws_o + (part0 + r) * 128 + col) = sum;
          }
        }
      }
      __syncthreads();
    }
    if (!whole && c.j0 == 0) {  // begins here and goes on: it is the last one
      join.valid = 1;
      join.last_cta = c.last_cta;
      join.token = token0;
      join.hk = c.hk;
      join.rows[0] = rows;
    }
  }
  if (tid == 0) p.join[cta] = join;
  cp_async_wait<0>();
}

template <typename T, typename Code, bool kCap, int kNT>
static int launch_one(const ChunkParams& p, CodePages pages, cudaStream_t st) {
  constexpr auto kernel = paged_codes_kernel<T, Code, kCap, kNT>;
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPcMaxShared);
  });
  if (e != cudaSuccess) return cuda_fail(e, "fi_paged_tree: kernel set-up");
  // as many stages as fit beside the line, which is as long as the batch can make it
  const int64_t units = (int64_t)p.b.total / p.unit_tokens + p.b.batch;
  pages.max_units = units < kCkMaxUnits ? (int)units : kCkMaxUnits;
  const size_t fixed = sizeof(PcShared<kNT>) + (size_t)(p.b.batch + 1 + pages.max_units + 1) * 4;
  const size_t stage = (size_t)PcShape<kNT>::kWarps * kPcStageBytes;
  pages.stages = kPcMaxStages;
  while (pages.stages > 2 && fixed + pages.stages * stage > kPcMaxShared) --pages.stages;
  static_assert(sizeof(PcShared<kNT>) + (kCkMaxBatch + kCkMaxUnits + 2) * 4 +
                        2 * PcShape<kNT>::kWarps * kPcStageBytes <=
                    kPcMaxShared,
                "shared memory");
  e = launch_pdl(kernel, dim3((unsigned)sm_count()), dim3(PcShape<kNT>::kThreads),
                 fixed + pages.stages * stage, st, p, pages);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_paged_tree: launch");
}

template <typename T, typename Code, bool kCap>
static int launch_rows(const ChunkParams& p, const CodePages& pages, int rows, cudaStream_t st) {
  return rows <= 8    ? launch_one<T, Code, kCap, 1>(p, pages, st)
         : rows <= 16 ? launch_one<T, Code, kCap, 2>(p, pages, st)
                      : launch_one<T, Code, kCap, 4>(p, pages, st);
}
template <typename T, typename Code>
static int launch_form(const ChunkParams& p, const CodePages& pages, int rows, cudaStream_t st) {
  return p.f.cap_log2 > 0.f ? launch_rows<T, Code, true>(p, pages, rows, st)
                            : launch_rows<T, Code, false>(p, pages, rows, st);
}

int launch_narrow_codes(const ChunkParams& p, const CodePages& pages, int64_t dtype,
                        int64_t cache_dtype, int rows, cudaStream_t st) {
  if (dtype == FI_DTYPE_F16)
    return cache_dtype == FI_DTYPE_I8 ? launch_form<__half, CodeI8>(p, pages, rows, st)
                                      : launch_form<__half, CodeE4M3>(p, pages, rows, st);
  return cache_dtype == FI_DTYPE_I8 ? launch_form<__nv_bfloat16, CodeI8>(p, pages, rows, st)
                                    : launch_form<__nv_bfloat16, CodeE4M3>(p, pages, rows, st);
}

}  // namespace fi
