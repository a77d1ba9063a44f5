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
//   a product. Rows of a unit are the product's 16 (or twice 16) rows.
// * A warp is on its own: it takes 16 of each tile's 128 keys, has a ring of stages filled by cp.async three
//   tiles ahead (across units too), and a running softmax of its own. The 8 warps meet once a unit. Work is cut
//   into equal parts of one line as in paged_chunk.cu, and units that several CTAs hold are joined likewise.
// * Scales stay out of the products: ks multiplies scores in fp32. vs_j cannot multiply codes (fp16) nor
//   P alone (vs may be 1e-6 or 1e30), so P' = p vs 2^(m - m') carries it, with m' a running maximum
//   of s + log2(vs): P' is at most 2^8, and the greatest of a row's is at least one at some key. A sum
//   of p in 32 bits goes with m, the sum of P' vc with m'.
// * q of bf16 is brought to fp16 by a power of two per row, exactly but for values 2^-15 and less of
//   the row's greatest (then to 2^-25 of that). P' is rounded to fp16, half a step of 2^-12 to 2^-11.
#include <float.h>

#include <type_traits>

#include "paged_chunk.cuh"
#include "quant8.cuh"

namespace fi {

constexpr int kPcWarps = 8;
constexpr int kPcThreads = kPcWarps * 32;
constexpr int kPcKeys = kChunkTile / kPcWarps;  // keys of a tile that a warp takes
constexpr int kPcStages = 4;
constexpr int kPcPad = 3;                       // steps that a unit's start and end are worth on the line
constexpr int kPcStageBytes = 2 * kPcKeys * 128 + 2 * kPcKeys * 4;
constexpr float kPcTop = 256.f;                 // p and P' up to which maxima stay as they are

struct PcShared {
  float part[kPcWarps][16][128];  // O of the warps, 16 rows at a time
  uint8_t ring[kPcWarps][kPcStages][kPcStageBytes];
  float m[kPcWarps][kCkNarrow], mv[kPcWarps][kCkNarrow], l[kPcWarps][kCkNarrow];
  float inv[kCkNarrow];
  uint32_t warp_sums[kPcWarps];
  uint32_t unit_off[kCkMaxBatch + 1];
  uint32_t work[kCkMaxUnits + 1];
};
static_assert(sizeof(PcShared) + 16 <= 227 * 1024, "shared memory");
static_assert(kPcStageBytes % 16 == 0, "16-byte copies");

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
  int np, lo, n;     // its key tiles (see ck_tiles)
  int j0, j1;        // those of this CTA
  int last_cta;
  bool valid;
};

__device__ __forceinline__ int pc_tile(const PcCursor& c, int j) {
  return j < c.np ? j : c.lo + (j - c.np);
}

// Fills in the cursor's unit, whose steps from `at` on are this CTA's; skips units of which it has no key
// tile. `w`: place of the unit's step `at` on the line.
__device__ __forceinline__ void pc_enter(const ChunkParams& p, const PcShared* s, uint32_t units,
                                         int64_t total, int active, int64_t end, int64_t& w, int at,
                                         PcCursor& c) {
  while (true) {
    c.valid = w < end;
    if (!c.valid) return;
    if (c.e < (int)s->unit_off[c.b] || c.e >= (int)s->unit_off[c.b + 1]) {
      if (c.e == 0) c.b = -1;
      do ++c.b; while ((int)s->unit_off[c.b + 1] <= c.e);
    }
    c.q = chunk_seq(p.b, c.b);
    const int len = (int)(s->work[c.e + 1] - s->work[c.e]);
    const int stop = len - at <= end - w ? len : at + (int)(end - w);
    c.last_cta = stop == len ? (int)blockIdx.x : (int)(((w - at + len) * active - 1) / total);
    const int64_t next = w + stop - at;
    if (stop > kPcPad) {
      c.t0 = (c.e - (int)s->unit_off[c.b]) * p.unit_tokens;
      int tiles;
      ck_tiles(p.b, c.q, c.t0, min(c.t0 + p.unit_tokens, c.q.n), c.np, c.lo, tiles);
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
__device__ __forceinline__ void pc_next(const ChunkParams& p, const PcShared* s, uint32_t units,
                                        int64_t total, int active, int64_t end, int64_t& w, PcCursor& c) {
  if (++c.e == (int)units) c.e = 0, ++c.hk;
  pc_enter(p, s, units, total, active, end, w, 0, c);
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

template <typename T, typename Code, bool kCap, int kMT>
__global__ void __launch_bounds__(kPcThreads, 1)
    paged_codes_kernel(const ChunkParams p, const CodePages pages) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  PcShared* s = reinterpret_cast<PcShared*>(smem_raw);
  const ChunkBatch& pb = p.b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x;

  // the line of work: units of each sequence, then key tiles of each unit, both as sums
  grid_dep_wait();
  grid_dep_launch();
  if (tid == 0) s->unit_off[0] = s->work[0] = 0;
#pragma unroll 1
  for (int b = tid; b < pb.batch; b += kPcThreads) {
    const ChunkSeq q = chunk_seq(pb, b);
    if (q.bad && cta == 0) set_error(p.err, FI_DEVERR_CONTEXT_LEN);
    s->unit_off[b + 1] = q.n * pb.group <= p.split_rows
                             ? (uint32_t)((q.n + p.unit_tokens - 1) / p.unit_tokens)
                             : 0u;
  }
  __syncthreads();
  block_scan(s->unit_off, pb.batch, s->warp_sums);
  // cu that is not ascending could name more units than the host counted: those are dropped
  const uint32_t units = min(s->unit_off[pb.batch], (uint32_t)kCkMaxUnits);
  if (units != s->unit_off[pb.batch] && tid == 0) set_error(p.err, FI_DEVERR_CONTEXT_LEN);
#pragma unroll 1
  for (int e = tid; e < (int)units; e += kPcThreads) {
    const int b = last_le(s->unit_off, pb.batch, (uint32_t)e);
    const ChunkSeq q = chunk_seq(pb, b);
    const int t0 = (e - (int)s->unit_off[b]) * p.unit_tokens;
    int np, lo, n;
    ck_tiles(pb, q, t0, min(t0 + p.unit_tokens, q.n), np, lo, n);
    s->work[e + 1] = (uint32_t)(n + kPcPad);
  }
  __syncthreads();
  block_scan(s->work, (int)units, s->warp_sums);

  const uint32_t per_head = s->work[units];
  const int64_t total = (int64_t)per_head * pb.hk;
  const int active = (int)(total < (int64_t)gridDim.x ? total : gridDim.x);
  const int64_t begin = cta < active ? total * cta / active : 0;
  const int64_t end = cta < active ? total * (cta + 1) / active : 0;
  PcCursor c = {};
  int64_t w_use = begin, w_load = begin;
  if (begin < end) {
    c.hk = (int)(begin / per_head);
    const uint32_t r = (uint32_t)(begin - (int64_t)c.hk * per_head);
    c.e = last_le(s->work, (int)units, r);
    c.b = last_le(s->unit_off, pb.batch, (uint32_t)c.e);
    pc_enter(p, s, units, total, active, end, w_use, (int)(r - s->work[c.e]), c);
    w_load = w_use;
  }
  PcCursor ld = c;  // where the loads are
  int ld_j = ld.j0;
  // the page of the next load, looked up one step ahead
  auto look_up = [&]() {
    return ld.valid ? chunk_page(pb, ld.b, ld.q.keys, pc_tile(ld, ld_j), warp >> 2) : 0;
  };
  int ld_page = look_up();
  const uint32_t ring = smem_u32(&s->ring[warp][0][0]);
  // 16 keys of K, V and their scales: a lane copies 16 bytes of rows lane / 8 + 4 i. Pieces of 16 bytes are
  // placed so that the reads below meet no bank twice (K by the row's low bit, V by its low three).
  uint32_t held_bits = 0;  // of the stages: whether their page exists
  auto load = [&](int stage) {
    if (ld.valid) {
      const int tile = pc_tile(ld, ld_j), key0 = tile * kChunkTile + warp * kPcKeys;
      const bool held = ld_page != pb.num_blocks;
      if (!held && key0 < ld.q.keys && lane == 0) set_error(p.err, FI_DEVERR_BAD_BLOCK);
      const int slot0 = key0 & (kChunkPage - 1), row0 = lane >> 3, piece = lane & 7;
      const uint32_t dst = ring + stage * kPcStageBytes;
      const int64_t page = held ? ld_page : 0;
      held_bits = (held_bits & ~(1u << stage)) | ((uint32_t)held << stage);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* src = pages.pool[kv] + page * pages.st[kv][0] +
                             (slot0 + row0) * pages.st[kv][1] + ld.hk * pages.st[kv][2] + piece * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = row0 + 4 * i;
          const int to = piece ^ (kv ? row & 7 : (row & 1) << 2);
          cp_async16(dst + kv * kPcKeys * 128 + row * 128 + to * 16, src + 4 * i * pages.st[kv][1],
                     held && key0 + row < ld.q.keys);
        }
      }
      const int kv = lane >> 4, row = lane & 15;
      cp_async4(dst + 2 * kPcKeys * 128 + lane * 4,
                p.scale[kv] + page * p.ss[kv][0] + ld.hk * p.ss[kv][1] + (slot0 + row) * p.ss[kv][2],
                held && key0 + row < ld.q.keys);
      if (++ld_j == ld.j1) {
        pc_next(p, s, units, total, active, end, w_load, ld);
        ld_j = ld.j0;
      }
      ld_page = look_up();
    }
    cp_async_commit();
  };
#pragma unroll 1
  for (int i = 0; i < kPcStages - 1; ++i) load(i);

  CkJoin join = {};
  int step = 0;
#pragma unroll 1
  for (; c.valid; pc_next(p, s, units, total, active, end, w_use, c)) {
    const int tokens = min(c.q.n - c.t0, p.unit_tokens), rows = tokens * pb.group;
    const int token0 = c.q.start + c.t0;
    // Q as fragments: the four dims of step i are those of word i of a lane's 32 codes of a key
    uint32_t qa[kMT][8][4];
    float rs[kMT][2];  // what a row's products are multiplied with
    int tok[kMT][2];   // its token of the unit
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = m * 16 + h * 8 + g;
        const bool live = row < rows;
        tok[m][h] = live ? row / pb.group : 0;
        const int head = c.hk * pb.group + (live ? row % pb.group : 0);
        const T* src = static_cast<const T*>(pages.q) + (int64_t)(token0 + tok[m][h]) * pages.qs[0] +
                       head * pages.qs[1] + t * 16;
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
        rs[m][h] = unit * (kCap ? p.f.cap_in : p.f.scale_log2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // word i: 4 dims, 8 bytes of `raw`
          const uint4& r = raw[i >> 1];
          qa[m][i][h] = i & 1 ? r.z : r.x;
          qa[m][i][2 + h] = i & 1 ? r.w : r.y;
        }
      }
    float o[kMT][16][4], l[kMT][2], mx[kMT][2], mv[kMT][2], neg[kMT][2], fv[kMT][2];
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][i][e] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // no score yet: any finite one gives 2^FLT_MAX, past every bound, and so does any weight of V
        l[m][h] = 0.f;
        mx[m][h] = mv[m][h] = -INFINITY;
        neg[m][h] = fv[m][h] = FLT_MAX;
      }
    }
    const int past = c.q.pos0;  // the sequence's first new slot
#pragma unroll 1
    for (int j = c.j0; j < c.j1; ++j, ++step) {
      cp_async_wait<kPcStages - 2>();
      __syncwarp();  // all lanes' copies are there, and all have left the stage that is filled next
      const bool page_ok = (held_bits >> (step % kPcStages)) & 1u;
      load((step + kPcStages - 1) % kPcStages);
      const uint8_t* st = s->ring[warp][step % kPcStages];
      const int tile = pc_tile(c, j), key0 = tile * kChunkTile + warp * kPcKeys;
      // ------------------------------------------------------------ scores
      float sc[kMT][2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint8_t* krow = st + (n * 8 + g) * 128;
        const uint4 lo = *reinterpret_cast<const uint4*>(krow + ((t ^ ((g & 1) << 2)) << 4));
        const uint4 hi = *reinterpret_cast<const uint4*>(krow + (((t + 4) ^ ((g & 1) << 2)) << 4));
        const uint32_t kw[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[m][n][e] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t b0, b1;
          Code::decode4(kw[i], b0, b1);
#pragma unroll
          for (int m = 0; m < kMT; ++m)
            mma_16816(sc[m][n], qa[m][i][0], qa[m][i][1], qa[m][i][2], qa[m][i][3], b0, b1);
        }
      }
      const float* scales = reinterpret_cast<const float*>(st + 2 * kPcKeys * 128);
      float2 vs[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float2 ks = *reinterpret_cast<const float2*>(scales + n * 8 + 2 * t);
        vs[n] = *reinterpret_cast<const float2*>(scales + kPcKeys + n * 8 + 2 * t);
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[m][n][e] *= (e & 1 ? ks.y : ks.x) * rs[m][e >> 1];
      }
      if constexpr (kCap) {
        float big = 0.f;
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(sc[m][n][e]));
        const bool small = __all_sync(0xffffffffu, big <= 1.f);
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = sc[m][n][e];
              sc[m][n][e] =
                  p.f.cap_log2 * (small || fabsf(x) <= 1.f ? tanh_poly(x) : tanh_any(x));
            }
      }
      // hidden keys: new tokens' (by position, or the tree's bits), those a window leaves behind, those past
      // the context or without a page (whose copies are zeros)
      if (!page_ok || key0 + kPcKeys > min(past, c.q.keys) || pb.window) {
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int token = token0 + tok[m][h];
            uint32_t see = page_ok ? low_bits(c.q.keys - key0, 0) : 0u;
            if (pb.tree) {
              uint32_t before = low_bits(past - key0, 0), inner = 0;
              if (pb.window)
                before &= ~low_bits(past + pb.depths[token] - pb.window + 1 - key0, 0);
              if (key0 + kPcKeys > past) inner = tree_bits(pb, token, key0 - past);
              if (key0 < past) inner &= ~low_bits(past - key0, 0);
              see &= before | inner;
            } else {
              const int pos = past + c.t0 + tok[m][h];
              see &= low_bits(pos + 1 - key0, 0);
              if (pb.window) see &= ~low_bits(pos - pb.window + 1 - key0, 0);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!((see >> (n * 8 + 2 * t + e)) & 1u)) sc[m][n][h * 2 + e] = -INFINITY;
          }
      }
      // -------------------------------------------------- weights; maxima move where one passes 2^8
      uint32_t pa[kMT][4];
      float ps[kMT][2];
#pragma unroll 1
      for (bool moved = false;; moved = true) {
        float top = 0.f;
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          ps[m][0] = ps[m][1] = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float p0 = fast_exp2(sc[m][n][2 * h] + neg[m][h]);
              const float p1 = fast_exp2(sc[m][n][2 * h + 1] + neg[m][h]);
              const float v0 = p0 * vs[n].x * fv[m][h], v1 = p1 * vs[n].y * fv[m][h];
              top = fmax3f(fmax3f(top, p0, p1), v0, v1);
              ps[m][h] += p0 + p1;
              pa[m][n * 2 + h] = pack_half2(v0, v1);
            }
        }
        if (moved || __all_sync(0xffffffffu, top <= kPcTop)) break;
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float a = fmaxf(fmaxf(sc[m][0][2 * h], sc[m][0][2 * h + 1]),
                            fmaxf(sc[m][1][2 * h], sc[m][1][2 * h + 1]));
            float b = fmaxf(fmaxf(sc[m][0][2 * h] + __log2f(vs[0].x), sc[m][0][2 * h + 1] + __log2f(vs[0].y)),
                            fmaxf(sc[m][1][2 * h] + __log2f(vs[1].x), sc[m][1][2 * h + 1] + __log2f(vs[1].y)));
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) {
              a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
              b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, off));
            }
            a = fmaxf(a, mx[m][h]);
            b = fmaxf(b, mv[m][h]);
            const float fl = mx[m][h] == -INFINITY ? 0.f : fast_exp2(mx[m][h] - a);
            const float fo = mv[m][h] == -INFINITY ? 0.f : fast_exp2(mv[m][h] - b);
            mx[m][h] = a;
            mv[m][h] = b;
            neg[m][h] = a == -INFINITY ? FLT_MAX : -a;
            fv[m][h] = b == -INFINITY ? FLT_MAX : fast_exp2(a - b);
            l[m][h] *= fl;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              o[m][i][2 * h] *= fo;
              o[m][i][2 * h + 1] *= fo;
            }
          }
      }
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        l[m][0] += ps[m][0];
        l[m][1] += ps[m][1];
      }
      // ------------------------------------------------------------ P' V
      const uint8_t* vrow = st + kPcKeys * 128;
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // (two of the four words of each row's 16 codes at a time)
        uint2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 2 * t + (i & 1) + (i >> 1) * 8;
          v[i] = *reinterpret_cast<const uint2*>(vrow + row * 128 + ((g ^ (row & 7)) << 4) + half * 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a = i ? v[0].y : v[0].x, b = i ? v[1].y : v[1].x;
          const uint32_t x = i ? v[2].y : v[2].x, y = i ? v[3].y : v[3].x;
          uint32_t b0[4], b1[4];  // of dims 0 .. 3 of this word
          Code::decode4(__byte_perm(a, b, 0x5140), b0[0], b0[1]);
          Code::decode4(__byte_perm(a, b, 0x7362), b0[2], b0[3]);
          Code::decode4(__byte_perm(x, y, 0x5140), b1[0], b1[1]);
          Code::decode4(__byte_perm(x, y, 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int m = 0; m < kMT; ++m)
              mma_16816(o[m][half * 8 + i * 4 + d], pa[m][0], pa[m][1], pa[m][2], pa[m][3], b0[d], b1[d]);
        }
      }
    }
    // ---------------------------------------------------------------- the warps meet
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 1);
        l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 2);
        const int row = m * 16 + h * 8 + g;
        if (t == 0) {
          s->m[warp][row] = mx[m][h];
          s->mv[warp][row] = mv[m][h];
          s->l[warp][row] = l[m][h];
        }
      }
    __syncthreads();
    const bool whole = c.j0 == 0 && c.j1 == c.n;
    const int64_t part0 = (int64_t)(cta * 2 + (c.j0 == 0 ? 1 : 0)) * p.rows_cap;
    if (tid < rows) {  // a thread per row: its sum, and what O is multiplied with
      float a = -INFINITY, b = -INFINITY;
#pragma unroll
      for (int w = 0; w < kPcWarps; ++w) {
        a = fmaxf(a, s->m[w][tid]);
        b = fmaxf(b, s->mv[w][tid]);
      }
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kPcWarps; ++w) {
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
    for (int m = 0; m < kMT; ++m) {
      if (m * 16 >= rows) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = h * 8 + g;
        float b = -INFINITY;
#pragma unroll
        for (int w = 0; w < kPcWarps; ++w) b = fmaxf(b, s->mv[w][m * 16 + row]);
        const float f = mv[m][h] == -INFINITY ? 0.f : fast_exp2(mv[m][h] - b);
        // a lane has dims [32 t, 32 t + 32) of its rows, written in an order that spreads the banks
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int q4 = i ^ (lane & 7);
          float4 x;
          float* xf = reinterpret_cast<float*>(&x);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // (a select over the registers: q4 is the lane's own)
            float pick = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float v = o[m][(k & 3) * 4 + e][2 * h + (k >> 2)];
              pick = q4 == k ? v : pick;
            }
            xf[e] = pick * f;
          }
          *reinterpret_cast<float4*>(&s->part[warp][row][32 * t + q4 * 4]) = x;
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = tid + i * kPcThreads, row = at >> 5, col = (at & 31) * 4, r = m * 16 + row;
        if (r < rows) {
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kPcWarps; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(&s->part[w][row][col]);
            sum.x += x.x;
            sum.y += x.y;
            sum.z += x.z;
            sum.w += x.w;
          }
          const float f = s->inv[r];
          sum.x *= f;
          sum.y *= f;
          sum.z *= f;
          sum.w *= f;
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

template <typename T, typename Code, bool kCap, int kMT>
static int launch_one(const ChunkParams& p, const CodePages& pages, cudaStream_t st) {
  constexpr auto kernel = paged_codes_kernel<T, Code, kCap, kMT>;
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)sizeof(PcShared));
  });
  if (e != cudaSuccess) return cuda_fail(e, "fi_paged_tree: kernel set-up");
  e = launch_pdl(kernel, dim3((unsigned)sm_count()), dim3(kPcThreads), sizeof(PcShared), st, p, pages);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_paged_tree: launch");
}

template <typename T, typename Code>
static int launch_form(const ChunkParams& p, const CodePages& pages, int rows, cudaStream_t st) {
  if (p.f.cap_log2 > 0.f)
    return rows > 16 ? launch_one<T, Code, true, 2>(p, pages, st)
                     : launch_one<T, Code, true, 1>(p, pages, st);
  return rows > 16 ? launch_one<T, Code, false, 2>(p, pages, st)
                   : launch_one<T, Code, false, 1>(p, pages, st);
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
