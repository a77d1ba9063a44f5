// What the kernels over a chunk of new tokens and a paged cache share: the description of
// the batch, which keys a token sees, and the form of a score.
//
// New tokens are packed: sequence b owns rows [cu[b], cu[b+1]), n_b of them; ctx[b] counts
// its cached tokens, the new ones among them, so its i-th new token has position
// p = ctx[b] - n_b + i. Token p sees key j when
//   j < ctx[b]  and  ((j <= p and (window == 0 or j > p - window)) or j < prefix[b]).
// Score: s = f(q.k * scale) - slope_h * |p - j|, f(x) = x or cap * tanh(x / cap).
//
// The query heads of one KV head are packed as rows with their token: row r of a sequence
// is token r / group, head r % group, so one 128-row tile serves the whole group and K and
// V are read once for it.
#pragma once

#include <math.h>

#include "host_common.h"
#include "umma.cuh"

namespace fi {

constexpr int kChunkPage = 64;      // tokens per page
constexpr int kChunkTile = 128;     // rows, keys and dims of a tile
constexpr int kChunkHalf = kChunkTile * 128;     // bytes: 128 rows x 64 values (one swizzle column)
constexpr int kChunkTileBytes = 2 * kChunkHalf;  // bytes: a 128 x 128 tile of 16-bit values
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct ChunkBatch {
  const int32_t* cu;
  const int32_t* ctx;
  const int32_t* prefix;  // may be null
  const int32_t* bt;
  int64_t bts[2];
  int batch, total, window;
  int hq, hk, group;
  int num_blocks, max_blocks;
  int tile_tokens;  // tokens of one 128-row tile: 128 / group
};

struct ScoreForm {
  float scale_log2;         // scale * log2(e)
  float cap_in;             // scale / cap
  float cap_log2;           // cap * log2(e)
  const float* slopes;      // [hq] or null
  // cap * log2(e) * tanh(x * cap_in) = x * (tiny[0] + tiny[1] x^2 + ...) where |x| <= tiny_max
  float tiny_max, tiny[4];
};

// One sequence as the kernels use it. Values read from the device are clamped, so that no
// row, page or key outside the tensors is ever addressed; `bad` says that they had to be.
struct ChunkSeq {
  int start, n;     // packed rows
  int pos0;         // position of its first new token (negative: cached tokens are missing)
  int keys;         // cached tokens that the block table can hold
  int prefix;
  bool bad;
};

__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkBatch& p, int b) {
  ChunkSeq s;
  const int c0 = p.cu[b], c1 = p.cu[b + 1], ctx = p.ctx[b];
  s.start = min(max(c0, 0), p.total);
  const int end = min(max(c1, s.start), p.total);
  s.n = end - s.start;
  const int span = p.max_blocks * kChunkPage;
  s.keys = min(max(ctx, 0), span);
  s.pos0 = max(ctx, -(1 << 29)) - s.n;
  s.prefix = p.prefix ? min(max(p.prefix[b], 0), s.keys) : 0;
  s.bad = s.start != c0 || end != c1 || s.keys != ctx;
  return s;
}

// Physical page of tile half `half` (0 or 1) of key tile `tile`; num_blocks (a coordinate
// outside the pool, which TMA fills with zeros) when the sequence has no such page or the
// table's entry is invalid.
__device__ __forceinline__ int chunk_page(const ChunkBatch& p, int b, int keys, int tile,
                                          int half) {
  const int pg = tile * 2 + half;
  if (pg * kChunkPage >= keys) return p.num_blocks;
  const int ph = p.bt[b * p.bts[0] + (int64_t)pg * p.bts[1]];
  return ph < 0 || ph >= p.num_blocks ? p.num_blocks : ph;
}

// The low n bits of word i of a 128-bit mask.
__device__ __forceinline__ uint32_t low_bits(int n, int i) {
  n -= 32 * i;
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

constexpr float kTanh0 = 0.9999999502f, kTanh1 = -0.3333283915f, kTanh2 = 0.1332520408f,
                kTanh3 = -0.05345702957f, kTanh4 = 0.02028998042f, kTanh5 = -0.006203379104f,
                kTanh6 = 0.001041022634f;
constexpr float kExp1 = 0.6931469440f, kExp2 = 0.2402212024f, kExp3 = 0.0555071309f,
                kExp4 = 0.0096755410f, kExp5 = 0.0013276472f;
// tanh(u) / u on |u| <= 1 as a polynomial in u^2 (minimax on the relative error, fitted
// here by a Remez exchange: 5.0e-8), for a pair.
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t tanh_poly_x2(uint64_t u) {
  const uint64_t z = mul_f32x2(u, u);
#define FI_C2(x) f32x2(x, x)
  uint64_t q = fma_f32x2(FI_C2(kTanh6), z, FI_C2(kTanh5));
  q = fma_f32x2(q, z, FI_C2(kTanh4));
  q = fma_f32x2(q, z, FI_C2(kTanh3));
  q = fma_f32x2(q, z, FI_C2(kTanh2));
  q = fma_f32x2(q, z, FI_C2(kTanh1));
  q = fma_f32x2(q, z, FI_C2(kTanh0));
#undef FI_C2
  return mul_f32x2(q, u);
}
// A capped score in log2 units over the raw product x, for |x| <= tiny_max (|u| <= 1/3, where most
// scores of a cap of 30 or 50 lie): a polynomial in x^2 of degree 3 (fitted likewise: 4.8e-8) with
// scale and cap in its coefficients, half the work of the one above. Multiply by x.
__device__ __forceinline__ uint64_t cap_tiny_x2(const ScoreForm& f, uint64_t x) {
  const uint64_t z = mul_f32x2(x, x);
  uint64_t q = fma_f32x2(f32x2(f.tiny[3], f.tiny[3]), z, f32x2(f.tiny[2], f.tiny[2]));
  q = fma_f32x2(q, z, f32x2(f.tiny[1], f.tiny[1]));
  return fma_f32x2(q, z, f32x2(f.tiny[0], f.tiny[0]));
}
// tanh(u) = 1 - 2 / (1 + e^(2u)) for any u (saturates without overflow); its error is
// absolute (about 1.2e-7), which the polynomial's is not: that one serves small u.
__device__ __forceinline__ float tanh_any(float u) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(u * (2.f * kLog2e))));
  return fmaf(-2.f, r, 1.f);
}

// 2^x for a pair on the FMA pipe, to 2.2e-7 relative (degree 5, fitted here by a Remez exchange
// with the constant term set to 1): x = n + f as in exp2_poly_x2. x <= -127, -inf among
// them, gives exactly 0; so does NaN, for callers that know of it otherwise.
__device__ __forceinline__ uint64_t exp2_poly5_x2(uint64_t x2) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
  float x0, x1;
  f32x2_split(x2, x0, x1);
  const uint64_t x = f32x2(fmaxf(x0, -127.0f), fmaxf(x1, -127.0f));
  const uint64_t t = add_f32x2(x, f32x2(kMagic, kMagic));
  const uint64_t n = add_f32x2(t, f32x2(-kMagic, -kMagic));
  const uint64_t f = fma_f32x2(n, f32x2(-1.0f, -1.0f), x);
  uint64_t q = fma_f32x2(f32x2(kExp5, kExp5), f, f32x2(kExp4, kExp4));
  q = fma_f32x2(q, f, f32x2(kExp3, kExp3));
  q = fma_f32x2(q, f, f32x2(kExp2, kExp2));
  q = fma_f32x2(q, f, f32x2(kExp1, kExp1));
  q = fma_f32x2(q, f, f32x2(1.0f, 1.0f));
  float q0, q1, t0, t1;
  f32x2_split(q, q0, q1);
  f32x2_split(t, t0, t1);
  return f32x2(__uint_as_float(__float_as_uint(q0) + (__float_as_uint(t0) << 23)),
               __uint_as_float(__float_as_uint(q1) + (__float_as_uint(t1) << 23)));
}

// sum + 2^x with the same polynomial for one value: the power of two is a factor, so that NaN stays
// NaN (in the bits of a sum of exponents it would not). x <= -127 adds exactly 0, x >= 127.5
// infinity.
__device__ __forceinline__ float add_exp2_poly5(float sum, float x) {
  constexpr float kMagic = 12582912.0f + 127.0f;  // 1.5 * 2^23, and the exponent's bias
  x = fmin_nan(fmax_nan(x, -127.0f), 128.0f);
  const float t = x + kMagic, f = x - (t - kMagic);
  float q = fmaf(kExp5, f, kExp4);
  q = fmaf(q, f, kExp3);
  q = fmaf(q, f, kExp2);
  q = fmaf(q, f, kExp1);
  q = fmaf(q, f, 1.0f);
  return fmaf(q, __uint_as_float(__float_as_uint(t) << 23), sum);
}
__device__ __forceinline__ float tanh_poly(float u) {  // tanh_poly_x2 for one value
  const float z = u * u;
  float q = fmaf(kTanh6, z, kTanh5);
  q = fmaf(q, z, kTanh4);
  q = fmaf(q, z, kTanh3);
  q = fmaf(q, z, kTanh2);
  q = fmaf(q, z, kTanh1);
  q = fmaf(q, z, kTanh0);
  return q * u;
}

// Inclusive sums of a[1..n] in place (a[0] stays); every thread of the block calls it.
// `warp_sums`: one word per warp. Each thread owns a run of consecutive entries.
template <typename U>
__device__ __forceinline__ void block_scan(U* a, int n, U* warp_sums) {
  const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (n + threads - 1) / threads;
  const int lo = 1 + min(tid * each, n), hi = 1 + min(tid * each + each, n);
  U sum = 0;
#pragma unroll 1
  for (int i = lo; i < hi; ++i) sum += a[i];
  U inc = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const U v = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += v;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  U run = inc - sum;
#pragma unroll 1
  for (int w = 0; w < warp; ++w) run += warp_sums[w];
#pragma unroll 1
  for (int i = lo; i < hi; ++i) {
    run += a[i];
    a[i] = run;
  }
  __syncthreads();
}

// The last i in [0, n) with a[i] <= x (a ascending, a[0] <= x).
template <typename U>
__device__ __forceinline__ int last_le(const U* a, int n, U x) {
  int lo = 0, hi = n;
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Host: fill the parts that both entry points check alike. Returns FI_OK or an error.
int chunk_batch_args(ChunkBatch& p, const char* what, const int32_t* cu, const int32_t* ctx,
                     const int32_t* prefix, const int32_t* bt, int64_t batch, int64_t total,
                     int64_t hq, int64_t hk, int64_t head_dim, int64_t num_blocks,
                     int64_t block_size, int64_t max_blocks, const int64_t* bts, int64_t window,
                     int64_t dtype);
int chunk_score_args(ScoreForm& f, const char* what, float sm_scale, float softcap,
                     const float* slopes);
// 4-D map over packed rows [T, Hq, 128] seen as (d, head of the group, KV head, token): a box
// is 64 values x the group x `tokens` tokens.
int chunk_q_map(CUtensorMap* m, CUtensorMapDataType type, const void* q, const ChunkBatch& p,
                const int64_t* qs, const char* what);
// 4-D map over a page pool [NB, 64, Hkv, 128] as (d, KV head, slot, page): a box is 64 values
// of the 64 slots of a page.
int chunk_kv_map(CUtensorMap* m, CUtensorMapDataType type, const void* kv, const ChunkBatch& p,
                 const int64_t* st, const char* what);

}  // namespace fi
