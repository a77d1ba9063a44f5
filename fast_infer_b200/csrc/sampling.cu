// Sampling of one token per row of logits, with temperature, top-k, top-p and min-p, from a given
// uniform number.
//
// With x the row, M its maximum and w_i = exp((x_i - M) / T), tokens are ordered by x descending, ties by
// index. Top-k keeps the first k, top-p those of them whose mass before them is below p times
// theirs all, min-p those with w >= min_p. All three keep a head of the order, so together they are one
// cut: a value c and how many of the tokens that equal c stay (the lowest indexes). The token is the
// first index whose running sum of kept w passes u times the whole.
//
// * Sums decide between neighbours whose masses lie 1e-6 apart or less, so weights are rounded to units of 2^-45
//   (from fp64: 2^(n/32) from a table times a polynomial) and added as integers: any order gives the same sum, on every run
//   and for every split of the row. Each is off by half a unit at most, so running sums of n tokens and their shares of the
//   whole by n 2^-46 (the whole is 1 at least): 3.7e-9 where 262144 equal small weights all err to one side, some 1e-11 or less for
//   logits that are spread. A token is the one of exact arithmetic but for a boundary that near to u, or to top_p.
// * 16-bit logits are counted by value: a bin for each of the values within 16 octaves (bf16; 8 of fp16) below M, and
//   below 0 as many above the least with a weight; what lies between, near 0, is one bin whose members are weighed one by
//   one. Weights are then worked out once a value, and cuts found by running sums over bins. A CTA, or a cluster of up
//   to 8, takes a row, as many as find room together; counts are held for each part of a slice, so that the part that
//   holds the target is known from them, and only its tokens are weighed, as far as the target. The row is read twice
//   more from L2 rather than held in shared memory, so that two CTAs find room on an SM.
// * 32-bit logits: a cluster holds a row in shared memory, read once. The cut is found by histograms over 512 bins, first
//   of M - x, then of the bits of x within the bin that holds it, until the bin is one value; bins add integers by
//   shared-memory atomics (three 15-bit limbs, so that no sum of a CTA's values overflows 32 bits) and are joined
//   through distributed shared memory. Where top_k leaves few tokens, one CTA gathers and finishes them. 16-bit rows
//   whose cut lies in the bin near 0 come this way too.
// * The last pass adds kept weights in index order, 256 tokens a warp at a time; the 256 that hold
//   the target are looked at again by one warp.
// * 253 rows of 128256: bf16 72 us (65 MB, 10 at a copy's rate), fp16 137, fp32 374. Counting bounds bf16: 13
//   instructions and a shared-memory atomic a token, 44000 cycles of the 98000 of an SM's two rows, then the last pass and the
//   chain of small steps. One row: fp32 with top_k 15.9 us, with top_p alone 48, bf16 19.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "host_common.h"

namespace cg = cooperative_groups;

namespace fi {

constexpr int kSaThreads = 512;
constexpr int kSaWarps = kSaThreads / 32;
constexpr int kSaBins = kSaThreads;     // a bin per thread where bins are joined
constexpr int kSaStep = 256;            // tokens of a cell: of a warp's step
constexpr int kSaRound = kSaWarps * kSaStep;
constexpr int kSaMaxCells = kSaThreads;  // of a CTA: a thread each
constexpr int kSaMaxCluster = 8;
constexpr int kSaRows32 = 8 * kSaRound;  // 32-bit logits that a CTA holds in shared memory at most
constexpr int64_t kSaMaxVocab = (int64_t)kSaMaxCluster * kSaRows32;
constexpr int kSaMaxTokens = (1 << 17) - 8;  // of a CTA, as limbs and cells allow
constexpr int64_t kSaPart = 4 * kSaRound;  // tokens from which on a slice is counted in parts
constexpr int kSaMaxParts = 4, kSaMaxBlocks = 128, kSaMaxOwn = 384;

struct SampleArgs {
  const void* x;
  int64_t stride;
  const float* u;
  const float* temperature;  // these four: null, or one value per row
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature1, top_p1, min_p1;
  int top_k1;
  int32_t* out;
  int vocab, parts, part;  // parts of a CTA's slice, positions of a part
};

template <typename T>
__device__ __forceinline__ float logit(T x);
template <>
__device__ __forceinline__ float logit(float x) { return x; }
template <>
__device__ __forceinline__ float logit(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float logit(__nv_bfloat16 x) { return __bfloat162float(x); }

// Low bits of a key that say nothing, by type.
template <typename T>
struct KeyGrain { static constexpr int kBits = 0; };
template <>
struct KeyGrain<__half> { static constexpr int kBits = 13; };
template <>
struct KeyGrain<__nv_bfloat16> { static constexpr int kBits = 16; };

template <typename T>
struct Bits16;

// A CTA's slice of the row by position, -inf where a position holds no token. 32-bit logits lie in shared memory;
// 16-bit ones, of which most passes need no more than their counts, are read again from L2: positions begin at the
// 16-byte boundary below the row (rows of an odd vocabulary begin anywhere).
template <typename T>
struct Slice {
  const T* p;
  int lo, hi;  // positions with tokens
  int cells;   // cells with tokens
  __device__ __noinline__ static uint4 edge(const T* p, int lo, int hi, int at) {
    uint32_t w[4] = {};
    if constexpr (sizeof(T) == 2) {
      const uint32_t none = Bits16<T>::bits_below(-INFINITY);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = at + i >= lo && at + i < hi;
        w[i >> 1] |= (in ? (uint32_t) reinterpret_cast<const uint16_t*>(p)[at + i] : none) << (i & 1) * 16;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // eight 16-bit values
  __device__ __forceinline__ uint4 raw8(int at) const {
    if (at >= lo && at + 8 <= hi) return *reinterpret_cast<const uint4*>(p + at);
    return edge(p, lo, hi, at);
  }
  // eight values, -0 as 0
  __device__ __forceinline__ void load8(int at, float* x) const {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p + at);
      *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(p + at + 4);
    } else {
      const uint4 raw = raw8(at);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = logit(t[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += 0.f;
  }
};

// Unsigned keys in the order of the floats.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}

// What a pass knows of its row.
struct Row {
  float top;      // M
  float floor_x;  // no weight below it: under half a unit, or x = -inf
  double m, c32;  // M, 32 * log2(e) / T
};

// exp((x - M) / T) in units of 2^-45, for x >= floor_x: 2^(n / 32) times e^r, |r| <= ln 2 / 64, by the
// series to r^6 (its rest is 4e-18).
__device__ __forceinline__ uint64_t weight(const Row& row, const double* tab, float x) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52
  constexpr double kC1 = 0.021660849392498291, kC2 = 2.3459619820224679e-4,
                   kC3 = 1.6938509724371820e-6, kC4 = 9.1725627018246433e-9,
                   kC5 = 3.9737099845494162e-11, kC6 = 1.4345655584131936e-13;
  const double y = ((double)x - row.m) * row.c32;
  const double t = y + kMagic;
  const int n = __double2loint(t);
  const double r = y - (t - kMagic);
  double q = fma(kC6, r, kC5);
  q = fma(q, r, kC4);
  q = fma(q, r, kC3);
  q = fma(q, r, kC2);
  q = fma(q, r, kC1);
  q = fma(q, r, 1.0);
  const double s = q * tab[n & 31];
  const double w = __hiloint2double(__double2hiint(s) + ((n >> 5) << 20), __double2loint(s));
  // 128's last bit is 2^-45
  return (uint64_t)__double_as_longlong(w + 128.0) - (uint64_t)__double_as_longlong(128.0);
}

// 16-bit logits: keys of the raw bits, in the order of the values, both zeros alike.
template <typename T>
struct Bits16 {
  static constexpr int kRegion = 0, kMaxParts = 1;
};
template <>
struct Bits16<__nv_bfloat16> {
  static constexpr int kRegion = 2048;  // 16 octaves
  static constexpr int kMaxParts = 4;
  static constexpr uint32_t kLowest = 0x8000 - 0x7f7f;
  __device__ static __forceinline__ float value(uint32_t k) {
    return __uint_as_float((k >= 0x8000 ? k - 0x8000 : (0x8000 - k) | 0x8000) << 16);
  }
  __device__ static __forceinline__ uint32_t bits_below(float x) {
    return __bfloat16_as_ushort(__float2bfloat16_rd(x));
  }
  __device__ static __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a),
                                         *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
};
template <>
struct Bits16<__half> {
  static constexpr int kRegion = 8192;  // 8 octaves
  static constexpr int kMaxParts = 3;
  static constexpr uint32_t kLowest = 0x8000 - 0x7bff;
  __device__ static __forceinline__ float value(uint32_t k) {
    return __half2float(
        __ushort_as_half((unsigned short)(k >= 0x8000 ? k - 0x8000 : (0x8000 - k) | 0x8000)));
  }
  __device__ static __forceinline__ uint32_t bits_below(float x) {
    return __half_as_ushort(__float2half_rd(x));
  }
  __device__ static __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
};
__device__ __forceinline__ uint32_t keys16(uint32_t pair) {
  uint32_t neg;  // 0xffff in the halves below 0
  asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(neg) : "r"(pair));
  return (pair ^ (neg | 0x80008000u)) + (neg & 0x00010001u);
}

// Bins of one 16-bit value each, descending: n1 from the row's greatest down, a bin for all that lies between (the lump:
// values near 0, of many octaves), n2 further ones of negative values, whose first lies `off2` below the greatest, and
// a bin for what has no weight.
struct Values {
  uint32_t top, lowest;  // keys: M, and of the least value with a weight
  uint32_t n1, off2, n2;
};
template <typename T>
__device__ __forceinline__ Values value_bins(const Row& row) {
  constexpr uint32_t R = Bits16<T>::kRegion;
  Values v;
  v.top = keys16(Bits16<T>::bits_below(row.top)) & 0xffff;
  v.lowest = max(keys16(Bits16<T>::bits_below(row.floor_x)) & 0xffff, Bits16<T>::kLowest);
  const bool positive = v.top >= 0x8000;
  const uint32_t limit = positive ? max(0x8000u, v.lowest) : v.lowest;
  v.n1 = min(v.top - limit + 1, R);
  v.n2 = 0;
  v.off2 = v.top - v.lowest + 1;
  if (positive && v.lowest < 0x8000) {
    const uint32_t top2 = min(v.lowest + R - 3, 0x7fffu);
    v.n2 = top2 - v.lowest + 1;
    v.off2 = v.top - top2;
  }
  return v;
}
// Bins of two values at once, d keys below the greatest: min(d, n1) + max(d, off2 - 1) - (off2 - 1), with d no more than one
// past the last that has a weight. 16-bit halves; none borrows or carries.
__device__ __forceinline__ uint32_t value_bins2(const Values& v, uint32_t pair) {
  const uint32_t edge = (v.off2 - 1) * 0x10001u;
  const uint32_t below = v.top * 0x10001u - keys16(pair);
  const uint32_t d = __vminu2(below, (v.top - v.lowest + 1) * 0x10001u);
  return __vminu2(d, v.n1 * 0x10001u) + (__vmaxu2(d, edge) - edge);
}
// Whether one of eight values (their bins) lies in the lump.
__device__ __forceinline__ bool any_lump(const Values& v, const uint32_t* bins) {
  const uint32_t lump = v.n1 * 0x10001u;
  const uint32_t least = __vminu2(__vminu2(bins[0] ^ lump, bins[1] ^ lump),
                                  __vminu2(bins[2] ^ lump, bins[3] ^ lump));
  return (least & 0xffff) == 0 || least >> 16 == 0;
}
// Greatest and least key of a bin up to the last with a weight.
__device__ __forceinline__ uint32_t bin_high(const Values& v, uint32_t bin) {
  return bin <= v.n1 ? v.top - bin : v.top - v.off2 - (bin - v.n1 - 1);
}
__device__ __forceinline__ uint32_t bin_low(const Values& v, uint32_t bin) {
  return bin == v.n1 ? v.top - v.off2 + 1 : bin_high(v, bin);
}
// Key of a bin of one value; 0 for others.
__device__ __forceinline__ uint32_t bin_key(const Values& v, uint32_t bin) {
  return bin == v.n1 || bin > v.n1 + v.n2 ? 0 : bin_high(v, bin);
}

struct SaPart {  // what a CTA tells the others about its slice
  float top, low;  // greatest logit; least of its threads' greatest ones
  float least;     // least logit above -inf
  int threads;     // threads with a logit above -inf
  int bad;         // NaN or +inf
  int index;       // greedy: first index of the greatest
  int ties;
  int lump_count[kSaMaxParts];                // per part of the slice
  unsigned long long lump_mass[kSaMaxParts];
  uint64_t mass[kSaMaxParts];                 // kept
};
constexpr int kSaList = 1024;  // candidates that one CTA finishes on its own
constexpr int kSaLumps = 4 * kSaMaxCells;  // values of the lump that a part lists
constexpr int kSaListK = 512;  // top_k up to which a list is tried

struct SaShared {
  double tab[32];
  uint64_t step_mass[kSaMaxCells];
  uint64_t scan[2 * kSaWarps];
  SaPart part;
  float w_top[kSaWarps], w_low[kSaWarps], w_least[kSaWarps];
  int w_ties[kSaWarps];
  // the bin that a search chose
  uint64_t above, held;
  int64_t tie_base[kSaMaxParts][2];
  int tie_end, list_n, lump_n[kSaMaxParts];
  uint32_t edge[2];
  int bin;
  uint32_t min_key;
  // of this CTA's share of the blocks of value bins: of all CTAs' tokens, and of each part's
  uint64_t block_mass[kSaMaxBlocks], block_own[kSaMaxOwn];
  uint32_t block_count[kSaMaxBlocks];
};
// Histograms: two of generic bins by turns, or of 16-bit values, one for each part of the slice. Where weights of all
// values fit (bf16) they take the same place afterwards; where not, counts are held two to a word.
template <typename T>
constexpr int kSaValueBins = 2 * Bits16<T>::kRegion;
constexpr int kSaBlock = 128;  // bins that a warp looks at together, four a lane
template <typename T>
constexpr int kSaBlocks = kSaValueBins<T> / kSaBlock;
template <typename T>
constexpr bool kSaTable = kSaValueBins<T> > 0 && kSaValueBins<T> * 8 <= 32768;
template <typename T>
constexpr int kSaValueWords = kSaTable<T> ? kSaValueBins<T> : kSaValueBins<T> / 2;  // of a part's histogram
template <typename T>
__host__ __device__ constexpr int sa_hist_bytes(int parts) {
  return kSaValueBins<T> == 0           ? 2 * kSaBins * 12 + kSaList * 8
         : kSaTable<T> && parts < 2 ? kSaValueBins<T> * 8
                                        : parts * kSaValueWords<T> * 4;
}
static_assert(sa_hist_bytes<__half>(1) >= 2 * kSaBins * 12, "a search's histograms take the values' place");
static_assert(kSaList * 12 <= 2 * kSaBins * 12, "a list's weights and order take the histograms' place");

// Sums over the block's threads before this one, and of all, of N 64-bit values. `warp_sums`: N x kSaWarps.
template <int N>
__device__ __forceinline__ void block_exclusive(const uint64_t* v, uint64_t* warp_sums, uint64_t* before,
                                                uint64_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) inc[i] = v[i];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint64_t o = __shfl_up_sync(0xffffffffu, inc[i], off);
      if (lane >= off) inc[i] += o;
    }
  if (lane == 31)
#pragma unroll
    for (int i = 0; i < N; ++i) warp_sums[i * kSaWarps + warp] = inc[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint64_t w = lane < kSaWarps ? warp_sums[i * kSaWarps + lane] : 0;
#pragma unroll
    for (int off = 1; off < kSaWarps; off <<= 1) {
      const uint64_t o = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += o;
    }
    all[i] = __shfl_sync(0xffffffffu, w, kSaWarps - 1);
    const uint64_t warps = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    before[i] = (warp ? warps : 0) + inc[i] - v[i];
  }
  __syncthreads();
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Sampling from a list of candidates, by one CTA: list[i] = key << 32 | ~index, all of the row's first k among them
// (and whatever ties with the last or lies beside it). Ranks are counted, n^2 / threads comparisons: of the list as it is
// for top-k and top-p, then of the indexes of what stays for the running sum.
__device__ __forceinline__ void sample_list(SaShared* s, const uint64_t* list, uint64_t* weights, int* order,
                                            int n, const Row& row, int64_t k, float top_p,
                                            uint32_t min_key, float u, int32_t* out) {
  constexpr int kEach = kSaList / kSaThreads;
  const int tid = threadIdx.x;
  int rank[kEach];
  uint64_t mine[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = tid + e * kSaThreads;
    rank[e] = 0;
    mine[e] = i < n ? list[i] : 0;
  }
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const uint64_t other = list[j];
#pragma unroll
    for (int e = 0; e < kEach; ++e) rank[e] += other > mine[e];
  }
  // the first k, in order
  const int m = (int)min((int64_t)n, k);
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = tid + e * kSaThreads;
    if (i < n && rank[e] < m) {
      const float x = of_key((uint32_t)(mine[e] >> 32));
      weights[rank[e]] = x >= row.floor_x ? weight(row, s->tab, x) : 0;
    }
  }
  __syncthreads();
  uint64_t w[kEach], sum = 0, before, all;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = tid * kEach + e;
    w[e] = i < m ? weights[i] : 0;
    sum += w[e];
  }
  block_exclusive<1>(&sum, s->scan, &before, &all);
  // how many of them top-p keeps: those before which the mass is below its share
  const double share = top_p < 1.f ? fmax((double)top_p * (double)all, 1.0) : INFINITY;
  int stay = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    stay += tid * kEach + e < m && (double)before < share;
    before += w[e];
  }
  if (tid == 0) s->bin = 0;
  __syncthreads();
  stay = __reduce_add_sync(0xffffffffu, stay);
  if ((tid & 31) == 0 && stay) atomicAdd(&s->bin, stay);
  __syncthreads();
  stay = s->bin;
  __syncthreads();
  // the kept ones by index
  bool in[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = tid + e * kSaThreads;
    in[e] = i < n && rank[e] < stay && (uint32_t)(mine[e] >> 32) >= min_key;
    if (i < n) order[i] = in[e] ? (int)~(uint32_t)mine[e] : INT_MAX;
    rank[e] = 0;
  }
  __syncthreads();
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const int other = order[j];
#pragma unroll
    for (int e = 0; e < kEach; ++e) rank[e] += other < (int)~(uint32_t)mine[e];
  }
  for (int i = tid; i < kSaList; i += kSaThreads) weights[i] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (!in[e]) continue;
    const float x = of_key((uint32_t)(mine[e] >> 32));
    weights[rank[e]] = x >= row.floor_x ? weight(row, s->tab, x) : 0;
  }
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    w[e] = weights[tid * kEach + e];
    sum += w[e];
  }
  block_exclusive<1>(&sum, s->scan, &before, &all);
  const double target = (double)u * (double)all;
  const bool none = !((double)all > target);
  if (tid == 0) s->bin = -1;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (w[e] > 0 && (none ? before + w[e] == all
                          : (double)(before + w[e]) > target &&
                                (before == 0 || !((double)before > target))))
      s->bin = tid * kEach + e;
    before += w[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (in[e] && rank[e] == s->bin) *out = (int32_t)~(uint32_t)mine[e];
}

// A cut: tokens whose key is above `key` stay, and of those that have it the first `ties` by index.
struct Cut {
  uint32_t key;
  int64_t ties;
  bool all_ties;
};

// How many of a group of equal weights w stay when the mass before them is `above`: those before which the
// mass is below the target.
__device__ __forceinline__ int64_t kept_ties(double target, uint64_t above, uint64_t w, int64_t group) {
  int64_t r = (int64_t)ceil((target - (double)above) / (double)w);
  r = max((int64_t)1, min(r, group));
  while (r > 1 && (double)(above + (uint64_t)(r - 1) * w) >= target) --r;
  while (r < group && (double)(above + (uint64_t)r * w) < target) ++r;
  return r;
}

// The bin of a value in a search's first level.
__device__ __forceinline__ int linear_bin(float top, float scale, float x) {
  return min((int)((top - x) * scale), kSaBins - 1);
}

// The cut at which the count of tokens reaches `want` (kMass = false), or the mass that `share` of all from
// lo_key on, less `drop`, asks for. `above` of the result's group: what lies before it.
template <typename T, bool kMass>
__device__ __noinline__ Cut search(cg::cluster_group& cluster, SaShared* s,
                                   uint32_t (*hists)[kSaBins][3], const Slice<T>& x, const Row& row,
                                   uint32_t lo_key, int64_t want, double share, uint64_t drop,
                                   int& level) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = (int)cluster.num_blocks();
  uint32_t hi_key = key_of(row.top);
  const float range = row.top - of_key(lo_key);
  const float scale = range > 0.f && range < FLT_MAX ? (float)(kSaBins - 1) / range : 0.f;
  uint64_t above = 0, held = 0;
  double target = 0.0;
  bool first = true;
  int shift = 0;
#pragma unroll 1
  while (true) {
    uint32_t(*hist)[3] = hists[level & 1];
#pragma unroll 1
    for (int c = warp; c < x.cells; c += kSaWarps) {
      float v[8];
      x.load8(c * kSaStep + lane * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t k = key_of(v[i]);
        if (k < lo_key || k > hi_key || v[i] == -INFINITY) continue;
        const int b = first ? linear_bin(row.top, scale, v[i])
                            : (int)((hi_key >> shift) - (k >> shift));
        if constexpr (kMass) {
          if (v[i] < row.floor_x) continue;
          const uint64_t w = weight(row, s->tab, v[i]);
          const uint32_t l0 = (uint32_t)w & 0x7fff, l1 = (uint32_t)(w >> 15) & 0x7fff,
                         l2 = (uint32_t)(w >> 30);
          if (l0) atomicAdd(&hist[b][0], l0);
          if (l1) atomicAdd(&hist[b][1], l1);
          if (l2) atomicAdd(&hist[b][2], l2);
        } else {
          atomicAdd(&hist[b][0], 1u);
        }
      }
    }
    cluster.sync();
    ++level;
    // every CTA has read the other buffer before it came here
    for (int i = tid; i < kSaBins * 3; i += kSaThreads) (&hists[level & 1][0][0])[i] = 0;
    uint64_t mine = 0;
    for (int r = 0; r < ctas; ++r) {
      const uint32_t* h = cluster.map_shared_rank(&hist[tid][0], r);
      mine += kMass ? (uint64_t)h[0] + ((uint64_t)h[1] << 15) + ((uint64_t)h[2] << 30) : h[0];
    }
    uint64_t all, before;
    block_exclusive<1>(&mine, s->scan, &before, &all);
    before += above;
    if (kMass && first) target = fmax(share * (double)(all - drop), 1.0);
    const bool pick = kMass ? (double)before < target && (double)(before + mine) >= target
                            : before < (uint64_t)want && before + mine >= (uint64_t)want;
    if (tid == 0) s->bin = -1;
    __syncthreads();
    if (pick && mine > 0) {
      s->bin = tid;
      s->above = before;
      s->held = mine;
    }
    __syncthreads();
    const int bin = s->bin;
    if (bin < 0) {  // fewer tokens than wanted: all stay
      return {0u, 0, true};
    }
    above = s->above;
    held = s->held;
    if (first) {
      // the bin's keys, by a 32-way search of each edge: bins fall as keys rise
      if (warp < 2) {
        uint32_t lo = lo_key, hi = hi_key;  // edge 0: least key in the bin; edge 1: greatest
#pragma unroll 1
        while (hi > lo) {
          const uint32_t gap = (hi - lo) / 32 + 1;
          const uint32_t probe = lo + min((uint32_t)lane * gap, hi - lo);
          const int b = linear_bin(row.top, scale, of_key(probe));
          const uint32_t in = __ballot_sync(0xffffffffu, warp == 0 ? b > bin : b >= bin);
          // probes of an edge's near side form a head of the lanes
          const int n = in == 0xffffffffu ? 32 : __ffs((int)~in) - 1;
          if (warp == 0) {  // the least key with b <= bin lies in (probe n-1, probe n]
            const uint32_t new_hi = n < 32 ? lo + min((uint32_t)n * gap, hi - lo) : hi;
            lo = n > 0 ? min(lo + min((uint32_t)(n - 1) * gap, hi - lo) + 1, new_hi) : lo;
            hi = new_hi;
          } else {  // the greatest key with b >= bin lies in [probe n-1, probe n)
            const uint32_t new_lo = n > 0 ? lo + min((uint32_t)(n - 1) * gap, hi - lo) : lo;
            hi = n < 32 ? max(lo + min((uint32_t)n * gap, hi - lo), new_lo + 1) - 1 : hi;
            lo = new_lo;
          }
        }
        if (lane == 0) s->edge[warp] = lo;
      }
      __syncthreads();
      lo_key = s->edge[0];
      hi_key = s->edge[1];
      first = false;
    } else {
      const uint32_t top_bits = (hi_key >> shift) - (uint32_t)bin;
      const uint32_t lo = top_bits << shift, hi = lo + ((1u << shift) - 1);
      lo_key = max(lo_key, lo);
      hi_key = min(hi_key, hi);
    }
    constexpr int grain = KeyGrain<T>::kBits;
    if ((lo_key >> grain) == (hi_key >> grain)) break;
    shift = grain;
    while ((hi_key >> shift) - (lo_key >> shift) >= kSaBins) ++shift;
  }
  // the group's one value: a positive number's key ends in zeros, a negative one's in ones
  constexpr uint32_t low = (1u << KeyGrain<T>::kBits) - 1;
  const uint32_t key = hi_key & 0x80000000u ? hi_key & ~low : hi_key | low;
  Cut cut = {key, 0, false};
  if constexpr (kMass) {
    const uint64_t w = weight(row, s->tab, of_key(key));
    const int64_t group = (int64_t)(held / w);
    cut.ties = kept_ties(target, above, w, group);
    cut.all_ties = cut.ties >= group;
  } else {
    cut.ties = want - (int64_t)above;
    cut.all_ties = cut.ties >= (int64_t)held;
  }
  if (tid == 0) s->held = held;
  __syncthreads();
  return cut;
}

__device__ __forceinline__ Cut tighter(const Cut& a, const Cut& b) {
  if (a.key != b.key) return a.key > b.key ? a : b;
  if (a.all_ties || b.all_ties) return a.all_ties ? b : a;
  return a.ties < b.ties ? a : b;
}

// Lists the row's first `want` tokens, and those beside the last of them, in the first CTA's `list`: all that lie in the bins of
// M - x (of a search's first level) up to the one where the count reaches `want`. Their number; -1 where the list
// is too short for them.
template <typename T>
__device__ __forceinline__ int candidates(cg::cluster_group& cluster, SaShared* s,
                                          uint32_t (*hists)[kSaBins][3], uint64_t* list,
                                          const Slice<T>& x, int base, const Row& row, uint32_t lo_key,
                                          int64_t want, int& level) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = (int)cluster.num_blocks();
  const float range = row.top - of_key(lo_key);
  const float scale = range > 0.f && range < FLT_MAX ? (float)(kSaBins - 1) / range : 0.f;
  uint32_t(*hist)[3] = hists[level & 1];
  const float least = of_key(lo_key);
#pragma unroll 1
  for (int c = warp; c < x.cells; c += kSaWarps) {
    float v[8];
    x.load8(c * kSaStep + lane * 8, v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v[i] >= least) atomicAdd(&hist[linear_bin(row.top, scale, v[i])][0], 1u);
  }
  if (tid == 0) s->bin = -1;
  cluster.sync();
  ++level;
  uint64_t mine = 0, before, all;
  for (int r = 0; r < ctas; ++r) mine += *cluster.map_shared_rank(&hist[tid][0], r);
  block_exclusive<1>(&mine, s->scan, &before, &all);
  if (before < (uint64_t)want && before + mine >= (uint64_t)want) {
    s->bin = tid;
    s->held = before + mine;
  }
  __syncthreads();
  const int bin = s->bin;
  const int n = bin < 0 || s->held > kSaList ? -1 : (int)s->held;
  if (n >= 0) {
    uint64_t* to = cluster.map_shared_rank(list, 0);
    int* count = cluster.map_shared_rank(&s->list_n, 0);
#pragma unroll 1
    for (int c = warp; c < x.cells; c += kSaWarps) {
      const int at = c * kSaStep + lane * 8;
      float v[8];
      x.load8(at, v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i] >= least && linear_bin(row.top, scale, v[i]) <= bin)
          to[atomicAdd(count, 1)] = (uint64_t)key_of(v[i]) << 32 | (uint32_t)~(base + at + i);
    }
  }
  cluster.sync();
  return n;
}

// The counts of four bins of block `block` a lane, in every part of the row in order; four reads of distributed shared memory in
// flight.
template <typename T, typename F>
__device__ __forceinline__ void each_part(cg::cluster_group& cluster, const uint32_t* counts, int parts,
                                          int block, F&& take) {
  const int all = (int)cluster.num_blocks() * parts;
  using Load = std::conditional_t<kSaTable<T>, uint4, uint2>;
  const int at = block * (kSaBlock * kSaValueWords<T> / kSaValueBins<T>) +
                 (threadIdx.x & 31) * (int)(sizeof(Load) / 4);
  int cta = 0, part = 0;
#pragma unroll 1
  for (int r0 = 0; r0 < all; r0 += 4) {
    Load h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (r0 + j >= all) break;
      h[j] = *reinterpret_cast<const Load*>(cluster.map_shared_rank(counts, cta) +
                                            part * kSaValueWords<T> + at);
      if (++part == parts) ++cta, part = 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (r0 + j >= all) break;
      if constexpr (kSaTable<T>) {
        const uint32_t n[4] = {h[j].x, h[j].y, h[j].z, h[j].w};
        take(r0 + j, n);
      } else {
        const uint32_t n[4] = {h[j].x & 0xffff, h[j].x >> 16, h[j].y & 0xffff, h[j].y >> 16};
        take(r0 + j, n);
      }
    }
  }
}

// Four value bins a lane of block `block`: keys (0: of no single value) and weights.
template <typename T>
struct BinQuad {
  uint32_t key[4];
  uint64_t w[4];
  int lump;  // which of them is the lump; -1: none
  __device__ __forceinline__ BinQuad(const Row& row, const double* tab, const Values& v, int block) {
    const uint32_t bin = block * kSaBlock + (threadIdx.x & 31) * 4;
    lump = bin <= v.n1 && v.n1 < bin + 4 ? (int)(v.n1 - bin) : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      key[j] = bin_key(v, bin + j);
      const float x = Bits16<T>::value(key[j]);
      w[j] = key[j] && x >= row.floor_x ? weight(row, tab, x) : 0;
    }
  }
  // tokens that count, of n in each bin, and their mass, `lump_mass` that of those in the lump
  __device__ __forceinline__ uint32_t tokens(const uint32_t* n, int j) const {
    return key[j] || j == lump ? n[j] : 0;
  }
  __device__ __forceinline__ uint64_t mass(const uint32_t* n, int j, uint64_t lump_mass) const {
    return j == lump ? lump_mass : n[j] * w[j];
  }
};

// The first value at which the running count reaches `want`, or the running mass `target`; thread i has the sums of block
// i of the bins, with `before` before them. False: it lies in the lump (or nowhere).
struct ValueCut {
  uint32_t key16;
  uint32_t group;       // tokens that have the value
  uint64_t count, mass; // before it
};
template <typename T, bool kMass>
__device__ __forceinline__ bool value_cross(cg::cluster_group& cluster, SaShared* s,
                                            const uint32_t* counts, int parts, const Row& row,
                                            const Values& v, uint64_t lump_mass, const uint64_t* sums, const uint64_t* before,
                                            uint64_t want, double target, ValueCut& cut) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool here = kMass ? (double)before[1] < target && (double)(before[1] + sums[1]) >= target
                          : before[0] < want && before[0] + sums[0] >= want;
  __syncthreads();
  if (tid == 0) s->bin = -1;
  __syncthreads();
  if (here && sums[0] > 0) {
    s->bin = tid;
    s->above = before[1];
    s->held = before[0];
  }
  __syncthreads();
  const int owner = s->bin;
  if (owner < 0) return false;
  if (warp == 0) {
    const BinQuad<T> q(row, s->tab, v, owner);
    uint32_t n[4] = {};
    each_part<T>(cluster, counts, parts, owner, [&](int, const uint32_t* h) {
#pragma unroll
      for (int j = 0; j < 4; ++j) n[j] += h[j];
    });
    uint64_t c = 0, m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      n[j] = q.tokens(n, j);
      c += n[j];
      m += q.mass(n, j, lump_mass);
    }
    uint64_t ci = c, mi = m;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint64_t oc = __shfl_up_sync(0xffffffffu, ci, off), om = __shfl_up_sync(0xffffffffu, mi, off);
      if (lane >= off) ci += oc, mi += om;
    }
    uint64_t rc = s->held + ci - c, rm = s->above + mi - m;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t nc = rc + n[j], nm = rm + q.mass(n, j, lump_mass);
      if (n[j] > 0 && (kMass ? (double)rm < target && (double)nm >= target : rc < want && nc >= want)) {
        s->edge[0] = q.key[j];
        s->edge[1] = n[j];
        s->held = rc;
        s->above = rm;
      }
      rc = nc;
      rm = nm;
    }
  }
  __syncthreads();
  cut.key16 = s->edge[0];
  cut.group = s->edge[1];
  cut.count = s->held;
  cut.mass = s->above;
  return cut.key16 != 0;
}

template <typename T>
__global__ void __launch_bounds__(kSaThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  SaShared* s = reinterpret_cast<SaShared*>(smem);
  uint32_t* counts = reinterpret_cast<uint32_t*>(smem + (sizeof(SaShared) + 15) / 16 * 16);
  auto hists = reinterpret_cast<uint32_t(*)[kSaBins][3]>(counts);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row_id = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hist_bytes = sa_hist_bytes<T>(a.parts);
  for (int i = tid; i < hist_bytes / 16; i += kSaThreads)
    reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
  if (tid < 32) s->tab[tid] = exp2(tid / 32.0);
  if (tid == 0) s->list_n = 0;
  if (tid < kSaMaxParts) s->lump_n[tid] = s->part.lump_mass[tid] = s->part.mass[tid] = 0;
  grid_dep_wait();
  grid_dep_launch();
  float top = -INFINITY, least = INFINITY;
  bool bad = false;
  const int slice = a.parts * a.part;
  const T* g = static_cast<const T*>(a.x) + row_id * a.stride;
  Slice<T> x;
  int base = rank * slice;  // token at position 0
  if constexpr (sizeof(T) == 4) {
    // into shared memory, 16 bytes at a time from the first aligned token on
    T* to = reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(counts) + hist_bytes);
    g += base;
    const int here = max(0, min(slice, a.vocab - base));
    constexpr int kVec = 16 / (int)sizeof(T);
    const int off = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T));
    const int head = min(here, off == 0 ? 0 : kVec - off), vecs = (here - head) / kVec;
    const uint4* gv = reinterpret_cast<const uint4*>(g + head);
    constexpr int kBatch = 8;
    for (int i0 = tid; i0 < vecs; i0 += kSaThreads * kBatch) {
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * kSaThreads < vecs) v[j] = gv[i0 + j * kSaThreads];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kSaThreads;
        if (i >= vecs) break;
        if (head == 0) {
          *reinterpret_cast<uint4*>(to + i * kVec) = v[j];
        } else {
          const T* t = reinterpret_cast<const T*>(&v[j]);
#pragma unroll
          for (int e = 0; e < kVec; ++e) to[head + i * kVec + e] = t[e];
        }
      }
    }
    for (int i = tid; i < head; i += kSaThreads) to[i] = g[i];
    for (int i = head + vecs * kVec + tid; i < here; i += kSaThreads) to[i] = g[i];
    for (int i = here + tid; i < slice; i += kSaThreads) to[i] = (T)(-INFINITY);
    __syncthreads();
    x = {to, 0, here, (here + kSaStep - 1) / kSaStep};
    // the row's greatest and least logits, and whether one is NaN or +inf
#pragma unroll 1
    for (int c = warp; c < x.cells; c += kSaWarps) {
      float v[8];
      x.load8(c * kSaStep + lane * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bad |= !(v[i] < INFINITY);
        top = fmaxf(top, v[i]);
        least = fminf(least, v[i] == -INFINITY ? INFINITY : v[i]);
      }
    }
  } else {
    // the greatest, NaN if any is
    const int lead = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T));
    x = {g - lead + base, base == 0 ? lead : 0, max(0, min(slice, a.vocab + lead - base)), 0};
    x.cells = (x.hi + kSaStep - 1) / kSaStep;
    base -= lead;
    constexpr int kBatch = 8;
    uint4 m;
    m.x = m.y = m.z = m.w = Bits16<T>::bits_below(-INFINITY) * 0x10001u;
#pragma unroll 1
    for (int c0 = warp; c0 < x.cells; c0 += kSaWarps * kBatch) {
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        v[j] = m;
        if (c0 + j * kSaWarps < x.cells) v[j] = x.raw8((c0 + j * kSaWarps) * kSaStep + lane * 8);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        m.x = Bits16<T>::max2(m.x, v[j].x);
        m.y = Bits16<T>::max2(m.y, v[j].y);
        m.z = Bits16<T>::max2(m.z, v[j].z);
        m.w = Bits16<T>::max2(m.w, v[j].w);
      }
    }
    const uint32_t both = Bits16<T>::max2(Bits16<T>::max2(m.x, m.y), Bits16<T>::max2(m.z, m.w));
    const T* t = reinterpret_cast<const T*>(&both);
    top = fmax_nan(logit(t[0]), logit(t[1])) + 0.f;
    bad = !(top < INFINITY);
    least = -FLT_MAX;  // (a bound is all that the search asks for)
  }
  float low = top > -INFINITY ? top : INFINITY;  // least of the threads' greatest
  const int threads = __syncthreads_count(top > -INFINITY);
  const int any_bad = __syncthreads_or(bad);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, off));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, off));
  }
  if (lane == 0) {
    s->w_top[warp] = top;
    s->w_low[warp] = low;
    s->w_least[warp] = least;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kSaWarps; ++w) {
      top = fmaxf(top, s->w_top[w]);
      low = fminf(low, s->w_low[w]);
      least = fminf(least, s->w_least[w]);
    }
    s->part.top = top;
    s->part.low = low;
    s->part.least = least;
    s->part.threads = threads;
    s->part.bad = any_bad;
  }
  cluster.sync();
  int with = 0, broken = 0;
  top = -INFINITY;
  low = least = INFINITY;
  for (int r = 0; r < ctas; ++r) {
    const SaPart* p = cluster.map_shared_rank(&s->part, r);
    top = fmaxf(top, p->top);
    low = fminf(low, p->low);
    least = fminf(least, p->least);
    with += p->threads;
    broken |= p->bad;
  }

  const float temp = a.temperature ? a.temperature[row_id] : a.temperature1;
  const int64_t k = a.top_k ? a.top_k[row_id] : a.top_k1;
  const float top_p = a.top_p ? a.top_p[row_id] : a.top_p1;
  const float min_p = a.min_p ? a.min_p[row_id] : a.min_p1;
  const float u = a.u[row_id];
  if (broken || top == -INFINITY) {
    if (rank == 0 && tid == 0) a.out[row_id] = -1;
    cluster.sync();  // (no CTA leaves while another may read its shared memory)
    return;
  }
  if (!(temp > 0.f)) {
    // the first of the greatest
    int at = INT_MAX;
#pragma unroll 1
    for (int c = warp; c < x.cells && at == INT_MAX; c += kSaWarps) {
      float v[8];
      x.load8(c * kSaStep + lane * 8, v);
#pragma unroll
      for (int i = 7; i >= 0; --i)
        if (v[i] == top) at = base + c * kSaStep + lane * 8 + i;
      at = __reduce_min_sync(0xffffffffu, at);
    }
    if (lane == 0) s->w_ties[warp] = at;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kSaWarps; ++w) at = min(at, s->w_ties[w]);
      s->part.index = at;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int r = 0; r < ctas; ++r) at = min(at, cluster.map_shared_rank(&s->part, r)->index);
      a.out[row_id] = at;
    }
    cluster.sync();
    return;
  }

  Row row;
  row.top = top;
  row.m = (double)top;
  row.c32 = 46.166241308446829 / (double)temp;  // 32 * log2(e)
  // 2^-46 and less rounds to no unit
  row.floor_x = fmaxf((float)((double)top - 32.3 * (double)temp), -FLT_MAX);
  // what min-p keeps, x - M >= T * log(min_p) (exp(x - M) would round to 1 near M): the least float
  // that passes, found beside its estimate
  Cut cut = {0u, 0, true};
  if (min_p > 0.f) {
    if (warp == 0) {
      const double least_d = (double)temp * log((double)min_p);
      const uint32_t mid = key_of((float)fmax((double)top + least_d, -(double)FLT_MAX));
      const uint32_t probe = min(mid - 16 + lane, key_of(top));
      const bool in = (double)of_key(probe) - row.m >= least_d || probe == key_of(top);
      const uint32_t hit = __ballot_sync(0xffffffffu, in);
      const uint32_t found = __shfl_sync(0xffffffffu, probe, max(__ffs((int)hit) - 1, 0));
      if (lane == 0) s->min_key = hit ? found : key_of(top);
    }
    __syncthreads();
    cut.key = s->min_key;
  }

  bool counted = false;  // whether the values' counts tell the cut and the parts' kept masses
  [[maybe_unused]] Values bins = {};
  if constexpr (sizeof(T) == 2) {
    constexpr int kBlocks = kSaBlocks<T>;
    static_assert(kBlocks % kSaMaxCluster == 0 && kBlocks <= kSaMaxBlocks &&
                  Bits16<T>::kMaxParts * kBlocks <= kSaMaxOwn);
    bins = value_bins<T>(row);
    const uint32_t end_bin = bins.n1 + 1 + bins.n2;  // (an add to one word by all lanes costs 32 of them)
    // values in the lump are listed, and weighed when the part is done
    uint16_t* lump_list = reinterpret_cast<uint16_t*>(s->step_mass);
    auto lump_weight = [&](uint32_t k) {
      const float v = Bits16<T>::value(k);
      return v >= row.floor_x ? weight(row, s->tab, v) : 0;
    };
#pragma unroll 1
    for (int part = 0; part < a.parts; ++part) {
      uint32_t* to = counts + part * kSaValueWords<T>;
      const int end = min((part + 1) * (a.part / kSaStep), x.cells);
      int c = part * (a.part / kSaStep) + warp;
      uint64_t lump_m = 0;
      uint4 next = make_uint4(0, 0, 0, 0);
      if (c < end) next = x.raw8(c * kSaStep + lane * 8);
#pragma unroll 1
      for (; c < end; c += kSaWarps) {
        const uint4 raw = next;
        if (c + kSaWarps < end) next = x.raw8((c + kSaWarps) * kSaStep + lane * 8);
        const uint32_t of[4] = {value_bins2(bins, raw.x), value_bins2(bins, raw.y),
                                value_bins2(bins, raw.z), value_bins2(bins, raw.w)};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t bin = i & 1 ? of[i >> 1] >> 16 : of[i >> 1] & 0xffff;
          if constexpr (kSaTable<T>) atomicAdd(&to[bin], 1u);
          else if (bin < end_bin) atomicAdd(&to[bin >> 1], 1u << (bin & 1) * 16);
        }
        if (any_lump(bins, of)) {
          uint32_t lumps = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if ((i & 1 ? of[i >> 1] >> 16 : of[i >> 1] & 0xffff) == bins.n1) lumps |= 1u << i;
#pragma unroll 1
          for (; lumps; lumps &= lumps - 1) {
            const int i = __ffs((int)lumps) - 1;
            const uint32_t key = keys16(i < 4 ? (i < 2 ? raw.x : raw.y) : (i < 6 ? raw.z : raw.w));
            const uint32_t k = i & 1 ? key >> 16 : key & 0xffff;
            const int at = atomicAdd(&s->lump_n[part], 1);
            if (at < kSaLumps) lump_list[at] = (uint16_t)k;
            else lump_m += lump_weight(k);
          }
        }
      }
      // the lump's weights, a thread each
      __syncthreads();
      const int lump_n = s->lump_n[part];
      if (lump_n > 0) {
        for (int i = tid; i < min(lump_n, kSaLumps); i += kSaThreads) lump_m += lump_weight(lump_list[i]);
        lump_m = warp_sum(lump_m);
        if (lane == 0) atomicAdd(&s->part.lump_mass[part], (unsigned long long)lump_m);
        __syncthreads();
      }
    }
    if (tid < kSaMaxParts) s->part.lump_count[tid] = s->lump_n[tid];
    cluster.sync();
    uint64_t lump_count = 0, lump_mass = 0;
    for (int r = 0; r < ctas; ++r) {
      const SaPart* p = cluster.map_shared_rank(&s->part, r);
      for (int part = 0; part < a.parts; ++part) {
        lump_count += p->lump_count[part];
        lump_mass += p->lump_mass[part];
      }
    }
    // the sums of every block of bins, of all tokens and of each part's: a share of the blocks each
    const int share = kBlocks / ctas;
#pragma unroll 1
    for (int i = warp; i < share; i += kSaWarps) {
      const int block = rank * share + i;
      const BinQuad<T> q(row, s->tab, bins, block);
      uint32_t n = 0;
      uint64_t m = 0;
      each_part<T>(cluster, counts, a.parts, block, [&](int r, const uint32_t* h) {
        uint64_t lump = 0, o = 0;
        if (q.lump >= 0)
          lump = cluster.map_shared_rank(&s->part, r / a.parts)->lump_mass[r % a.parts];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          n += q.tokens(h, j);
          o += q.mass(h, j, lump);
        }
        o = warp_sum(o);
        m += o;
        if (lane == 0) s->block_own[r * share + i] = o;
      });
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) {
        s->block_count[i] = n;
        s->block_mass[i] = m;
      }
    }
    cluster.sync();
    uint64_t sums[2] = {0, 0}, before[2], all[2];
    if (tid < kBlocks) {
      const SaShared* at = cluster.map_shared_rank(s, tid / share);
      sums[0] = at->block_count[tid % share];
      sums[1] = at->block_mass[tid % share];
    }
    block_exclusive<2>(sums, s->scan, before, all);
    counted = true;
    Cut c = {0u, 0, true};
    ValueCut vc;
    if (k > 0 && (uint64_t)k < all[0]) {
      counted = value_cross<T, false>(cluster, s, counts, a.parts, row, bins, lump_mass, sums, before,
                                        (uint64_t)k, 0.0, vc);
      if (counted) {
        const float v = Bits16<T>::value(vc.key16);
        c = {key_of(v), k - (int64_t)vc.count, k - (int64_t)vc.count >= (int64_t)vc.group};
        all[1] = vc.mass + (v >= row.floor_x ? c.ties * weight(row, s->tab, v) : 0);
      }
    }
    if (counted && top_p < 1.f) {
      const double target = fmax((double)top_p * (double)all[1], 1.0);
      counted = value_cross<T, true>(cluster, s, counts, a.parts, row, bins, lump_mass, sums, before, 0,
                                       target, vc);
      if (counted) {
        const float v = Bits16<T>::value(vc.key16);
        const int64_t r = kept_ties(target, vc.mass, weight(row, s->tab, v), vc.group);
        c = tighter(c, {key_of(v), r, r >= (int64_t)vc.group});
      }
    }
    if (counted) {
      c = tighter(cut, c);
      // a cut (of min-p) within the lump is left to the search
      if (lump_count > 0 && c.key > key_of(Bits16<T>::value(bin_low(bins, bins.n1))) &&
          c.key <= key_of(Bits16<T>::value(bin_high(bins, bins.n1))))
        counted = false;
      if (counted) {
        // kept masses of this CTA's parts, a warp each: blocks above the cut, and of the one that holds it the bins
        // above and a share of the ties
        if (warp < a.parts) {
          const int mine = rank * a.parts + warp;
          uint64_t m = 0;
          int cut_block = -1;
          for (int block = lane; block < kBlocks; block += 32) {
            const uint32_t first = block * kSaBlock, end = bins.n1 + 1 + bins.n2;
            if (first >= end) continue;
            const uint32_t last = min(first + (uint32_t)kSaBlock, end) - 1;
            if (key_of(Bits16<T>::value(bin_low(bins, last))) > c.key)
              m += cluster.map_shared_rank(s, block / share)->block_own[mine * share + block % share];
            else if (key_of(Bits16<T>::value(bin_high(bins, first))) >= c.key)
              cut_block = block;
          }
          cut_block = __reduce_max_sync(0xffffffffu, cut_block);
          if (cut_block >= 0) {
            uint32_t ahead[4] = {}, own[4] = {};
            each_part<T>(cluster, counts, a.parts, cut_block, [&](int r, const uint32_t* h) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (r < mine) ahead[j] += h[j];
                if (r == mine) own[j] = h[j];
              }
            });
            const BinQuad<T> q(row, s->tab, bins, cut_block);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (j == q.lump && lump_count > 0 &&
                  c.key <= key_of(Bits16<T>::value(bin_low(bins, bins.n1))))
                m += s->part.lump_mass[warp];
              const uint32_t key = q.key[j] ? key_of(Bits16<T>::value(q.key[j])) : 0;
              if (q.key[j] == 0 || key < c.key) continue;
              int64_t n = own[j];
              if (key == c.key && !c.all_ties) {
                s->tie_base[warp][0] = ahead[j];
                s->tie_base[warp][1] = n;
                n = max((int64_t)0, min(n, c.ties - (int64_t)ahead[j]));
              }
              m += n * q.w[j];
            }
          }
          m = warp_sum(m);
          if (lane == 0) s->part.mass[warp] = m;
        }
        cut = c;
      }
    }
    if (!counted) {  // the histograms' place is taken by the search's
      cluster.sync();
      for (int i = tid; i < 2 * kSaBins * 3; i += kSaThreads) counts[i] = 0;
      __syncthreads();
    }
  }
  if (!counted) {
    int level = 0;
    uint64_t drop = 0;
    if constexpr (sizeof(T) == 4) {
      // few tokens stay: one CTA takes them (128256 fp32, top-k of 50, top-p and min-p: 15.9 us; when this was added 19,
      // and 36 by the search below)
      if (k > 0 && k <= kSaListK && k <= with) {
        uint64_t* list = reinterpret_cast<uint64_t*>(&hists[2][0][0]);
        const int n = candidates<T>(cluster, s, hists, list, x, base, row, key_of(low), k, level);
        if (n >= 0) {
          if (rank == 0)
            sample_list(s, list, reinterpret_cast<uint64_t*>(counts),
                        reinterpret_cast<int*>(counts) + 2 * kSaList, n, row, k, top_p, cut.key, u,
                        a.out + row_id);
          return;
        }
      }
    }
    if (k > 0 && k < a.vocab) {
      // as many threads as `with` have a logit of at least `low`
      const float from = k <= with ? low : least;
      const Cut c = search<T, false>(cluster, s, hists, x, row, key_of(from), k, 0.0, 0, level);
      if (c.key != 0 && !c.all_ties) {
        const float value = of_key(c.key);
        if (value >= row.floor_x) drop = (s->held - (uint64_t)c.ties) * weight(row, s->tab, value);
      }
      __syncthreads();
      const Cut before = cut;
      cut = c;
      if (top_p < 1.f) {
        const Cut p = search<T, true>(cluster, s, hists, x, row, max(c.key, key_of(row.floor_x)), 0, (double)top_p, drop, level);
        cut = tighter(cut, p);
      }
      cut = tighter(before, cut);
    } else if (top_p < 1.f) {
      const Cut p = search<T, true>(cluster, s, hists, x, row, max(key_of(least), key_of(row.floor_x)), 0, (double)top_p, 0, level);
      cut = tighter(cut, p);
    }
  }

  // Which ties stay: those at positions below tie_end. Where that lies within the cells from `first` to `end`, their
  // ties are counted cell by cell.
  int first = 0, end = x.cells;
  auto tie_counts = [&]() {  // of this thread's cell
#pragma unroll 1
    for (int c = first + warp; c < end; c += kSaWarps) {
      float v[8];
      x.load8(c * kSaStep + lane * 8, v);
      int n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) n += key_of(v[i]) == cut.key;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) s->step_mass[c] = (uint64_t)n;
    }
    __syncthreads();
    return first + tid < end ? s->step_mass[first + tid] : 0;
  };
  auto find_tie_end = [&](int64_t keep, uint64_t in_cell) {  // place of tie number `keep` of them
    uint64_t before, all;
    block_exclusive<1>(&in_cell, s->scan, &before, &all);
    if (in_cell > 0 && (int64_t)before <= keep && keep < (int64_t)(before + in_cell)) {
      s->bin = first + tid;
      s->above = before;
    }
    __syncthreads();
    const int cell = s->bin;
    if (warp == 0) {
      float v[8];
      x.load8(cell * kSaStep + lane * 8, v);
      int n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) n += key_of(v[i]) == cut.key;
      int inc = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += o;
      }
      int64_t at = (int64_t)s->above + inc - n;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (key_of(v[i]) == cut.key && at++ == keep) s->tie_end = cell * kSaStep + lane * 8 + i;
    }
    __syncthreads();
    return s->tie_end;
  };
  int tie_end = INT_MAX;
  if (!cut.all_ties && !counted) {
    const uint64_t in_cell = tie_counts();
    uint64_t before, all;
    block_exclusive<1>(&in_cell, s->scan, &before, &all);
    if (tid == 0) s->part.ties = (int)all;
    cluster.sync();
    int64_t ties_before = 0;
    for (int r = 0; r < rank; ++r) ties_before += cluster.map_shared_rank(&s->part, r)->ties;
    const int64_t keep = cut.ties - ties_before;
    if (keep < (int64_t)all) tie_end = keep > 0 ? find_tie_end(keep, in_cell) : 0;
  }
  // kept weights of the 8 tokens at `at`
  auto kept = [&](int at, uint64_t* w) {
    uint64_t sum = 0;
    float v[8];
    x.load8(at, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t key = key_of(v[i]);
      const bool in = v[i] >= row.floor_x && (key > cut.key || (key == cut.key && at + i < tie_end));
      w[i] = in ? weight(row, s->tab, v[i]) : 0;
      sum += w[i];
    }
    return sum;
  };
  uint64_t cell = 0, before = 0, all = 0;  // a thread's cell
  if (!counted) {
#pragma unroll 1
    for (int c = warp; c < end; c += kSaWarps) {
      uint64_t w[8];
      const uint64_t sum = warp_sum(kept(c * kSaStep + lane * 8, w));
      if (lane == 0) s->step_mass[c] = sum;
    }
    __syncthreads();
    cell = tid < end ? s->step_mass[tid] : 0;
    block_exclusive<1>(&cell, s->scan, &before, &all);
    if (tid == 0) s->part.mass[0] = all;
  }
  if (tid == 0) s->bin = -1;
  cluster.sync();
  // the first part, cell and token whose running sum passes the target; the last kept one where none
  // does (u = 1, NaN). A lane per part.
  uint64_t own = 0;
  if (lane < ctas * a.parts) own = cluster.map_shared_rank(&s->part, lane / a.parts)->mass[lane % a.parts];
  cluster.barrier_arrive();  // (this CTA has read; from here on it is on its own)
  uint64_t ahead = own;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t o = __shfl_up_sync(0xffffffffu, ahead, off);
    if (lane >= off) ahead += o;
  }
  const uint64_t mass = __shfl_sync(0xffffffffu, ahead, 31);
  const double target = (double)u * (double)mass;
  const bool none = !((double)mass > target);
  auto passes = [&](uint64_t sum_before, uint64_t part) {
    return (double)(sum_before + part) > target && (sum_before == 0 || !((double)sum_before > target));
  };
  const uint32_t in_part =
      __ballot_sync(0xffffffffu, own > 0 && (none ? ahead == mass : passes(ahead - own, own)));
  const int part = __ffs((int)in_part) - 1;
  if (part < 0 || part / a.parts != rank) {
    cluster.barrier_wait();
    return;
  }
  ahead = __shfl_sync(0xffffffffu, ahead - own, part);
  own = __shfl_sync(0xffffffffu, own, part);
  int found = -1;         // the cell
  uint64_t above = 0;     // kept mass before it
  uint64_t w[8], sum;     // of this lane's tokens in it
  if (counted) {
    first = part % a.parts * (a.part / kSaStep);
    end = min(first + a.part / kSaStep, x.cells);
    if (!cut.all_ties) {
      const int64_t keep = cut.ties - s->tie_base[part % a.parts][0];
      if (keep < s->tie_base[part % a.parts][1]) tie_end = keep > 0 ? find_tie_end(keep, tie_counts()) : 0;
    }
    [[maybe_unused]] uint32_t tie_bin = 0xffffffffu;  // of the cut, where only some of its tokens stay
    if constexpr (kSaTable<T>) {  // the values' kept weights, over their counts
      if (tie_end != INT_MAX)
        tie_bin = value_bins2(bins, Bits16<T>::bits_below(of_key(cut.key)) * 0x10001u) & 0xffff;
      __syncthreads();
      for (int bin = tid; bin < kSaValueBins<T>; bin += kSaThreads) {
        const uint32_t key16 = bin_key(bins, bin);
        const float v = Bits16<T>::value(key16);
        reinterpret_cast<uint64_t*>(counts)[bin] =
            key16 != 0 && v >= row.floor_x && key_of(v) >= cut.key ? weight(row, s->tab, v) : 0;
      }
      __syncthreads();
    }
    auto kept_by_value = [&](int at, uint64_t* w) {
      if constexpr (!kSaTable<T>) {
        return kept(at, w);
      } else {
        const uint64_t* table = reinterpret_cast<const uint64_t*>(counts);
        const uint4 raw = x.raw8(at);
        const uint32_t of[4] = {value_bins2(bins, raw.x), value_bins2(bins, raw.y),
                                value_bins2(bins, raw.z), value_bins2(bins, raw.w)};
        if (any_lump(bins, of)) return kept(at, w);
        uint64_t sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t bin = i & 1 ? of[i >> 1] >> 16 : of[i >> 1] & 0xffff;
          w[i] = table[bin];
          if (bin == tie_bin && at + i >= tie_end) w[i] = 0;
          sum += w[i];
        }
        return sum;
      }
    };
    // 256 tokens a warp in index order, as far as the target
    uint64_t run = ahead;
#pragma unroll 1
    for (int cell0 = first; found < 0 && cell0 < end; cell0 += kSaWarps) {
      sum = 0;
      if (cell0 + warp < end) sum = kept_by_value((cell0 + warp) * kSaStep + lane * 8, w);
      const uint64_t mass_here = warp_sum(sum);
      if (lane == 0) s->step_mass[cell0 + warp] = mass_here;
      __syncthreads();
      const uint64_t cell = lane < kSaWarps ? s->step_mass[cell0 + lane] : 0;
      uint64_t to = cell;
#pragma unroll
      for (int off = 1; off < kSaWarps; off <<= 1) {
        const uint64_t o = __shfl_up_sync(0xffffffffu, to, off);
        if (lane >= off) to += o;
      }
      const bool here = cell > 0 && (none ? run + to == ahead + own : passes(run + to - cell, cell));
      const uint32_t hit = __ballot_sync(0xffffffffu, here);
      if (hit) {
        const int which = __ffs((int)hit) - 1;
        found = cell0 + which;
        above = __shfl_sync(0xffffffffu, run + to - cell, which);
      }
      run += __shfl_sync(0xffffffffu, to, kSaWarps - 1);
    }
    if (warp != (found - first) % kSaWarps) found = -1;
  } else {
    if (cell > 0 && (none ? before + cell == all : passes(ahead + before, cell))) {
      s->bin = tid;
      s->above = ahead + before;
    }
    __syncthreads();
    above = s->above;
    if (s->bin >= 0 && warp == s->bin % kSaWarps) {
      found = s->bin;
      sum = kept(found * kSaStep + lane * 8, w);
    }
  }
  cluster.barrier_wait();
  if (found < 0) return;
  const int at0 = found * kSaStep + lane * 8;
  uint64_t inc = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  uint64_t run = above + inc - sum;
  int at = none ? -1 : INT_MAX;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    run += w[i];
    if (w[i] > 0) {
      if (none) at = max(at, base + at0 + i);
      else if ((double)run > target) at = min(at, base + at0 + i);
    }
  }
  at = none ? __reduce_max_sync(0xffffffffu, at) : __reduce_min_sync(0xffffffffu, at);
  if (lane == 0) a.out[row_id] = at;
}

template <typename T>
static int launch_sample(const SampleArgs& a, int64_t rows, int ctas, cudaStream_t st) {
  const size_t shared = (sizeof(SaShared) + 15) / 16 * 16;
  constexpr int kHeld = sizeof(T) == 4 ? 4 : 0;  // bytes of a token in shared memory
  const size_t smem = shared + sa_hist_bytes<T>(a.parts) + (size_t)a.part * kHeld;
  static DeviceOnce once;
  cudaError_t e = once.run([&] {
    return cudaFuncSetAttribute(
        sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
        (int)shared + sa_hist_bytes<T>(Bits16<T>::kMaxParts) + kSaRows32 * kHeld);
  });
  if (e != cudaSuccess) return cuda_fail(e, "fi_sample_tokens: kernel set-up");
  e = launch_pdl_cluster(sample_kernel<T>, dim3((unsigned)(rows * ctas)), dim3(kSaThreads), smem, st,
                         (unsigned)ctas, a);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_sample_tokens launch");
}

}  // namespace fi

extern "C" int fi_sample_tokens(const void* logits, const float* u, const float* temperature,
                                const int32_t* top_k, const float* top_p, const float* min_p,
                                float temperature_scalar, int64_t top_k_scalar, float top_p_scalar,
                                float min_p_scalar, int32_t* out, int64_t rows, int64_t vocab,
                                int64_t row_stride, int64_t dtype, void* stream) {
  using namespace fi;
  clear_error();
  if (rows < 0 || vocab <= 0) return fail(FI_ERR_INVALID_ARG, "fi_sample_tokens: bad sizes");
  if (dtype != FI_DTYPE_F16 && dtype != FI_DTYPE_BF16 && dtype != FI_DTYPE_F32)
    return fail(FI_ERR_INVALID_ARG, "fi_sample_tokens: unknown dtype %lld", (long long)dtype);
  if (vocab > kSaMaxVocab || rows > (1 << 24))
    return fail(FI_ERR_UNSUPPORTED, "fi_sample_tokens: at most %lld tokens a row and %d rows",
                (long long)kSaMaxVocab, 1 << 24);
  if (rows == 0) return FI_OK;
  if (!logits || !u || !out)
    return fail(FI_ERR_INVALID_ARG, "fi_sample_tokens: null pointer argument");
  const int size = dtype == FI_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size != 0)
    return fail(FI_ERR_ALIGNMENT, "fi_sample_tokens: logits not aligned to their type");
  // As many CTAs a row as find room at the same time, two an SM, and as its tokens need. 32-bit logits: 16384 tokens each
  // (two CTAs an SM), but 32768 rather than eight CTAs (253 rows of 128256: four 374 us, eight 567; 64 rows 120 and 176; of
  // 32000, 1000 rows: two 261, one 293). 16-bit ones (253 rows of 128256 bf16: 72 us, with
  // two CTAs a row 90; 64 rows: four 37, eight 61) count their slice in parts (253 rows: in one 119 us).
  int ctas = 1, parts = 1;
  int64_t part = 0;
  const int64_t room = 2 * sm_count();
  auto split = [&] {
    if (dtype != FI_DTYPE_F32) {
      parts = (int)((vocab + ctas * kSaPart - 1) / (ctas * kSaPart));
      parts = std::min(parts, dtype == FI_DTYPE_BF16 ? Bits16<__nv_bfloat16>::kMaxParts
                                                     : Bits16<__half>::kMaxParts);
    }
    const int64_t each = (vocab + (size == 2 ? 7 : 0) + ctas * parts - 1) / (ctas * parts);
    part = (each + kSaRound - 1) / kSaRound * kSaRound;
  };
  split();
  while (ctas < kSaMaxCluster) {
    const int64_t most = size == 4 ? kSaRows32 / (ctas < 4 ? 2 : 1) : kSaMaxTokens;
    const bool needs = (parts * part < vocab ? parts * part : vocab) > most;
    const bool wants = (int64_t)ctas * kSaRound < vocab && rows * ctas * 2 <= room;
    if (!needs && !wants) break;
    ctas *= 2;
    split();
  }
  SampleArgs a = {};
  a.x = logits;
  a.stride = row_stride;
  a.u = u;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.temperature1 = temperature_scalar;
  a.top_k1 = top_k_scalar > vocab ? (int)vocab : (int)(top_k_scalar < 0 ? 0 : top_k_scalar);
  a.top_p1 = top_p_scalar;
  a.min_p1 = min_p_scalar;
  a.out = out;
  a.vocab = (int)vocab;
  a.parts = parts;
  a.part = (int)part;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FI_DTYPE_F32) return launch_sample<float>(a, rows, ctas, st);
  return dtype == FI_DTYPE_F16 ? launch_sample<__half>(a, rows, ctas, st)
                               : launch_sample<__nv_bfloat16>(a, rows, ctas, st);
}
