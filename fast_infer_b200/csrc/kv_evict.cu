// Eviction from the paged KV cache by accumulated attention weight.
//
// For every (layer, sequence, KV head) with more than `budget` cached tokens, the first `sinks`,
// the last `recent` and, of those between, the ones of greatest weight stay, `budget` in all;
// ties go to the lowest index, and a weight that is negative or NaN counts as 0. What stays
// keeps its order and moves to slots 0 .. budget-1, of the same pages (in place) or of another
// pool's.
//
// evict_row_kernel, a CTA per (layer, sequence, KV head), finds the weight of the last token that
// stays, the edge, by its bits: a non-negative float orders like its bits. One histogram of 2048
// bins over the 16 octaves below the greatest weight leaves a bin of few weights, among which the
// edge is found by rank. Where that bin holds many (weights far below the greatest, or equal),
// three histograms of the plain bits (11, 11 and 10, from the top) do it instead (taken first, 88
// us for 28 layers x 8 heads of 32768 tokens against 62; counting bit by bit in registers, 109).
// Then each warp lists what it keeps of its run of tokens. The move of the rows, 256 bytes each, is
// bound by HBM (600 us for 3.76 GB read and written), so it keeps many independent 16-byte loads in
// flight; it follows in the same kernel or in evict_copy_kernel.
#include "common.cuh"
#include "host_common.h"

namespace fi {

constexpr int kEvPage = 64;
// threads of a selection: 28 x 16 x 8 rows of 900 to 4096 tokens take 90 us with 512 (256: 94, 128:
// 215), 28 x 8 rows of 32768 take 62 us with 1024 (512: 83)
constexpr int kEvShort = 512, kEvLong = 1024;
constexpr int kEvBins = 2048;
constexpr int kEvStageMax = 12 * 1024;           // tokens whose weights are kept in shared memory
constexpr int kEvList = 1024;                    // weights of the edge's bin that are ranked
constexpr int kEvCopyThreads = 256;
constexpr int kEvSeg = 128;                      // tokens a copy CTA moves, out of place
constexpr int kEvInThreads = 512;                // copy in place
constexpr int kEvRowSeg = 128;                   // tokens a CTA that selected them moves at a time
constexpr int kEvInSeg = 64;                     // tokens it moves between two barriers

struct EvictArgs {
  const char* k;
  const char* v;
  char* ko;
  char* vo;
  const int32_t* bt;
  const int32_t* bto;
  const int32_t* lens;
  const float* mass;
  int32_t* kept;    // [layers, batch, heads, budget]
  float* mass_out;  // [layers, batch, heads, budget]
  int* err;
  int64_t ks[4], vs[4], kos[4], vos[4];  // bytes: layer, page, slot, head
  int64_t bts[2], btos[2];
  int64_t cap;  // tokens of a row of mass
  int layers, batch, heads, num_blocks, num_blocks_out, max_blocks, max_blocks_out;
  int budget, recent, sinks, stage;
};

// Cached tokens of sequence b that the tables can hold.
__device__ __forceinline__ int evict_len(const EvictArgs& a, int b) {
  const int n = a.lens[b];
  return max(0, (int)min((int64_t)n, min((int64_t)a.max_blocks * kEvPage, a.cap)));
}

__device__ __forceinline__ uint32_t weight_bits(float w) { return w > 0.f ? __float_as_uint(w) : 0u; }

// The bin, from the top, in which the count of larger values reaches `want`: on return `want`
// is how many of that bin's values stay. hist has kEvBins counts; all threads call it.
template <int kThreads>
__device__ __forceinline__ int top_bin(const uint32_t* hist, int bins, int& want, uint32_t* sums,
                                       int* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (bins + kThreads - 1) / kThreads;  // this thread's bins, from the top
  uint32_t sum = 0;
  for (int i = 0; i < each; ++i) {
    const int bin = bins - 1 - (tid * each + i);
    if (bin >= 0) sum += hist[bin];
  }
  uint32_t inc = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += x;
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  uint32_t above = inc - sum;
  for (int w = 0; w < warp; ++w) above += sums[w];
  if (above < (uint32_t)want && above + sum >= (uint32_t)want) {
    for (int i = 0; i < each; ++i) {
      const int bin = bins - 1 - (tid * each + i);
      if (above + hist[bin] >= (uint32_t)want) {
        found[0] = bin;
        found[1] = want - (int)above;
        break;
      }
      above += hist[bin];
    }
  }
  __syncthreads();
  want = found[1];
  return found[0];
}

// Lists in kept and mass_out what stays of one row; all threads of the CTA call it.
template <int kThreads>
__device__ __forceinline__ void evict_select(const EvictArgs& a, int64_t row) {
  extern __shared__ uint32_t ev_smem[];
  uint32_t* hist = ev_smem;             // [kEvBins]
  uint32_t* stage = ev_smem + kEvBins;  // [a.stage]
  __shared__ uint32_t sums[kThreads / 32];
  __shared__ uint32_t run_over[kThreads / 32], run_same[kThreads / 32];
  __shared__ int found[2];
  __shared__ uint32_t listed, list[kEvList];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = (int)(row / a.heads % a.batch);
  const float* mass = a.mass + row * a.cap;
  int32_t* kept = a.kept + row * a.budget;
  float* mass_out = a.mass_out + row * a.budget;
  const int n = evict_len(a, b);
  if (tid == 0 && row % ((int64_t)a.batch * a.heads) == (int64_t)b * a.heads &&
      row < (int64_t)a.batch * a.heads && n != a.lens[b])
    set_error(a.err, FI_DEVERR_CONTEXT_LEN);
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += kThreads) {
      kept[i] = i < n ? i : -1;
      mass_out[i] = i < n ? mass[i] : 0.f;
    }
    return;
  }
  const int lo = a.sinks, hi = n - a.recent;  // the tokens that compete
  const bool staged = n <= a.stage;
  // f(token, weight's bits) for tokens [from, to): eight reads on their way at a time
  auto sweep = [&](int from, int to, bool first, auto&& f) {
#pragma unroll 1
    for (int j0 = from + tid; j0 < to; j0 += 8 * kThreads) {
      uint32_t x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = j0 + k * kThreads;
        x[k] = 0;
        if (j < to) x[k] = staged && !first ? stage[j] : __float_as_uint(mass[j]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (j0 + k * kThreads < to) f(j0 + k * kThreads, x[k]);
    }
  };
  int want = a.budget - a.sinks - a.recent;
  uint32_t edge = 0xffffffffu;  // weights above it stay, and `want` of its equals
  uint32_t top = 0;             // the greatest weight that competes
  sweep(0, n, true, [&](int j, uint32_t raw) {
    if (staged) stage[j] = raw;
    if (j >= lo && j < hi) top = max(top, weight_bits(__uint_as_float(raw)));
  });
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane == 0) sums[warp] = top;
  for (int i = tid; i < kEvBins; i += kThreads) hist[i] = 0;
  if (tid == 0) listed = 0;
  __syncthreads();
  if (want > 0) {
    for (int w = 0; w < kThreads / 32; ++w) top = max(top, sums[w]);
    // bin: 7 bits below the exponent over 16 octaves; all that is smaller shares bin 0, whose
    // count no one needs
    const int base = (int)(top >> 16) - (kEvBins - 1);
    auto bin_of = [&](uint32_t x) { return max((int)(x >> 16) - base, 0); };
    sweep(lo, hi, false, [&](int, uint32_t raw) {
      const int k = bin_of(weight_bits(__uint_as_float(raw)));
      if (k > 0) atomicAdd(&hist[k], 1u);
    });
    __syncthreads();
    if (tid == 0) hist[0] = 0x3fffffffu;  // whatever is left
    __syncthreads();
    int in_bin = want;
    const int bin = top_bin<kThreads>(hist, kEvBins, in_bin, sums, found);
    sweep(lo, hi, false, [&](int, uint32_t raw) {
      const uint32_t x = weight_bits(__uint_as_float(raw));
      if (bin_of(x) == bin) {
        const uint32_t at = atomicAdd(&listed, 1u);
        if (at < kEvList) list[at] = x;
      }
    });
    __syncthreads();
    if (listed <= kEvList) {
      for (int i = tid; i < (int)listed; i += kThreads) {
        const uint32_t x = list[i];
        int over = 0, same = 0;
        for (int k = 0; k < (int)listed; ++k) {
          over += list[k] > x;
          same += list[k] == x;
        }
        if (over < in_bin && in_bin <= over + same) {  // all that are equal write the same
          found[0] = (int)x;
          found[1] = in_bin - over;
        }
      }
      __syncthreads();
      edge = (uint32_t)found[0];
      want = found[1];
    } else {
      uint32_t prefix = 0;
#pragma unroll 1
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bins = pass == 2 ? 1024 : 2048;
        const int high = pass == 0 ? 31 : pass == 1 ? 21 : 10;  // (bit 31 is never set)
        __syncthreads();
        for (int i = tid; i < bins; i += kThreads) hist[i] = 0;
        __syncthreads();
        sweep(lo, hi, false, [&](int, uint32_t raw) {
          const uint32_t x = weight_bits(__uint_as_float(raw));
          if (x >> high == prefix) atomicAdd(&hist[(x >> shift) & (bins - 1)], 1u);
        });
        __syncthreads();
        prefix = (prefix << (pass == 2 ? 10 : 11)) | (uint32_t)top_bin<kThreads>(hist, bins, want, sums, found);
      }
      edge = prefix;
    }
  }
  // Each warp has a run of tokens: it counts what is over the edge and what equals it, then lists
  // what stays; 8 x 32 tokens at a time.
  const int each = ((n + kThreads - 1) / kThreads) * 32;
  const int j0 = min(warp * each, n), j1 = min(j0 + each, n);
  uint32_t before_over = 0, before_same = 0;
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll 1
  for (int list_now = 0; list_now < 2; ++list_now) {
    uint32_t n_over = 0, n_same = 0;
#pragma unroll 1
    for (int base = j0; base < j1; base += 256) {
      uint32_t raw[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = base + k * 32 + lane;
        raw[k] = 0;
        if (j < j1) raw[k] = staged ? stage[j] : __float_as_uint(mass[j]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (base + k * 32 >= j1) break;
        const int j = base + k * 32 + lane;
        const bool in = j < j1, mid = in && j >= lo && j < hi;
        const uint32_t x = weight_bits(__uint_as_float(raw[k]));
        const bool is_over = in && (!mid || x > edge), is_same = mid && x == edge;
        const uint32_t bo = __ballot_sync(0xffffffffu, is_over), bs = __ballot_sync(0xffffffffu, is_same);
        if (list_now) {
          const uint32_t same_rank = before_same + n_same + __popc(bs & below);
          if (is_over || (is_same && same_rank < (uint32_t)want)) {
            const uint32_t at =
                before_over + n_over + __popc(bo & below) + min(same_rank, (uint32_t)want);
            kept[at] = j;
            mass_out[at] = __uint_as_float(raw[k]);
          }
        }
        n_over += __popc(bo);
        n_same += __popc(bs);
      }
    }
    if (list_now) break;
    if (lane == 0) {
      run_over[warp] = n_over;
      run_same[warp] = n_same;
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w) {
      before_over += run_over[w];
      before_same += run_same[w];
    }
  }
}

// Page and slot of a token, or page -1 if the table's entry is invalid.
__device__ __forceinline__ int2 evict_slot(const int32_t* bt, const int64_t* bts, int b, int j,
                                           int max_blocks, int num_blocks) {
  const int pg = j / kEvPage;
  int page = -1;
  if (pg < max_blocks) page = bt[b * bts[0] + (int64_t)pg * bts[1]];
  if (page >= num_blocks) page = -1;
  return make_int2(page, j % kEvPage);
}

__device__ __forceinline__ uint4 ld_stream(const char* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// Moves the kept tokens [t0, t1) of a row, kSeg at a time, a half warp per token and iteration. In
// place that is safe when one CTA walks all of the row: a token's new slot is never past its old
// one, so what a segment writes, later segments do not read; within one, every load comes before
// any store. The places of the next segment are looked up while this one's values are on their way
// (in place, 28 x 16 x 8 rows: 779 -> 695 us; segments of 128 tokens 768).
template <int kThreads, int kSeg, bool kInPlace>
__device__ __forceinline__ void evict_move(const EvictArgs& a, int layer, int b, int h, int t0, int t1) {
  constexpr int kPer = kSeg * 16 / kThreads;  // 16-byte pieces of K, and of V, a thread moves
  __shared__ int2 src_ring[3][kSeg], dst_ring[3][kSeg];
  const int tid = threadIdx.x, piece = tid & 15;
  const int n = evict_len(a, b);
  const int count = min(min(n, a.budget), t1);
  if (kInPlace && n <= a.budget) return;
  const int32_t* kept = a.kept + (((int64_t)layer * a.batch + b) * a.heads + h) * a.budget;
  const char* k = a.k + layer * a.ks[0] + h * a.ks[3] + piece * 16;
  const char* v = a.v + layer * a.vs[0] + h * a.vs[3] + piece * 16;
  char* ko = a.ko + layer * a.kos[0] + h * a.kos[3] + piece * 16;
  char* vo = a.vo + layer * a.vos[0] + h * a.vos[3] + piece * 16;
  auto look_up = [&](int from, int2* src, int2* dst) {
    for (int i = tid; i < min(kSeg, count - from); i += kThreads) {
      const int j = kept[from + i];
      int2 at = evict_slot(a.bt, a.bts, b, j, a.max_blocks, a.num_blocks);
      dst[i] = evict_slot(a.bto, a.btos, b, from + i, a.max_blocks_out, a.num_blocks_out);
      if (at.x < 0 || dst[i].x < 0) {
        set_error(a.err, FI_DEVERR_BAD_BLOCK);
        at.x = -1;
      } else if (kInPlace && j == from + i) {
        at.x = -1;  // it stays where it is
      }
      src[i] = at;
    }
  };
  look_up(t0, src_ring[0], dst_ring[0]);
  __syncthreads();
#pragma unroll 1
  for (int slot = 0; t0 < count; t0 += kSeg) {
    const int2 *src = src_ring[slot], *dst = dst_ring[slot];
    slot = slot == 2 ? 0 : slot + 1;
    uint4 kx[kPer], vx[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = (tid >> 4) + i * (kThreads / 16);
      if (t0 + t < count && src[t].x >= 0) {
        kx[i] = ld_stream(k + src[t].x * a.ks[1] + src[t].y * a.ks[2]);
        vx[i] = ld_stream(v + src[t].x * a.vs[1] + src[t].y * a.vs[2]);
      }
    }
    look_up(t0 + kSeg, src_ring[slot], dst_ring[slot]);  // (last read two barriers ago)
    __syncthreads();  // the loads of all threads are done, the next segment's places known
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = (tid >> 4) + i * (kThreads / 16);
      if (t0 + t < count && src[t].x >= 0) {
        *reinterpret_cast<uint4*>(ko + dst[t].x * a.kos[1] + dst[t].y * a.kos[2]) = kx[i];
        *reinterpret_cast<uint4*>(vo + dst[t].x * a.vos[1] + dst[t].y * a.vos[2]) = vx[i];
      }
    }
  }
}

// A CTA per row: selection, then (kMove) the row's move.
template <int kThreads, bool kMove, bool kInPlace>
__global__ void __launch_bounds__(kThreads) evict_row_kernel(const EvictArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int64_t row = blockIdx.x;
  evict_select<kThreads>(a, row);
  if (kMove) {
    __syncthreads();
    const int64_t seq = row / a.heads;
    evict_move<kThreads, kInPlace ? kEvInSeg : kEvRowSeg, kInPlace>(
        a, (int)(seq / a.batch), (int)(seq % a.batch), (int)(row % a.heads), 0, a.budget);
  }
}

// The move of rows that evict_row_kernel has listed: a CTA per row in place, else per kSeg tokens.
template <int kThreads, int kSeg, bool kInPlace>
__global__ void __launch_bounds__(kThreads) evict_copy_kernel(const EvictArgs a, int segs) {
  grid_dep_wait();
  grid_dep_launch();
  // the heads of one stretch of tokens run side by side: their rows are neighbours in memory
  int64_t r = blockIdx.x;
  const int h = (int)(r % a.heads);
  r /= a.heads;
  const int seg = kInPlace ? 0 : (int)(r % segs);
  if (!kInPlace) r /= segs;
  evict_move<kThreads, kSeg, kInPlace>(a, (int)(r / a.batch), (int)(r % a.batch), h, seg * kSeg,
                                       kInPlace ? a.budget : min((seg + 1) * kSeg, a.budget));
}

}  // namespace fi

extern "C" int fi_kv_evict(const void* k, const void* v, const int32_t* block_table,
                           const int32_t* seq_lens, const float* mass, void* k_out, void* v_out,
                           const int32_t* block_table_out, int32_t* kept, float* mass_out,
                           int64_t layers, int64_t batch, int64_t num_heads, int64_t head_dim,
                           int64_t num_blocks, int64_t num_blocks_out, int64_t block_size,
                           int64_t max_blocks_per_seq, int64_t max_blocks_per_seq_out,
                           int64_t mass_capacity, int64_t budget, int64_t recent, int64_t sinks,
                           const int64_t* k_strides, const int64_t* v_strides,
                           const int64_t* ko_strides, const int64_t* vo_strides,
                           const int64_t* bt_strides, const int64_t* bto_strides,
                           int32_t* error_flag, void* stream) {
  using namespace fi;
  clear_error();
  if (layers < 0 || batch < 0 || num_heads <= 0 || num_blocks <= 0 || num_blocks_out <= 0 ||
      max_blocks_per_seq <= 0 || max_blocks_per_seq_out <= 0 || mass_capacity < 0)
    return fail(FI_ERR_INVALID_ARG, "fi_kv_evict: bad sizes");
  if (budget <= 0 || recent < 0 || sinks < 0 || recent > budget || sinks > budget - recent)
    return fail(FI_ERR_INVALID_ARG,
                "fi_kv_evict: needs budget >= 1 and recent + sinks <= budget (got %lld, %lld, %lld)",
                (long long)budget, (long long)recent, (long long)sinks);
  if (head_dim != 128)
    return fail(FI_ERR_UNSUPPORTED, "fi_kv_evict: head_dim %lld != 128", (long long)head_dim);
  if (block_size != kEvPage)
    return fail(FI_ERR_UNSUPPORTED, "fi_kv_evict: block_size %lld != 64", (long long)block_size);
  if (budget > max_blocks_per_seq_out * kEvPage)
    return fail(FI_ERR_INVALID_ARG, "fi_kv_evict: budget %lld does not fit the output block table",
                (long long)budget);
  if (layers == 0 || batch == 0) return FI_OK;
  if (!k || !v || !block_table || !seq_lens || !mass || !k_out || !v_out || !block_table_out ||
      !kept || !mass_out || !k_strides || !v_strides || !ko_strides || !vo_strides || !bt_strides ||
      !bto_strides)
    return fail(FI_ERR_INVALID_ARG, "fi_kv_evict: null pointer argument");
  const bool in_place = k_out == k;
  if (in_place != (v_out == v) || in_place != (block_table_out == block_table))
    return fail(FI_ERR_INVALID_ARG,
                "fi_kv_evict: in place needs k, v and the block table themselves as outputs, out of "
                "place none of them");
  if (num_blocks > (1 << 30) || num_blocks_out > (1 << 30) || max_blocks_per_seq > (1 << 24) ||
      max_blocks_per_seq_out > (1 << 24))
    return fail(FI_ERR_UNSUPPORTED, "fi_kv_evict: sizes too large");
  const int64_t rows = layers * batch * num_heads;
  const int64_t segs = in_place ? 1 : (budget + kEvSeg - 1) / kEvSeg;
  if (layers > (1 << 20) || batch > (1 << 20) || num_heads > 65535 || rows > 0x7fffffff ||
      segs > 0x7fffffff / rows)
    return fail(FI_ERR_UNSUPPORTED, "fi_kv_evict: sizes too large");
  EvictArgs a = {};
  bool ok = aligned16(k) && aligned16(v) && aligned16(k_out) && aligned16(v_out);
  const int64_t* strides[4] = {k_strides, v_strides, ko_strides, vo_strides};
  int64_t* bytes[4] = {a.ks, a.vs, a.kos, a.vos};
  const int64_t sizes[4] = {layers, num_blocks, block_size, num_heads};
  for (int t = 0; t < 4; ++t) {
    ok = ok && strides[t][4] == 1;
    for (int i = 0; i < 4; ++i) {
      ok = ok && stride_ok(t >= 2 && i == 1 ? num_blocks_out : sizes[i], strides[t][i]);
      bytes[t][i] = strides[t][i] * 2;
      if (in_place && t >= 2 && strides[t][i] != strides[t - 2][i])
        return fail(FI_ERR_INVALID_ARG, "fi_kv_evict: in place with other strides");
    }
  }
  if (!ok)
    return fail(FI_ERR_ALIGNMENT,
                "fi_kv_evict: caches need 16-byte aligned bases, unit innermost strides and other "
                "strides that are multiples of 8 elements");
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.ko = static_cast<char*>(k_out);
  a.vo = static_cast<char*>(v_out);
  a.bt = block_table;
  a.bto = block_table_out;
  a.lens = seq_lens;
  a.mass = mass;
  a.kept = kept;
  a.mass_out = mass_out;
  a.err = error_flag;
  a.bts[0] = bt_strides[0];
  a.bts[1] = bt_strides[1];
  a.btos[0] = bto_strides[0];
  a.btos[1] = bto_strides[1];
  a.cap = mass_capacity;
  a.layers = (int)layers;
  a.batch = (int)batch;
  a.heads = (int)num_heads;
  a.num_blocks = (int)num_blocks;
  a.num_blocks_out = (int)num_blocks_out;
  a.max_blocks = (int)max_blocks_per_seq;
  a.max_blocks_out = (int)max_blocks_per_seq_out;
  a.budget = (int)budget;
  a.recent = (int)recent;
  a.sinks = (int)sinks;
  const int64_t longest = max_blocks_per_seq * kEvPage < mass_capacity
                              ? max_blocks_per_seq * kEvPage : mass_capacity;
  a.stage = (int)(longest <= kEvStageMax ? longest : 0);
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    const void* kernels[] = {(const void*)evict_row_kernel<kEvLong, false, false>,
                             (const void*)evict_row_kernel<kEvShort, false, false>,
                             (const void*)evict_row_kernel<kEvShort, true, false>,
                             (const void*)evict_row_kernel<kEvShort, true, true>};
    for (const void* f : kernels) {
      const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (kEvBins + kEvStageMax) * 4);
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  });
  if (e != cudaSuccess) return cuda_fail(e, "fi_kv_evict: cudaFuncSetAttribute");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = (size_t)(kEvBins + a.stage) * 4;
  const dim3 grid((unsigned)rows);
  const bool is_short = longest <= 16 * kEvShort;
  // Many short rows: one kernel, whose selections run beside other rows' moves (28 x 16 x 8 rows of
  // 2048 tokens to 1024: 633 us, 690 in two, in place 645 and 695; 1 x 100 x 8: 155 and 164, in
  // place 161 and 168). Fewer rows leave SMs without one to move (28 x 3 x 8 of 8192 to 2048: 281
  // and 271; a few short rows, whose move is less than a launch, were not measured).
  if (is_short && rows >= 5 * sm_count()) {
    e = in_place ? launch_pdl(evict_row_kernel<kEvShort, true, true>, grid, dim3(kEvShort), smem, st, a)
                 : launch_pdl(evict_row_kernel<kEvShort, true, false>, grid, dim3(kEvShort), smem, st, a);
    return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_kv_evict: launch");
  }
  e = is_short ? launch_pdl(evict_row_kernel<kEvShort, false, false>, grid, dim3(kEvShort), smem, st, a)
               : launch_pdl(evict_row_kernel<kEvLong, false, false>, grid, dim3(kEvLong), smem, st, a);
  if (e != cudaSuccess) return cuda_fail(e, "fi_kv_evict: select launch");
  if (in_place)
    e = launch_pdl(evict_copy_kernel<kEvInThreads, kEvInSeg, true>, grid, dim3(kEvInThreads), 0, st, a, 1);
  else
    e = launch_pdl(evict_copy_kernel<kEvCopyThreads, kEvSeg, false>, dim3((unsigned)(rows * segs)),
                   dim3(kEvCopyThreads), 0, st, a, (int)segs);
  if (e != cudaSuccess) return cuda_fail(e, "fi_kv_evict: copy launch");
  return FI_OK;
}
