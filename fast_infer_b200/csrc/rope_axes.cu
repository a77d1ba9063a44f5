// Rotary positions with several axes (time, height, width, ...) and the KV-cache slot write, for
// packed new tokens whose position is not their slot.
//
// Rotate-half RoPE of q and k: with D = 128 and frequency f < 64 of axis a(f),
//   out[f]      = x[f]      * cos[p, f]      - x[f + 64] * sin[p, f],
//   out[f + 64] = x[f + 64] * cos[p, f + 64] + x[f]      * sin[p, f + 64],  p = positions[a(f), t],
// in fp32 with one rounding at the end; v is copied. Token t of the packed rows belongs to the
// sequence b with cu[b] <= t < cu[b+1] and goes to slot ctx[b] - (cu[b+1] - t).
//
// Bound by HBM (each value read and written once; the tables' rows are shared by all heads of
// a token and stay in L1 and L2). A warp takes a token's heads four at a time: 8 lanes hold the
// 8-value pieces of one half of a head each, with their partners 64 further on, so every access is
// 16 bytes and the cos / sin values stay in registers for all heads of the token.
#include "chunk_common.cuh"

namespace fi {

struct RopeAxesArgs {
  const void* qkv;
  void* q_out;
  void* kc;
  void* vc;
  const float* cos_tab;
  const float* sin_tab;
  const int32_t* pos;  // [axes, total], pos_stride between axes
  const int32_t* cu;
  const int32_t* ctx;
  const int32_t* bt;
  int* err;
  int64_t pos_stride, table_rows, table_stride;
  int64_t xs, qs[2], kcs[3], vcs[3], bts[2];
  uint64_t axis_end;  // 16 bits per axis: one past its last frequency
  int total, batch, nq, nkv, num_blocks, max_blocks;
};

template <typename T>
struct Unpack;
template <>
struct Unpack<__half> {
  __device__ static __forceinline__ float2 two(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
};
template <>
struct Unpack<__nv_bfloat16> {
  __device__ static __forceinline__ float2 two(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};

constexpr int kRaThreads = 256;

__device__ __forceinline__ int axis_of(uint64_t axis_end, int f) {
  int axis = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) axis += f >= (int)((axis_end >> (16 * i)) & 0xffff);
  return axis;
}

// 64 registers, so that 32 warps an SM have loads in flight: 33 us for 7742 tokens of 24 + 8 heads
// (4.8 TB/s); 80 registers 38 us, reading further ahead in each warp instead 40 to 57 us.
// `split` warps share a token (small batches have too few tokens to fill the GPU).
template <typename T>
__global__ void __launch_bounds__(kRaThreads, 4) rope_axes_kernel(const RopeAxesArgs a, int split) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kRaThreads / 32);
  const int64_t work = (int64_t)a.total * split;
  const int c = lane & 7, sub = lane >> 3;  // 8-value piece, head within the group of four
  const int end = min(max(a.cu[a.batch], 0), a.total);
  const int heads = a.nq + 2 * a.nkv;
  const int axis8 = axis_of(a.axis_end, c * 8);
  const bool vector_tables =
      __all_sync(0xffffffffu, axis8 == axis_of(a.axis_end, c * 8 + 7)) && a.table_stride % 4 == 0 &&
      ((reinterpret_cast<uintptr_t>(a.cos_tab) | reinterpret_cast<uintptr_t>(a.sin_tab)) & 15) == 0;
  if (a.err && blockIdx.x == 0)
    for (int b = threadIdx.x; b < a.batch; b += kRaThreads)
      if (a.cu[b] < 0 || a.cu[b + 1] < a.cu[b] || a.cu[b + 1] > a.total)
        set_error(a.err, FI_DEVERR_CONTEXT_LEN);
  for (int64_t w = (int64_t)blockIdx.x * (kRaThreads / 32) + (threadIdx.x >> 5); w < work;
       w += warps) {
    const int t = (int)(w / split), part = (int)(w % split);
    // the first heads are on their way while the token's place is looked up
    const T* x = static_cast<const T*>(a.qkv) + (int64_t)t * a.xs + c * 8;
    const int h0 = part * 4 + sub, step = split * 4;
    uint4 lo_next = make_uint4(0, 0, 0, 0), hi_next = lo_next;
    if (h0 < heads) {
      lo_next = *reinterpret_cast<const uint4*>(x + h0 * 128);
      hi_next = *reinterpret_cast<const uint4*>(x + h0 * 128 + 64);
    }
    if (t < a.cu[0] || t >= end) continue;  // rows outside every sequence stay as they were
    // the last b with cu[b] <= t: the lanes probe 32 places at a time
    int lo = 0, n = a.batch;
    while (n > 1) {
      const int gap = (n + 31) / 32, probe = lane * gap;
      const uint32_t le = __ballot_sync(0xffffffffu, probe < n && a.cu[lo + (probe < n ? probe : 0)] <= t);
      const int i = max(31 - __clz((int)le), 0);  // (cu not ascending: any of them)
      n = min(gap, n - i * gap);
      lo += i * gap;
    }
    if (t >= a.cu[lo + 1]) continue;  // cu is not ascending: the token has no sequence
    const int64_t slot = (int64_t)a.ctx[lo] - (a.cu[lo + 1] - t);
    // where k and v go; a slot without a page is reported and not written
    int64_t page = -1;
    if (slot >= 0 && slot < (int64_t)a.max_blocks * kChunkPage)
      page = a.bt[lo * a.bts[0] + (slot / kChunkPage) * a.bts[1]];
    const bool store = page >= 0 && page < a.num_blocks;
    if (!store && lane == 0) set_error(a.err, FI_DEVERR_BAD_BLOCK);
    // this lane's 8 frequencies and their cos / sin in both halves: as vectors where one axis has
    // all 8 and the tables allow
    float cl[8], sl[8], ch[8], sh[8];
    bool in_table = true;
    if (vector_tables) {
      const int64_t p = a.pos[axis8 * a.pos_stride + t];
      in_table = p >= 0 && p < a.table_rows;
      const int64_t off = (in_table ? p : 0) * a.table_stride + c * 8;
      const float* ct = a.cos_tab + off;
      const float* st = a.sin_tab + off;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        *reinterpret_cast<float4*>(cl + e) = *reinterpret_cast<const float4*>(ct + e);
        *reinterpret_cast<float4*>(sl + e) = *reinterpret_cast<const float4*>(st + e);
        *reinterpret_cast<float4*>(ch + e) = *reinterpret_cast<const float4*>(ct + 64 + e);
        *reinterpret_cast<float4*>(sh + e) = *reinterpret_cast<const float4*>(st + 64 + e);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t p = a.pos[axis_of(a.axis_end, c * 8 + e) * a.pos_stride + t];
        const bool in = p >= 0 && p < a.table_rows;
        in_table &= in;
        const int64_t off = (in ? p : 0) * a.table_stride + c * 8 + e;
        cl[e] = a.cos_tab[off];
        sl[e] = a.sin_tab[off];
        ch[e] = a.cos_tab[off + 64];
        sh[e] = a.sin_tab[off + 64];
      }
    }
    if (!__all_sync(0xffffffffu, in_table)) {
      if (lane == 0) set_error(a.err, FI_DEVERR_CONTEXT_LEN);
      continue;
    }
    for (int h = h0; h < heads; h += step) {
      const uint4 lo_raw = lo_next, hi_raw = hi_next;
      if (h + step < heads) {
        lo_next = *reinterpret_cast<const uint4*>(x + (h + step) * 128);
        hi_next = *reinterpret_cast<const uint4*>(x + (h + step) * 128 + 64);
      }
      uint4 lo_out = lo_raw, hi_out = hi_raw;
      if (h < a.nq + a.nkv) {
        const uint32_t* pl = reinterpret_cast<const uint32_t*>(&lo_raw);
        const uint32_t* ph = reinterpret_cast<const uint32_t*>(&hi_raw);
        uint32_t* ol = reinterpret_cast<uint32_t*>(&lo_out);
        uint32_t* oh = reinterpret_cast<uint32_t*>(&hi_out);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 l = Unpack<T>::two(pl[i]), r = Unpack<T>::two(ph[i]);
          ol[i] = Half16<T>::pack(l.x * cl[2 * i] - r.x * sl[2 * i],
                                  l.y * cl[2 * i + 1] - r.y * sl[2 * i + 1]);
          oh[i] = Half16<T>::pack(r.x * ch[2 * i] + l.x * sh[2 * i],
                                  r.y * ch[2 * i + 1] + l.y * sh[2 * i + 1]);
        }
      }
      T* dst;
      if (h < a.nq) {
        dst = static_cast<T*>(a.q_out) + (int64_t)t * a.qs[0] + h * a.qs[1];
      } else {
        if (!store) continue;
        const bool is_v = h >= a.nq + a.nkv;
        const int64_t* cs = is_v ? a.vcs : a.kcs;
        dst = static_cast<T*>(is_v ? a.vc : a.kc) + page * cs[0] + (slot % kChunkPage) * cs[1] +
              (h - a.nq - (is_v ? a.nkv : 0)) * cs[2];
      }
      *reinterpret_cast<uint4*>(dst + c * 8) = lo_out;
      *reinterpret_cast<uint4*>(dst + 64 + c * 8) = hi_out;
    }
  }
}

}  // namespace fi

extern "C" int fi_rope_axes_store(const void* qkv, void* q_out, void* k_cache, void* v_cache,
                                  const float* cos_table, const float* sin_table,
                                  const int32_t* positions, const int32_t* cu_seqlens,
                                  const int32_t* context_lens, const int32_t* block_table,
                                  int64_t total_tokens, int64_t batch, int64_t num_q_heads,
                                  int64_t num_kv_heads, int64_t head_dim, int64_t axes,
                                  const int64_t* sections, int64_t positions_stride,
                                  int64_t table_rows, int64_t table_stride, int64_t num_blocks,
                                  int64_t block_size, int64_t max_blocks_per_seq,
                                  const int64_t* qkv_strides, const int64_t* q_out_strides,
                                  const int64_t* kc_strides, const int64_t* vc_strides,
                                  const int64_t* bt_strides, int64_t dtype, int32_t* error_flag,
                                  void* stream) {
  using namespace fi;
  clear_error();
  if (total_tokens < 0 || batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0 || table_rows <= 0)
    return fail(FI_ERR_INVALID_ARG, "fi_rope_axes_store: bad sizes");
  if (dtype != FI_DTYPE_F16 && dtype != FI_DTYPE_BF16)
    return fail(FI_ERR_INVALID_ARG, "fi_rope_axes_store: unknown dtype %lld", (long long)dtype);
  if (head_dim != 128)
    return fail(FI_ERR_UNSUPPORTED, "fi_rope_axes_store: head_dim %lld != 128", (long long)head_dim);
  if (block_size != kChunkPage)
    return fail(FI_ERR_UNSUPPORTED, "fi_rope_axes_store: block_size %lld != 64",
                (long long)block_size);
  if (axes < 1 || axes > 4 || !sections)
    return fail(FI_ERR_INVALID_ARG, "fi_rope_axes_store: needs 1 to 4 axes with their sections");
  uint64_t ends = 0;
  int64_t f = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < axes) {
      if (sections[i] < 0 || sections[i] > 64)
        return fail(FI_ERR_INVALID_ARG, "fi_rope_axes_store: section %d out of range", i);
      f += sections[i];
    }
    ends |= (uint64_t)(i < axes ? f : 64) << (16 * i);
  }
  if (f != 64)
    return fail(FI_ERR_INVALID_ARG, "fi_rope_axes_store: sections add up to %lld, not head_dim / 2",
                (long long)f);
  if (total_tokens == 0 || batch == 0) return FI_OK;
  if (!qkv || !q_out || !k_cache || !v_cache || !cos_table || !sin_table || !positions ||
      !cu_seqlens || !context_lens || !block_table || !qkv_strides || !q_out_strides ||
      !kc_strides || !vc_strides || !bt_strides)
    return fail(FI_ERR_INVALID_ARG, "fi_rope_axes_store: null pointer argument");
  if (table_stride < head_dim)
    return fail(FI_ERR_INVALID_ARG, "fi_rope_axes_store: table_stride < head_dim");
  if (total_tokens > (1 << 28) || batch > (1 << 28) || num_q_heads > 65535 ||
      num_kv_heads > 65535 || num_blocks > (1 << 30) || max_blocks_per_seq > (1 << 24))
    return fail(FI_ERR_UNSUPPORTED, "fi_rope_axes_store: sizes too large");
  bool ok = qkv_strides[1] == 1 && q_out_strides[2] == 1 && kc_strides[3] == 1 &&
            vc_strides[3] == 1 && stride_ok(total_tokens, qkv_strides[0]) &&
            stride_ok(total_tokens, q_out_strides[0]) && stride_ok(num_q_heads, q_out_strides[1]);
  const int64_t cache_sizes[3] = {num_blocks, block_size, num_kv_heads};
  for (int i = 0; i < 3; ++i)
    ok = ok && stride_ok(cache_sizes[i], kc_strides[i]) && stride_ok(cache_sizes[i], vc_strides[i]);
  ok = ok && aligned16(qkv) && aligned16(q_out) && aligned16(k_cache) && aligned16(v_cache);
  if (!ok)
    return fail(FI_ERR_ALIGNMENT,
                "fi_rope_axes_store: tensors need 16-byte aligned bases, unit innermost strides and "
                "other strides that are multiples of 8 elements");
  RopeAxesArgs a = {};
  a.qkv = qkv;
  a.q_out = q_out;
  a.kc = k_cache;
  a.vc = v_cache;
  a.cos_tab = cos_table;
  a.sin_tab = sin_table;
  a.pos = positions;
  a.cu = cu_seqlens;
  a.ctx = context_lens;
  a.bt = block_table;
  a.err = error_flag;
  a.pos_stride = positions_stride;
  a.table_rows = table_rows;
  a.table_stride = table_stride;
  a.xs = qkv_strides[0];
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = q_out_strides[i];
    a.bts[i] = bt_strides[i];
  }
  for (int i = 0; i < 3; ++i) {
    a.kcs[i] = kc_strides[i];
    a.vcs[i] = vc_strides[i];
  }
  a.axis_end = ends;
  a.total = (int)total_tokens;
  a.batch = (int)batch;
  a.nq = (int)num_q_heads;
  a.nkv = (int)num_kv_heads;
  a.num_blocks = (int)num_blocks;
  a.max_blocks = (int)max_blocks_per_seq;
  // enough warps for the GPU: up to one per four heads when there are few tokens
  const int64_t groups = (num_q_heads + 2 * num_kv_heads + 3) / 4;
  const int64_t fill = (int64_t)sm_count() * 32;
  int64_t split = (fill + total_tokens - 1) / total_tokens;
  if (split > groups) split = groups;
  int64_t blocks = (total_tokens * split + kRaThreads / 32 - 1) / (kRaThreads / 32);
  const int64_t cap = (int64_t)sm_count() * 16;
  if (blocks > cap) blocks = cap;
  const cudaError_t e =
      dtype == FI_DTYPE_F16
          ? launch_pdl(rope_axes_kernel<__half>, dim3((unsigned)blocks), dim3(kRaThreads), 0,
                       static_cast<cudaStream_t>(stream), a, (int)split)
          : launch_pdl(rope_axes_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(kRaThreads), 0,
                       static_cast<cudaStream_t>(stream), a, (int)split);
  if (e != cudaSuccess) return cuda_fail(e, "fi_rope_axes_store launch");
  return FI_OK;
}
