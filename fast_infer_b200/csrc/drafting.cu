// The token side of drafting: the shape of draft trees, the acceptance of drafts, and the move of the
// accepted tokens' K and V. New tokens are packed: sequence b owns rows [cu[b], cu[b+1]); its i-th
// new token is node i of its tree, parents[i] < i its parent's number, anything else makes a root.
#include "chunk_common.cuh"

namespace fi {

constexpr int kDrThreads = 128;
constexpr int kDrSmemNodes = 4096;  // parents of one sequence held in shared memory

struct DrRange {
  int start, n;
};
// Rows of sequence b, clamped to the tensors.
__device__ __forceinline__ DrRange dr_range(const int32_t* cu, int b, int total, int* err) {
  const int c0 = cu[b], c1 = cu[b + 1];
  const int start = min(max(c0, 0), total), end = min(max(c1, start), total);
  if ((start != c0 || end != c1) && threadIdx.x == 0) set_error(err, FI_DEVERR_CONTEXT_LEN);
  return {start, end - start};
}

// Ancestor bits and depth of every node. A thread walks from its node to the root; as a parent's number is
// below its child's, the walk leaves a mask word for good when it passes below it, so a word is
// built in a register and stored once. Bound by the launch and the walk's chain of shared-memory
// reads (26 nodes 2.4 us, 256 trees of 40 to 250 nodes 5.5 us); pointer doubling would touch log2 as
// many links a node but needs a barrier and the masks in shared memory for each.
__global__ void __launch_bounds__(kDrThreads)
    draft_tree_kernel(const int32_t* parents, const int32_t* cu, int32_t* mask, int32_t* depths,
                      int total, int words, int window, int* err) {
  __shared__ int32_t par[kDrSmemNodes];
  grid_dep_wait();
  grid_dep_launch();
  const DrRange r = dr_range(cu, blockIdx.x, total, err);
  const int first = blockIdx.y * kDrThreads;
  if (first >= r.n) return;
  const int32_t* gpar = parents + r.start;
  const int held = min(r.n, kDrSmemNodes);
  for (int i = threadIdx.x; i < held; i += kDrThreads) par[i] = gpar[i];
  __syncthreads();
  for (int node = first + threadIdx.x; node < r.n; node += gridDim.y * kDrThreads) {
    int32_t* row = mask + (int64_t)(r.start + node) * words;
    int at = node, depth = 0, word = words - 1;
    uint32_t bits = 0;
    if (node >= words * 32) set_error(err, FI_DEVERR_CONTEXT_LEN);  // (bits past the mask are dropped)
    while (true) {
      if (depth < window && at < words * 32) {
        for (; word > at >> 5; --word) {
          row[word] = (int32_t)bits;
          bits = 0;
        }
        bits |= 1u << (at & 31);
      }
      const int up = at < held ? par[at] : gpar[at];
      if (up < 0 || up >= at) break;
      at = up;
      ++depth;
    }
    for (; word >= 0; --word) {
      row[word] = (int32_t)bits;
      bits = 0;
    }
    depths[r.start + node] = depth;
  }
}

// Acceptance. A warp per sequence walks from node 0: from an accepted node to its first child whose
// token is the one sampled after the node; a negative one is no token (a row that could not be sampled gives -1) and ends
// the walk. Children have greater numbers, so one pass over the nodes,
// 32 at a time in registers, finds the whole path. Bound by the launch (26 nodes 1.4 us, 48 trees of 20 to 64 nodes 2.3).
__global__ void __launch_bounds__(kDrThreads)
    accept_kernel(const int32_t* tokens, const int32_t* sampled, const int32_t* parents,
                  const int32_t* cu, int32_t* path, int32_t* counts, int32_t* follow, int total,
                  int batch, int* err) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, b = blockIdx.x * (kDrThreads / 32) + (threadIdx.x >> 5);
  if (b >= batch) return;
  const int c0 = cu[b], c1 = cu[b + 1];
  const int start = min(max(c0, 0), total), n = min(max(c1, start), total) - start;
  if ((start != c0 || start + n != c1) && lane == 0) set_error(err, FI_DEVERR_CONTEXT_LEN);
  int count = 0, cur = 0, want = -1;
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane;
    const bool live = i < n;
    const int tok = live ? tokens[start + i] : 0, smp = live ? sampled[start + i] : 0;
    const int par = live ? parents[start + i] : -1;
    if (base == 0) {
      want = __shfl_sync(0xffffffffu, smp, 0);
      if (lane == 0) path[start] = 0;
      count = 1;
    }
    while (true) {
      const uint32_t hit = __ballot_sync(0xffffffffu, live && want >= 0 && i > cur && par == cur && tok == want);
      if (hit == 0) break;
      const int at = __ffs((int)hit) - 1;
      cur = base + at;
      want = __shfl_sync(0xffffffffu, smp, at);
      if (lane == 0) path[start + count] = cur;
      ++count;
    }
  }
  for (int d = count + lane; d < n; d += 32) path[start + d] = -1;
  if (lane == 0) {
    counts[b] = count;
    follow[b] = want;
  }
}

// The move: for every layer, K and V of accepted node path[d] go from slot past + path[d] to slot
// past + d. A thread owns 16 bytes of a head (and, with scales, 4) for all d, in ascending order:
// path[d] >= d, so a slot written for d is read by no later d, and by an earlier one before. Batches of
// kMvBatch loads are in flight before the first store. A CTA per sequence and layer; bound by latency for few tokens (28
// layers of 8 heads, one request: 2.8 us) and mostly for many (48 requests, 66 MB: 11.4 us, 5.8 TB/s of a copy's 6.5).
struct MoveArgs {
  uint8_t* pool[2];   // k, v
  float* scale[2];    // their scales, or null
  int64_t st[2][4];   // bytes: layer, page, slot, head
  int64_t ss[2][4];   // elements: layer, page, head, slot
  const int32_t* bt;
  const int32_t* cu;
  const int32_t* ctx;
  const int32_t* path;
  const int32_t* counts;
  int64_t bts[2];
  int total, heads, pieces, num_blocks, max_blocks;
  int* err;
};
constexpr int kMvThreads = 256;
constexpr int kMvBatch = 8;
constexpr int kMvPlan = 64;  // moves whose places are looked up at a time

__global__ void __launch_bounds__(kMvThreads) keep_kernel(const MoveArgs a) {
  __shared__ int from_page[kMvPlan], to_page[kMvPlan], from_slot[kMvPlan], to_slot[kMvPlan];
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x, layer = blockIdx.y;
  const DrRange r = dr_range(a.cu, b, a.total, a.err);
  const int count = min(max(a.counts[b], 0), r.n);
  const int64_t past = (int64_t)a.ctx[b] - r.n;
  if (count == 0) return;
  const int rows = a.heads * a.pieces;
  const int items = 2 * rows + (a.scale[0] ? 2 * a.heads : 0);
  for (int d0 = 1; d0 < count; d0 += kMvPlan) {
    const int moves = min(kMvPlan, count - d0);
    if (threadIdx.x < moves) {
      const int d = d0 + threadIdx.x, node = a.path[r.start + d];
      int page[2] = {-1, -1};
      const int64_t slot[2] = {past + node, past + d};
      // a node that stays where it is, or that the path leaves out, is not moved
      if (node > d && node < r.n) {
        for (int i = 0; i < 2; ++i) {
          if (slot[i] >= 0 && slot[i] < (int64_t)a.max_blocks * kChunkPage)
            page[i] = a.bt[b * a.bts[0] + (slot[i] / kChunkPage) * a.bts[1]];
          if (page[i] < 0 || page[i] >= a.num_blocks) {
            page[i] = -1;
            set_error(a.err, FI_DEVERR_BAD_BLOCK);
          }
        }
      }
      from_page[threadIdx.x] = page[1] < 0 ? -1 : page[0];
      to_page[threadIdx.x] = page[1];
      from_slot[threadIdx.x] = (int)(slot[0] & (kChunkPage - 1));
      to_slot[threadIdx.x] = (int)(slot[1] & (kChunkPage - 1));
    }
    __syncthreads();
    for (int it = threadIdx.x; it < items; it += kMvThreads) {
      if (it < 2 * rows) {
        const int kv = it >= rows, x = kv ? it - rows : it;
        const int64_t* st = a.st[kv];
        uint8_t* base = a.pool[kv] + layer * st[0] + (x / a.pieces) * st[3] + (x % a.pieces) * 16;
        for (int m0 = 0; m0 < moves; m0 += kMvBatch) {
          uint4 v[kMvBatch];
#pragma unroll
          for (int m = 0; m < kMvBatch; ++m)
            if (m0 + m < moves && from_page[m0 + m] >= 0)
              v[m] = *reinterpret_cast<const uint4*>(base + from_page[m0 + m] * st[1] +
                                                     from_slot[m0 + m] * st[2]);
#pragma unroll
          for (int m = 0; m < kMvBatch; ++m)
            if (m0 + m < moves && from_page[m0 + m] >= 0)
              *reinterpret_cast<uint4*>(base + to_page[m0 + m] * st[1] + to_slot[m0 + m] * st[2]) =
                  v[m];
        }
      } else {
        const int kv = it - 2 * rows >= a.heads, h = it - 2 * rows - (kv ? a.heads : 0);
        const int64_t* st = a.ss[kv];
        float* base = a.scale[kv] + layer * st[0] + h * st[2];
        for (int m0 = 0; m0 < moves; m0 += kMvBatch) {
          float v[kMvBatch];
#pragma unroll
          for (int m = 0; m < kMvBatch; ++m)
            if (m0 + m < moves && from_page[m0 + m] >= 0)
              v[m] = base[from_page[m0 + m] * st[1] + from_slot[m0 + m] * st[3]];
#pragma unroll
          for (int m = 0; m < kMvBatch; ++m)
            if (m0 + m < moves && from_page[m0 + m] >= 0)
              base[to_page[m0 + m] * st[1] + to_slot[m0 + m] * st[3]] = v[m];
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace fi

extern "C" int fi_draft_tree(const int32_t* parents, const int32_t* cu_seqlens, int32_t* mask,
                             int32_t* depths, int64_t total_tokens, int64_t batch,
                             int64_t mask_words, int64_t window, int32_t* error_flag,
                             void* stream) {
  using namespace fi;
  clear_error();
  if (total_tokens < 0 || batch < 0 || mask_words <= 0 || window < 0)
    return fail(FI_ERR_INVALID_ARG, "fi_draft_tree: bad sizes");
  if (total_tokens > (1 << 28) || batch > (1 << 20) || mask_words > (1 << 16))
    return fail(FI_ERR_UNSUPPORTED, "fi_draft_tree: sizes too large");
  if (total_tokens == 0 || batch == 0) return FI_OK;
  if (!parents || !cu_seqlens || !mask || !depths)
    return fail(FI_ERR_INVALID_ARG, "fi_draft_tree: null pointer argument");
  const int seen = window == 0 || window > 0x7fffffff ? 0x7fffffff : (int)window;
  const int64_t parts = (mask_words * 32 + kDrThreads - 1) / kDrThreads;
  const cudaError_t e = launch_pdl(
      draft_tree_kernel, dim3((unsigned)batch, (unsigned)(parts < 64 ? parts : 64)), dim3(kDrThreads),
      0, static_cast<cudaStream_t>(stream), parents, cu_seqlens, mask, depths, (int)total_tokens,
      (int)mask_words, seen, error_flag);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_draft_tree launch");
}

extern "C" int fi_accept_drafts(const int32_t* tokens, const int32_t* sampled,
                                const int32_t* parents, const int32_t* cu_seqlens, int32_t* path,
                                int32_t* counts, int32_t* next_tokens, int64_t total_tokens,
                                int64_t batch, int32_t* error_flag, void* stream) {
  using namespace fi;
  clear_error();
  if (total_tokens < 0 || batch < 0)
    return fail(FI_ERR_INVALID_ARG, "fi_accept_drafts: bad sizes");
  if (total_tokens > (1 << 28) || batch > (1 << 20))
    return fail(FI_ERR_UNSUPPORTED, "fi_accept_drafts: sizes too large");
  if (batch == 0) return FI_OK;
  if (!cu_seqlens || !counts || !next_tokens ||
      (total_tokens > 0 && (!tokens || !sampled || !parents || !path)))
    return fail(FI_ERR_INVALID_ARG, "fi_accept_drafts: null pointer argument");
  const int per = kDrThreads / 32;
  const cudaError_t e = launch_pdl(accept_kernel, dim3((unsigned)((batch + per - 1) / per)),
                                   dim3(kDrThreads), 0, static_cast<cudaStream_t>(stream), tokens,
                                   sampled, parents, cu_seqlens, path, counts, next_tokens,
                                   (int)total_tokens, (int)batch, error_flag);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_accept_drafts launch");
}

extern "C" int fi_keep_accepted(void* k, void* v, float* k_scale, float* v_scale,
                                const int32_t* block_table, const int32_t* cu_seqlens,
                                const int32_t* context_lens, const int32_t* path,
                                const int32_t* counts, int64_t layers, int64_t batch,
                                int64_t total_tokens, int64_t num_heads, int64_t head_dim,
                                int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq,
                                const int64_t* k_strides, const int64_t* v_strides,
                                const int64_t* ks_strides, const int64_t* vs_strides,
                                const int64_t* bt_strides, int64_t dtype, int32_t* error_flag,
                                void* stream) {
  using namespace fi;
  clear_error();
  if (layers < 0 || batch < 0 || total_tokens < 0 || num_heads <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0)
    return fail(FI_ERR_INVALID_ARG, "fi_keep_accepted: bad sizes");
  if (dtype < FI_DTYPE_F16 || dtype > FI_DTYPE_E4M3)
    return fail(FI_ERR_INVALID_ARG, "fi_keep_accepted: unknown dtype %lld", (long long)dtype);
  const bool coded = dtype == FI_DTYPE_I8 || dtype == FI_DTYPE_E4M3;
  if (head_dim != 128)
    return fail(FI_ERR_UNSUPPORTED, "fi_keep_accepted: head_dim %lld != 128", (long long)head_dim);
  if (block_size != kChunkPage)
    return fail(FI_ERR_UNSUPPORTED, "fi_keep_accepted: block_size %lld != 64",
                (long long)block_size);
  if (layers > 65535 || batch > (1 << 20) || total_tokens > (1 << 28) || num_heads > 65535 ||
      num_blocks > (1 << 30) || max_blocks_per_seq > (1 << 24))
    return fail(FI_ERR_UNSUPPORTED, "fi_keep_accepted: sizes too large");
  if (layers == 0 || batch == 0 || total_tokens == 0) return FI_OK;
  if (!k || !v || !block_table || !cu_seqlens || !context_lens || !path || !counts || !k_strides ||
      !v_strides || !bt_strides || (coded && (!k_scale || !v_scale || !ks_strides || !vs_strides)))
    return fail(FI_ERR_INVALID_ARG, "fi_keep_accepted: null pointer argument");
  const int bytes = coded ? 1 : 2;
  bool ok = aligned16(k) && aligned16(v) && k_strides[4] == 1 && v_strides[4] == 1;
  const int64_t sizes[4] = {layers, num_blocks, block_size, num_heads};
  for (int i = 0; i < 4; ++i)
    ok = ok && (sizes[i] == 1 || (k_strides[i] * bytes % 16 == 0 && v_strides[i] * bytes % 16 == 0));
  if (!ok)
    return fail(FI_ERR_ALIGNMENT,
                "fi_keep_accepted: k and v need 16-byte aligned bases, unit innermost strides and "
                "other strides that are multiples of 16 bytes");
  MoveArgs a = {};
  a.pool[0] = static_cast<uint8_t*>(k);
  a.pool[1] = static_cast<uint8_t*>(v);
  for (int i = 0; i < 4; ++i) {
    a.st[0][i] = k_strides[i] * bytes;
    a.st[1][i] = v_strides[i] * bytes;
    if (coded) {
      a.ss[0][i] = ks_strides[i];
      a.ss[1][i] = vs_strides[i];
    }
  }
  if (coded) {
    a.scale[0] = k_scale;
    a.scale[1] = v_scale;
  }
  a.bt = block_table;
  a.cu = cu_seqlens;
  a.ctx = context_lens;
  a.path = path;
  a.counts = counts;
  a.bts[0] = bt_strides[0];
  a.bts[1] = bt_strides[1];
  a.total = (int)total_tokens;
  a.heads = (int)num_heads;
  a.pieces = 128 * bytes / 16;
  a.num_blocks = (int)num_blocks;
  a.max_blocks = (int)max_blocks_per_seq;
  a.err = error_flag;
  const cudaError_t e =
      launch_pdl(keep_kernel, dim3((unsigned)batch, (unsigned)layers), dim3(kMvThreads), 0,
                 static_cast<cudaStream_t>(stream), a);
  return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_keep_accepted launch");
}
