// Host side shared by the entry points over a chunk of new tokens: argument checks and the
// tensor maps over packed query rows and page pools.
#include "chunk_common.cuh"

namespace fi {

int chunk_batch_args(ChunkBatch& p, const char* what, const int32_t* cu, const int32_t* ctx,
                     const int32_t* prefix, const int32_t* bt, int64_t batch, int64_t total,
                     int64_t hq, int64_t hk, int64_t head_dim, int64_t num_blocks,
                     int64_t block_size, int64_t max_blocks, const int64_t* bts, int64_t window,
                     int64_t dtype) {
  if (batch < 0 || total < 0 || hq <= 0 || hk <= 0 || num_blocks <= 0 || max_blocks <= 0 ||
      window < 0)
    return fail(FI_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (dtype != FI_DTYPE_F16 && dtype != FI_DTYPE_BF16)
    return fail(FI_ERR_INVALID_ARG, "%s: unknown dtype %lld", what, (long long)dtype);
  if (head_dim != kChunkTile)
    return fail(FI_ERR_UNSUPPORTED, "%s: head_dim %lld != 128", what, (long long)head_dim);
  if (block_size != kChunkPage)
    return fail(FI_ERR_UNSUPPORTED, "%s: block_size %lld != 64", what, (long long)block_size);
  if (hq % hk != 0)
    return fail(FI_ERR_INVALID_ARG, "%s: num_q_heads %% num_kv_heads != 0", what);
  if (hq / hk > 64)
    return fail(FI_ERR_UNSUPPORTED, "%s: more than 64 query heads per KV head", what);
  if (total > (1 << 28) || hq > 65535 || num_blocks > (1 << 30) || max_blocks > (1 << 20) ||
      batch > (1 << 20))
    return fail(FI_ERR_UNSUPPORTED, "%s: sizes too large", what);
  p.cu = cu;
  p.ctx = ctx;
  p.prefix = prefix;
  p.bt = bt;
  p.bts[0] = bts ? bts[0] : 0;
  p.bts[1] = bts ? bts[1] : 0;
  p.batch = (int)batch;
  p.total = (int)total;
  p.window = (int)(window > (1 << 30) ? 1 << 30 : window);
  p.hq = (int)hq;
  p.hk = (int)hk;
  p.group = (int)(hq / hk);
  p.num_blocks = (int)num_blocks;
  p.max_blocks = (int)max_blocks;
  p.tile_tokens = kChunkTile / p.group;
  return FI_OK;
}

int chunk_score_args(ScoreForm& f, const char* what, float sm_scale, float softcap,
                     const float* slopes) {
  if (!(sm_scale > 0.f) || !isfinite(sm_scale))
    return fail(FI_ERR_INVALID_ARG, "%s: sm_scale must be positive and finite", what);
  if (!(softcap >= 0.f) || !isfinite(softcap))
    return fail(FI_ERR_INVALID_ARG, "%s: softcap must be finite and not negative", what);
  const double log2e = 1.4426950408889634;
  f.scale_log2 = (float)((double)sm_scale * log2e);
  f.cap_in = softcap > 0.f ? (float)((double)sm_scale / (double)softcap) : 0.f;
  f.cap_log2 = (float)((double)softcap * log2e);
  f.slopes = slopes;
  // tanh(u) / u in u^2 on |u| <= 1/3, minimax (2.4e-8 before the coefficients' rounding); where their
  // powers of cap_in could leave fp32's range, no score takes this form
  const double c[4] = {0.9999999763, -0.3333264747, 0.1330220246, -0.04939617807};
  f.tiny_max = -1.f;
  if (f.cap_in > 1e-5f && f.cap_in < 1e4f) {
    const double in = (double)sm_scale / (double)softcap;
    double to = (double)sm_scale * log2e;
    for (int i = 0; i < 4; ++i, to *= in * in) f.tiny[i] = (float)(c[i] * to);
    f.tiny_max = (float)(1.0 / 3.0 / in);
  }
  if (!isfinite(f.cap_in) || !isfinite(f.scale_log2) || !isfinite(f.cap_log2))
    return fail(FI_ERR_INVALID_ARG, "%s: sm_scale or softcap outside what fp32 scores hold", what);
  return FI_OK;
}

int chunk_q_map(CUtensorMap* m, CUtensorMapDataType type, const void* q, const ChunkBatch& p,
                const int64_t* qs, const char* what) {
  if (qs[2] != 1) return fail(FI_ERR_ALIGNMENT, "%s: innermost stride must be 1", what);
  const uint64_t dims[4] = {(uint64_t)kChunkTile, (uint64_t)p.group, (uint64_t)p.hk,
                            (uint64_t)p.total};
  uint64_t sb[3] = {(uint64_t)qs[1] * 2, (uint64_t)qs[1] * 2 * p.group, (uint64_t)qs[0] * 2};
  // A dimension of size 1 is never stepped over; give it any legal stride.
  if (p.hq == 1) sb[0] = sb[1] = (uint64_t)kChunkTile * 2;
  if (p.total == 1) sb[2] = (uint64_t)kChunkTile * 2;
  const uint32_t box[4] = {64, (uint32_t)p.group, 1, (uint32_t)p.tile_tokens};
  return encode_tiled(m, type, 4, q, dims, sb, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

int chunk_kv_map(CUtensorMap* m, CUtensorMapDataType type, const void* kv, const ChunkBatch& p,
                 const int64_t* st, const char* what) {
  if (st[3] != 1) return fail(FI_ERR_ALIGNMENT, "%s: innermost stride must be 1", what);
  const uint64_t dims[4] = {(uint64_t)kChunkTile, (uint64_t)p.hk, (uint64_t)kChunkPage,
                            (uint64_t)p.num_blocks};
  uint64_t sb[3] = {(uint64_t)st[2] * 2, (uint64_t)st[1] * 2, (uint64_t)st[0] * 2};
  if (p.hk == 1) sb[0] = (uint64_t)kChunkTile * 2;
  if (p.num_blocks == 1) sb[2] = (uint64_t)kChunkTile * 2;
  const uint32_t box[4] = {64, 1, (uint32_t)kChunkPage, 1};
  return encode_tiled(m, type, 4, kv, dims, sb, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

int chunk_code_map(CUtensorMap* m, const void* codes, const ChunkBatch& p, const int64_t* st,
                   const char* what) {
  if (st[3] != 1) return fail(FI_ERR_ALIGNMENT, "%s: innermost stride must be 1", what);
  const uint64_t dims[4] = {(uint64_t)kChunkTile, (uint64_t)p.hk, (uint64_t)kChunkPage,
                            (uint64_t)p.num_blocks};
  uint64_t sb[3] = {(uint64_t)st[2], (uint64_t)st[1], (uint64_t)st[0]};
  if (p.hk == 1) sb[0] = (uint64_t)kChunkTile;
  if (p.num_blocks == 1) sb[2] = (uint64_t)kChunkTile;
  const uint32_t box[4] = {(uint32_t)kChunkTile, 1, (uint32_t)kChunkPage, 1};
  // (promoted to 256 bytes, as 16-bit rows are, they bring the next head's along: 612 MB from HBM for 412)
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, codes, dims, sb, box,
                      CU_TENSOR_MAP_SWIZZLE_128B, what, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

}  // namespace fi
