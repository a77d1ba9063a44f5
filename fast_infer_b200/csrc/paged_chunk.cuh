// What the kernels of attention over the paged cache share beside the batch: the parts of a launch's line of work, the
// workspace where they leave parts of units, and the launches between the files.
#pragma once

#include "chunk_common.cuh"

namespace fi {

constexpr int kCkMaxBatch = 2048;    // sequences per launch
constexpr int kCkMaxUnits = 4608;    // token units per launch (per KV head)
constexpr int kCkNarrow = 32;        // rows up to which a unit runs transposed

// The unit whose first part a CTA holds when the rest lies in the next CTAs.
struct CkJoin {
  int valid, last_cta, token, hk, rows[2], pad[2];
};

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
  const float* scale[2];  // of k and v, with 8-bit codes
  int64_t ss[2][3];       // page, head, slot
  int* err;
};

// Key tiles that the unit of tokens [t0, t1) of a sequence visits: [0, np) for the prefix and
// [lo, lo + n - np). A unit that sees nothing visits one (all of it masked).
__device__ __forceinline__ void ck_tiles(const ChunkBatch& p, const ChunkSeq& s, int t0, int t1,
                                         int& np, int& lo, int& n) {
  // (a tree's token may see any new token, and stands at the first new slot or behind it)
  const int p0 = s.pos0 + (p.tree ? 0 : t0), p1 = s.pos0 + t1 - 1;
  const int end = p.tree ? s.keys : min(s.keys, max(p1 + 1, s.prefix));
  const int hi = end > 0 ? (end - 1) / kChunkTile : 0;
  lo = p.window ? min(max(p0 - p.window + 1, 0) / kChunkTile, hi) : 0;
  np = min((s.prefix + kChunkTile - 1) / kChunkTile, lo);
  n = np + hi - lo + 1;
}

// Few-row units over pages of 8-bit codes (paged_codes.cu): what the kernel takes beside ChunkParams.
struct CodePages {
  const void* q;
  const uint8_t* pool[2];  // k, v
  int64_t qs[2];
  int64_t st[2][3];        // page, slot, head
  int stages, max_units;   // (set at the launch)
};
// Rows of a unit there: 8, 16 or 32 (columns of the products).
int launch_narrow_codes(const ChunkParams& p, const CodePages& pages, int64_t dtype,
                        int64_t cache_dtype, int rows, cudaStream_t st);

}  // namespace fi
