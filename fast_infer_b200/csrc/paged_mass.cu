// Attention weight that each cached token receives from the new tokens:
//
//   mass[b, hk, j] (+)= sum over the query rows i of KV head hk of exp(s_ij - lse_i)
//
// (the batch, visibility and score are described in chunk_common.cuh; lse is what the
// attention call over the same tokens returned). It is what an eviction from the cache goes
// by. Reads K once and no V; one product and one exponential per visible (row, key).
//
// Design:
// * The product is transposed, S^T = K Q^T: keys are the 128 tensor-memory lanes, so a thread
//   owns one key and sums over the columns (query rows) in registers: no atomics.
// * A unit is 256 consecutive keys (two tiles) of one sequence and KV head; its steps are the
//   128-row query tiles that see any of them. The launch's line of (KV head, sequence, unit,
//   step) is cut into equal parts, one per CTA; a unit cut between CTAs leaves 256 partial
//   sums each, joined by mass_join_kernel in CTA order (the same bits on every run). One new
//   token per sequence makes it a stream over K; a whole chunk a stream over Q with K resident.
// * What bounds a step of 256 keys x 128 rows is its 32768 exponentials (2048 cycles of the SM's
//   MUFU, against 1024 of the tensor core): 3 of 8 pairs take a polynomial on the FMA pipe.
// * Roles (640 threads): warps 0-15 = the sums, four warpgroups = two key tiles x two halves of
//   the columns (four warps per scheduler, or their latencies would show: eight warps took twice
//   the time), warp 16 = TMA, warp 17 = UMMA issue, warp 18 = the rows' lse (and slopes and
//   positions) into shared memory, warp 19 = scheduler, then zeros where no new token sees.
//   Tensor memory: two S buffers per key tile.
#include "chunk_common.cuh"

namespace fi {

constexpr int kMsThreads = 640;
constexpr int kMsStages = 2;         // K (256 keys) and Q ring slots
constexpr int kMsKeys = 256;         // keys of a unit
constexpr int kMsMaxBatch = 2048;
constexpr int kMsEmuPairs = 3;       // of 8 column pairs, exp2 on the FMA pipe
constexpr int kMsSlots = 4;          // units that the scheduler is ahead
constexpr int kMsParts = 4;          // unit sums of the second column half in flight

// A CTA's part of a unit: query tiles [q0, q1).
struct alignas(16) MsUnit {
  int b, hk, u;
  int q0, q1;
  int start, n, pos0, keys, prefix;
  int many;      // the sequence has more than one query tile: every step loads one
  int fresh;     // first unit of its (sequence, KV head): its step loads the only query tile
  int last;      // last such unit: its step gives it back
  int whole;     // all of the unit's steps are here
  int begins;    // the first of them is
  int pages_ok;  // no block-table entry of its keys is invalid
  int valid, pad[3];
};

struct MsBarriers {
  uint64_t k_full[kMsStages], k_empty[kMsStages];
  uint64_t q_full[kMsStages], q_empty[kMsStages];
  uint64_t s_full[2][2], s_empty[2][2];  // [key tile][buffer]
  uint64_t part_full[2][kMsParts];       // [key tile]
  uint64_t unit_full[kMsSlots], unit_empty[kMsSlots];
  uint64_t mma_done;
  uint64_t seq[kMsMaxBatch + 1];         // steps before each sequence
  uint64_t warp_sums[kMsThreads / 32];
  uint32_t tmem_base;
  MsUnit units[kMsSlots];
  alignas(16) float neg_lse[kMsStages][kChunkTile];  // -lse * log2(e), -inf: no such row
  alignas(16) float slope[kMsStages][kChunkTile];    // distance bias, log2 units
  alignas(16) float pos[kMsStages][kChunkTile];
  float part[2][kMsParts][kChunkTile];   // sums of the second column half
};
constexpr int kMsSmemBytes =
    1024 + kMsStages * 3 * kChunkTileBytes + (int)sizeof(MsBarriers);
static_assert(kMsSmemBytes <= 227 * 1024, "shared memory");

struct MsJoin {
  int valid, last_cta;
  int keys, span;  // values that hold a key, and that mass has room for
  int64_t at;      // first value in mass
};

struct MassParams {
  ChunkBatch b;
  ScoreForm f;
  const float* lse;  // [total, hq]
  float* mass;       // [batch, hk, cap]
  int64_t cap;
  int accumulate;
  float* ws;     // [cta][first, last unit][256]
  MsJoin* join;  // [cta]
  int* err;
};

// Query tiles [a, b) that see any key of unit u.
__device__ __forceinline__ void ms_steps(const ChunkBatch& p, const ChunkSeq& s, int u, int& a,
                                         int& b) {
  const int k0 = u * kMsKeys, k1 = min(k0 + kMsKeys, s.keys) - 1;
  int lo = 0, hi = s.n;
  if (k0 >= s.prefix) {
    lo = max(k0 - s.pos0, 0);
    if (p.window) hi = min(hi, k1 + p.window - s.pos0);
  }
  a = lo / p.tile_tokens;
  b = lo < hi ? (hi - 1) / p.tile_tokens + 1 : a;
}
__device__ __forceinline__ int ms_units(const ChunkSeq& s) {
  return (s.keys + kMsKeys - 1) / kMsKeys;
}

// The scheduler (one warp): walks the CTA's part of the line and hands its units to the other
// roles through a ring in shared memory.
__device__ __forceinline__ void ms_schedule(const ChunkBatch& p, MsBarriers* m, int64_t cap,
                                            MsJoin* join_out, int* err) {
  const int G = gridDim.x, cta = blockIdx.x, lane = threadIdx.x & 31;
  const int64_t per_head = (int64_t)m->seq[p.batch];
  const int64_t total = per_head * p.hk;
  const int active = (int)(total < G ? total : G);
  // total * (cta + 1) stays below 2^63: at most 2^28 rows x 2^18 units x 2^9 CTAs
  int64_t w = cta < active ? total * cta / active : 0;
  const int64_t end = cta < active ? total * (cta + 1) / active : 0;
  int hk = 0, b = 0, u = 0, skip = 0, tiles = 0;  // `skip` steps of unit u are the CTA's before
  ChunkSeq s = {};
  if (w < end) {
    hk = (int)(w / per_head);
    const uint64_t r0 = (uint64_t)(w - hk * per_head);
    b = last_le(m->seq, p.batch, r0);
    s = chunk_seq(p, b);
    uint64_t r = r0 - m->seq[b];
#pragma unroll 1
    for (int base = 0;; base += 32) {  // the unit that holds step r of the sequence
      int a = 0, e = 0;
      if (base + lane < ms_units(s)) ms_steps(p, s, base + lane, a, e);
      uint64_t inc = (uint64_t)(e - a);
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint64_t v = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += v;
      }
      const uint64_t sum = __shfl_sync(0xffffffffu, inc, 31);
      if (sum > r) {
        const int i = __ffs(__ballot_sync(0xffffffffu, inc > r)) - 1;
        u = base + i;
        skip = (int)(r - __shfl_sync(0xffffffffu, inc - (uint64_t)(e - a), i));
        break;
      }
      r -= sum;
    }
    tiles = (s.n + p.tile_tokens - 1) / p.tile_tokens;
  }
  bool fresh = true;
  MsJoin join = {};
#pragma unroll 1
  for (int i = 0;; ++i) {
    const int slot = i % kMsSlots;
    if (i >= kMsSlots &&
        !__all_sync(0xffffffffu, mbar_wait(&m->unit_empty[slot], ((i / kMsSlots) - 1) & 1, err)))
      break;
    MsUnit v = {};
    bool pages_ok = true;
    v.valid = w < end;
    if (v.valid) {
      int a, e;
      while (true) {  // the line holds only units with steps
        ms_steps(p, s, u, a, e);
        if (e > a) break;
        ++u;
      }
      const int n = e - a;
      v.q0 = a + skip;
      v.q1 = (int)(e - v.q0 <= end - w ? e : v.q0 + (end - w));
      v.b = b;
      v.hk = hk;
      v.u = u;
      v.start = s.start;
      v.n = s.n;
      v.pos0 = s.pos0;
      v.keys = s.keys;
      v.prefix = s.prefix;
      v.many = tiles > 1;
      v.fresh = fresh;
      v.begins = skip == 0;
      v.whole = v.begins && v.q1 == e;
      if (lane < 4 && (u * 4 + lane) * kChunkPage < s.keys)
        pages_ok = chunk_page(p, b, s.keys, u * 2 + (lane >> 1), lane & 1) != p.num_blocks;
      if (v.begins && !v.whole) {  // it goes on in the next CTA: the last one here
        const int64_t keys = min((int64_t)s.keys, cap);
        join.valid = 1;
        join.last_cta = (int)(((w + n) * active - 1) / total);
        join.keys = (int)min(keys - u * (int64_t)kMsKeys, (int64_t)kMsKeys);
        join.span = (int)min(cap - u * (int64_t)kMsKeys, (int64_t)kMsKeys);
        join.at = ((int64_t)b * p.hk + hk) * cap + u * (int64_t)kMsKeys;
      }
      w += v.q1 - v.q0;
      skip = 0;
      ++u;
      const bool leave = w >= end || w - hk * per_head >= (int64_t)m->seq[b + 1];
      v.last = leave;
      fresh = leave;
      if (leave && w < end) {
        hk = (int)(w / per_head);
        b = last_le(m->seq, p.batch, (uint64_t)(w - hk * per_head));
        s = chunk_seq(p, b);
        tiles = (s.n + p.tile_tokens - 1) / p.tile_tokens;
        u = 0;
      }
    }
    v.pages_ok = __all_sync(0xffffffffu, pages_ok);
    if (lane == 0) {
      m->units[slot] = v;
      mbar_arrive(&m->unit_full[slot]);  // released to the waits that read it
    }
    if (!v.valid) break;
  }
  if (lane == 0) *join_out = join;
}

// The next unit of the ring, null when none is left; it stays in shared memory until ms_done.
template <bool kWarp>
__device__ __forceinline__ const MsUnit* ms_next(MsBarriers* m, int i, int* err) {
  const int slot = i % kMsSlots;
  bool ok = mbar_wait(&m->unit_full[slot], (i / kMsSlots) & 1, err);
  if (kWarp) ok = __all_sync(0xffffffffu, ok);
  return ok && m->units[slot].valid ? &m->units[slot] : nullptr;
}
template <bool kWarp>
__device__ __forceinline__ void ms_done(MsBarriers* m, int& i) {
  if (kWarp) __syncwarp();
  if (!kWarp || (threadIdx.x & 31) == 0) mbar_arrive(&m->unit_empty[i % kMsSlots]);
  ++i;
}
// Whether step q loads a query tile, and is the last one on it: a sequence with one query tile
// keeps it for all of its units.
__device__ __forceinline__ bool ms_loads(const MsUnit& u) { return u.many || u.fresh; }
__device__ __forceinline__ bool ms_frees(const MsUnit& u) { return u.many || u.last; }

template <typename T, bool kCap, bool kAlibi>
__global__ void __launch_bounds__(kMsThreads, 1)
    paged_mass_kernel(const __grid_constant__ CUtensorMap tm_q,
                      const __grid_constant__ CUtensorMap tm_k, const MassParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align1024(smem_raw);
  uint8_t* sK = smem;                                      // [stage][2 tiles]
  uint8_t* sQ = smem + kMsStages * 2 * kChunkTileBytes;    // [stage]
  MsBarriers* bars = reinterpret_cast<MsBarriers*>(sQ + kMsStages * kChunkTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  const ChunkBatch& pb = p.b;
  const int tile_rows = pb.tile_tokens * pb.group;

  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < kMsStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->q_full[s], 2);    // TMA, warp 18
      mbar_init(&bars->q_empty[s], 17);  // UMMA, the 16 summing warps
    }
    for (int t = 0; t < 2; ++t) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars->s_full[t][i], 1);
        mbar_init(&bars->s_empty[t][i], 8);
      }
      for (int i = 0; i < kMsParts; ++i) mbar_init(&bars->part_full[t][i], 4);
    }
    for (int i = 0; i < kMsSlots; ++i) {
      mbar_init(&bars->unit_full[i], 1);
      mbar_init(&bars->unit_empty[i], 19);  // TMA, UMMA, warp 18, the 16 summing warps
    }
    mbar_init(&bars->mma_done, 1);
    fence_barrier_init();
  }
  // Query rows that TMA never writes: zeros, so that their columns hold finite scores.
#pragma unroll 1
  for (int i = threadIdx.x; i < kMsStages * 2 * (kChunkTile - tile_rows) * 8; i += kMsThreads) {
    const int part = i / ((kChunkTile - tile_rows) * 8), k = i % ((kChunkTile - tile_rows) * 8);
    *reinterpret_cast<uint4*>(sQ + part * kChunkHalf + tile_rows * 128 + k * 16) =
        make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();

  grid_dep_wait();
  grid_dep_launch();
  // Steps of every sequence, a warp each, then their sums.
  if (threadIdx.x == 0) bars->seq[0] = 0;
#pragma unroll 1
  for (int b = warp; b < pb.batch; b += kMsThreads / 32) {
    const ChunkSeq s = chunk_seq(pb, b);
    if (lane == 0 && cta == 0 && (s.bad || s.keys > p.cap)) set_error(p.err, FI_DEVERR_CONTEXT_LEN);
    uint64_t steps = 0;
    if (s.n > 0) {
#pragma unroll 1
      for (int u = lane; u < ms_units(s); u += 32) {
        int a, e;
        ms_steps(pb, s, u, a, e);
        steps += e - a;
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) steps += __shfl_xor_sync(0xffffffffu, steps, off);
    if (lane == 0) bars->seq[b + 1] = steps;
  }
  __syncthreads();
  block_scan(bars->seq, pb.batch, bars->warp_sums);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == 16) {
    if (lane == 0) {
      // ---------------------------------------------------------- TMA producer
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_k);
      int kc = 0, qc = 0, next_unit = 0;
      bool ok = true;
#pragma unroll 1
      for (const MsUnit* up; ok && (up = ms_next<false>(bars, next_unit, p.err)) != nullptr;
           ms_done<false>(bars, next_unit)) {
        const MsUnit& u = *up;
        int ph[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ph[i] = chunk_page(pb, u.b, u.keys, u.u * 2 + (i >> 1), i & 1);
          if (ph[i] == pb.num_blocks && (u.u * 4 + i) * kChunkPage < u.keys)
            set_error(p.err, FI_DEVERR_BAD_BLOCK);
        }
        const int ks = kc % kMsStages;
        if (kc >= kMsStages && !(ok = mbar_wait(&bars->k_empty[ks], ((kc / kMsStages) - 1) & 1, p.err)))
          break;
        ++kc;
        mbar_arrive_expect_tx(&bars->k_full[ks], 2 * kChunkTileBytes);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint8_t* dst = sK + (ks * 2 + (i >> 1)) * kChunkTileBytes + (i & 1) * (kChunkHalf / 2);
          tma_load_4d(dst, &tm_k, &bars->k_full[ks], 0, u.hk, 0, ph[i]);
          tma_load_4d(dst + kChunkHalf, &tm_k, &bars->k_full[ks], 64, u.hk, 0, ph[i]);
        }
        if (!ms_loads(u)) continue;
#pragma unroll 1
        for (int q = u.q0; q < u.q1; ++q) {
          const int qs = qc % kMsStages;
          if (qc >= kMsStages && !(ok = mbar_wait(&bars->q_empty[qs], ((qc / kMsStages) - 1) & 1, p.err)))
            break;
          ++qc;
          const int token = u.start + q * pb.tile_tokens;
          uint8_t* dst = sQ + qs * kChunkTileBytes;
          mbar_arrive_expect_tx(&bars->q_full[qs], (uint32_t)(tile_rows * 256));
          tma_load_4d(dst, &tm_q, &bars->q_full[qs], 0, 0, u.hk, token);
          tma_load_4d(dst + kChunkHalf, &tm_q, &bars->q_full[qs], 64, 0, u.hk, token);
        }
      }
    }
  } else if (warp == 17) {
    if (lane == 0) {
      // ---------------------------------------------------------- UMMA issuer
      const uint32_t k_addr = smem_u32(sK), q_addr = smem_u32(sQ);
      int kc = 0, qc = 0, sc = 0, next_unit = 0;
      bool ok = true;
#pragma unroll 1
      for (const MsUnit* up; ok && (up = ms_next<false>(bars, next_unit, p.err)) != nullptr;
           ms_done<false>(bars, next_unit)) {
        const MsUnit& u = *up;
        const int ks = kc % kMsStages;
        if (!(ok = mbar_wait(&bars->k_full[ks], (kc / kMsStages) & 1, p.err))) break;
        ++kc;
#pragma unroll 1
        for (int q = u.q0; q < u.q1; ++q, ++sc) {
          if (ms_loads(u)) {
            if (!(ok = mbar_wait(&bars->q_full[qc % kMsStages], (qc / kMsStages) & 1, p.err))) break;
            ++qc;
          }
          const int qs = (qc - 1) % kMsStages, buf = sc & 1;
          const int rows = min(u.n - q * pb.tile_tokens, pb.tile_tokens) * pb.group;
          const uint32_t idesc = umma_idesc<T>(128, (uint32_t)(rows + 15) / 16 * 16, 0, 0);
          const uint64_t db = umma_desc_sw128(q_addr + qs * kChunkTileBytes, 16, 1024);
#pragma unroll 1
          for (int t = 0; t < 2 && ok; ++t) {
            if (sc >= 2) ok = mbar_wait(&bars->s_empty[t][buf], ((sc >> 1) - 1) & 1, p.err);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = umma_desc_sw128(k_addr + (ks * 2 + t) * kChunkTileBytes, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t off = ((kk >> 2) * kChunkHalf + (kk & 3) * 32) >> 4;
              umma_ss(tmem + (t * 2 + buf) * 128, da + off, db + off, idesc, kk > 0);
            }
            umma_commit(&bars->s_full[t][buf]);
          }
          if (!ok) break;
          if (ms_frees(u)) umma_commit(&bars->q_empty[qs]);
        }
        if (!ok) break;
        umma_commit(&bars->k_empty[ks]);
      }
      umma_commit(&bars->mma_done);
      mbar_wait(&bars->mma_done, 0, p.err);
    }
  } else if (warp == 18) {
    // -------------------------------------------------- the rows' lse, a column each
    int qc = 0, next_unit = 0;
    bool ok = true;
#pragma unroll 1
    for (const MsUnit* up; ok && (up = ms_next<true>(bars, next_unit, p.err)) != nullptr;
         ms_done<true>(bars, next_unit)) {
      const MsUnit& u = *up;
      if (!ms_loads(u)) continue;
#pragma unroll 1
      for (int q = u.q0; ok && q < u.q1; ++q) {
        const int qs = qc % kMsStages;
        float nl[4], sl[4], ps[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = lane + 32 * i, tok = q * pb.tile_tokens + c / pb.group;
          const int head = u.hk * pb.group + c % pb.group;
          nl[i] = -INFINITY;
          sl[i] = ps[i] = 0.f;
          if (c < tile_rows && tok < u.n) {
            const float v = p.lse[(int64_t)(u.start + tok) * pb.hq + head];
            if (v != -INFINITY) nl[i] = -v * kLog2e;
            if (kAlibi) {
              sl[i] = p.f.slopes[head] * kLog2e;
              ps[i] = (float)(u.pos0 + tok);
            }
          }
        }
        if (qc >= kMsStages)
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&bars->q_empty[qs], ((qc / kMsStages) - 1) & 1, p.err));
        if (!ok) break;
        ++qc;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bars->neg_lse[qs][lane + 32 * i] = nl[i];
          if (kAlibi) {
            bars->slope[qs][lane + 32 * i] = sl[i];
            bars->pos[qs][lane + 32 * i] = ps[i];
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->q_full[qs]);
      }
    }
  } else if (warp == 19) {
    ms_schedule(pb, bars, p.cap, p.join + cta, p.err);
    // zeros where no new token sees (unless the call adds to mass)
    if (!p.accumulate) {
#pragma unroll 1
      for (int64_t r = cta; r < (int64_t)pb.batch * pb.hk; r += gridDim.x) {
        const ChunkSeq s = chunk_seq(pb, (int)(r / pb.hk));
        float* row = p.mass + r * p.cap;
#pragma unroll 1
        for (int64_t k0 = 0; k0 < p.cap; k0 += kMsKeys) {
          int a = 0, e = 0;
          if (s.n > 0 && k0 < s.keys) ms_steps(pb, s, (int)(k0 / kMsKeys), a, e);
          if (e > a) continue;
          for (int64_t j = k0 + lane; j < k0 + kMsKeys && j < p.cap; j += 32) row[j] = 0.f;
        }
      }
    }
  } else {
    // ------------------------------------------------------------- sums, warps 0-15
    const int t = warp >> 3, second = (warp >> 2) & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t tS = tmem + ((uint32_t)(quarter * 32) << 16) + t * 256;
    const uint64_t sc2 = f32x2(p.f.scale_log2, p.f.scale_log2);
    int sc = 0, qc = 0, next_unit = 0;
    // false once a wait ran out; the warp then goes on without waiting, its sums no longer count
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err));
    };
#pragma unroll 1
    for (const MsUnit* up; (up = ms_next<true>(bars, next_unit, p.err)) != nullptr;
         ms_done<true>(bars, next_unit)) {
      const MsUnit& u = *up;
      const int key = u.u * kMsKeys + t * kChunkTile + row;
      const bool page_ok = u.pages_ok || chunk_page(pb, u.b, u.keys, u.u * 2 + t, row >> 6) !=
                                             pb.num_blocks;
      float acc = 0.f;
#pragma unroll 1
      for (int q = u.q0; q < u.q1; ++q, ++sc) {
        const bool loads = ms_loads(u);
        if (loads) ++qc;
        const int qs = (qc - 1) % kMsStages, buf = sc & 1;
        // columns [c_lo, c_hi) see this key
        const int tok0 = q * pb.tile_tokens;
        const int rows = min(u.n - tok0, pb.tile_tokens) * pb.group;
        int c_lo = 0, c_hi = rows;
        if (key >= u.prefix) {
          c_lo = min(max(key - u.pos0 - tok0, 0), kChunkTile) * pb.group;
          if (pb.window)
            c_hi = min(rows, min(max(key + pb.window - u.pos0 - tok0, 0), kChunkTile) * pb.group);
        }
        if (!page_ok) c_hi = 0;
        // this warpgroup's columns: one half, in 16s
        const int cols = (rows + 15) / 16 * 16, mid = (cols / 2 + 15) / 16 * 16;
        const int c0 = second ? mid : 0, c1 = second ? cols : mid;
        if (loads) wait(&bars->q_full[qs], ((qc - 1) / kMsStages) & 1);
        wait(&bars->s_full[t][buf], (sc >> 1) & 1);
        tc_fence_after();
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll 1
        for (int cc = c0; cc < c1; cc += 16) {
          uint32_t raw[16];
          tmem_ld16(tS + buf * 128 + cc, raw);
          const float4* nl4 = reinterpret_cast<const float4*>(&bars->neg_lse[qs][cc]);
          uint64_t x[8];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float4 v = nl4[c];
            x[2 * c] = f32x2(v.x, v.y);
            x[2 * c + 1] = f32x2(v.z, v.w);
          }
          if constexpr (kAlibi) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float4 sl = reinterpret_cast<const float4*>(&bars->slope[qs][cc])[c];
              const float4 ps = reinterpret_cast<const float4*>(&bars->pos[qs][cc])[c];
              const float k = (float)key;
              x[2 * c] = add_f32x2(x[2 * c], f32x2(-sl.x * fabsf(k - ps.x), -sl.y * fabsf(k - ps.y)));
              x[2 * c + 1] =
                  add_f32x2(x[2 * c + 1], f32x2(-sl.z * fabsf(k - ps.z), -sl.w * fabsf(k - ps.w)));
            }
          }
          tmem_wait_ld();
          reg_fence<16>(raw);
          if constexpr (kCap) {
            const uint64_t cin = f32x2(p.f.cap_in, p.f.cap_in);
            const uint64_t cout = f32x2(p.f.cap_log2, p.f.cap_log2);
            float big = 0.f;
#pragma unroll
            for (int c = 0; c < 16; c += 2)
              big = fmax3f(big, fabsf(__uint_as_float(raw[c])), fabsf(__uint_as_float(raw[c + 1])));
            const bool small = __all_sync(0xffffffffu, big * p.f.cap_in <= 1.f);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint64_t v = mul_f32x2(
                  f32x2(__uint_as_float(raw[2 * c]), __uint_as_float(raw[2 * c + 1])), cin);
              uint64_t y = tanh_poly_x2(v);
              if (!small) {
                float v0, v1, y0, y1;
                f32x2_split(v, v0, v1);
                f32x2_split(y, y0, y1);
                y = f32x2(fabsf(v0) <= 1.f ? y0 : tanh_any(v0), fabsf(v1) <= 1.f ? y1 : tanh_any(v1));
              }
              x[c] = fma_f32x2(y, cout, x[c]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              x[c] = fma_f32x2(f32x2(__uint_as_float(raw[2 * c]), __uint_as_float(raw[2 * c + 1])),
                               sc2, x[c]);
          }
          if (!__all_sync(0xffffffffu, c_lo <= cc && c_hi >= min(cc + 16, tile_rows))) {
            const uint32_t vis = low_bits(c_hi - cc, 0) & ~low_bits(c_lo - cc, 0);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              float a, b;
              f32x2_split(x[c], a, b);
              x[c] = f32x2((vis >> (2 * c)) & 1u ? a : -INFINITY,
                           (vis >> (2 * c + 1)) & 1u ? b : -INFINITY);
            }
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint64_t e;
            if (c < kMsEmuPairs) {
              e = exp2_poly5_x2(x[c]);
            } else {
              float a, b;
              f32x2_split(x[c], a, b);
              e = f32x2(fast_exp2(a), fast_exp2(b));
            }
            sum2[c & 1] = add_f32x2(sum2[c & 1], e);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars->s_empty[t][buf]);
          if (ms_frees(u)) mbar_arrive(&bars->q_empty[qs]);
        }
        float s0, s1;
        f32x2_split(add_f32x2(sum2[0], sum2[1]), s0, s1);
        acc += s0 + s1;
      }
      // The second half's sum goes to the first half's warp through shared memory. A slot is
      // free again kMsParts units later: the S buffers keep the halves within two steps, and so
      // within two units, of each other.
      const int slot = next_unit % kMsParts;
      if (second) {
        bars->part[t][slot][row] = acc;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->part_full[t][slot]);
        continue;
      }
      wait(&bars->part_full[t][slot], (next_unit / kMsParts) & 1);
      acc += bars->part[t][slot][row];
      if (u.whole) {
        const int64_t keys = min((int64_t)u.keys, p.cap);
        float* dst = p.mass + ((int64_t)u.b * pb.hk + u.hk) * p.cap + key;
        if (p.accumulate) {
          if (key < keys) *dst += acc;
        } else if (key < p.cap) {
          *dst = key < keys ? acc : 0.f;
        }
      } else {
        p.ws[(cta * 2 + (u.begins ? 1 : 0)) * (int64_t)kMsKeys + t * kChunkTile + row] = acc;
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The sums of a unit that several CTAs hold, added in CTA order. A thread per key.
__global__ void __launch_bounds__(kMsKeys) mass_join_kernel(const MassParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const int cta = blockIdx.x, i = threadIdx.x;
  const MsJoin jn = p.join[cta];
  if (!jn.valid || i >= jn.span) return;
  float sum = 0.f;
  for (int c = cta; c <= jn.last_cta; ++c)
    sum += p.ws[(c * 2 + (c == cta ? 1 : 0)) * (int64_t)kMsKeys + i];
  float* dst = p.mass + jn.at + i;
  if (p.accumulate) {
    if (i < jn.keys) *dst += sum;
  } else {
    *dst = i < jn.keys ? sum : 0.f;
  }
}

template <typename T, bool kCap, bool kAlibi>
static int launch_mass(const CUtensorMap& tq, const CUtensorMap& tk, const MassParams& p,
                       cudaStream_t st) {
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(paged_mass_kernel<T, kCap, kAlibi>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, kMsSmemBytes);
  });
  if (e != cudaSuccess) return cuda_fail(e, "fi_attention_mass: cudaFuncSetAttribute");
  const int grid = sm_count();
  e = launch_pdl(paged_mass_kernel<T, kCap, kAlibi>, dim3((unsigned)grid), dim3(kMsThreads),
                 kMsSmemBytes, st, tq, tk, p);
  if (e != cudaSuccess) return cuda_fail(e, "fi_attention_mass: launch");
  e = launch_pdl(mass_join_kernel, dim3((unsigned)grid), dim3(kMsKeys), 0, st, p);
  if (e != cudaSuccess) return cuda_fail(e, "fi_attention_mass: join launch");
  return FI_OK;
}

template <typename T>
static int launch_mass_form(const CUtensorMap& tq, const CUtensorMap& tk, const MassParams& p,
                            bool cap, cudaStream_t st) {
  if (cap)
    return p.f.slopes ? launch_mass<T, true, true>(tq, tk, p, st)
                      : launch_mass<T, true, false>(tq, tk, p, st);
  return p.f.slopes ? launch_mass<T, false, true>(tq, tk, p, st)
                    : launch_mass<T, false, false>(tq, tk, p, st);
}

}  // namespace fi

extern "C" size_t fi_attention_mass_workspace_size(void) {
  using namespace fi;
  return (size_t)sm_count() * (2 * kMsKeys * sizeof(float) + sizeof(MsJoin));
}

extern "C" int fi_attention_mass(const void* q, const void* k_cache, const float* lse, float* mass,
                                 const int32_t* block_table, const int32_t* cu_seqlens,
                                 const int32_t* context_lens, const int32_t* prefix_lens,
                                 const float* alibi_slopes, int64_t batch, int64_t total_tokens,
                                 int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                 int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq,
                                 const int64_t* q_strides, const int64_t* kc_strides,
                                 const int64_t* bt_strides, int64_t mass_capacity,
                                 int64_t accumulate, float sm_scale, float softcap, int64_t window,
                                 int64_t dtype, void* workspace, size_t workspace_bytes,
                                 int32_t* error_flag, void* stream) {
  using namespace fi;
  clear_error();
  const char* what = "fi_attention_mass";
  MassParams p = {};
  int r = chunk_batch_args(p.b, what, cu_seqlens, context_lens, prefix_lens, block_table, batch,
                           total_tokens, num_q_heads, num_kv_heads, head_dim, num_blocks,
                           block_size, max_blocks_per_seq, bt_strides, window, dtype);
  if (r != FI_OK) return r;
  r = chunk_score_args(p.f, what, sm_scale, softcap, alibi_slopes);
  if (r != FI_OK) return r;
  if (mass_capacity < 0) return fail(FI_ERR_INVALID_ARG, "fi_attention_mass: bad sizes");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (batch == 0 || mass_capacity == 0) return FI_OK;
  if (!mass) return fail(FI_ERR_INVALID_ARG, "fi_attention_mass: null pointer argument");
  if (total_tokens == 0) {  // no rows: nothing to add
    if (accumulate) return FI_OK;
    const cudaError_t e = cudaMemsetAsync(
        mass, 0, (size_t)(batch * num_kv_heads * mass_capacity) * sizeof(float), st);
    return e == cudaSuccess ? FI_OK : cuda_fail(e, "fi_attention_mass: memset");
  }
  if (!q || !k_cache || !lse || !block_table || !cu_seqlens || !context_lens || !q_strides ||
      !kc_strides || !bt_strides)
    return fail(FI_ERR_INVALID_ARG, "fi_attention_mass: null pointer argument");
  if (batch > kMsMaxBatch)
    return fail(FI_ERR_UNSUPPORTED, "fi_attention_mass: at most %d sequences; split the batch",
                kMsMaxBatch);
  const size_t need = fi_attention_mass_workspace_size();
  if (!workspace || workspace_bytes < need)
    return fail(FI_ERR_WORKSPACE, "fi_attention_mass: workspace of %zu bytes, needs %zu",
                workspace ? workspace_bytes : (size_t)0, need);
  if (!aligned16(workspace))
    return fail(FI_ERR_ALIGNMENT, "fi_attention_mass: workspace not 16-byte aligned");
  const CUtensorMapDataType type = dtype == FI_DTYPE_F16 ? Half16<__half>::kTmap
                                                         : Half16<__nv_bfloat16>::kTmap;
  CUtensorMap tq, tk;
  if ((r = chunk_q_map(&tq, type, q, p.b, q_strides, "fi_attention_mass q")) != FI_OK) return r;
  if ((r = chunk_kv_map(&tk, type, k_cache, p.b, kc_strides, "fi_attention_mass k_cache")) != FI_OK)
    return r;
  p.lse = lse;
  p.mass = mass;
  p.cap = mass_capacity;
  p.accumulate = accumulate != 0;
  p.ws = static_cast<float*>(workspace);
  p.join = reinterpret_cast<MsJoin*>(p.ws + (size_t)sm_count() * 2 * kMsKeys);
  p.err = error_flag;
  return dtype == FI_DTYPE_F16 ? launch_mass_form<__half>(tq, tk, p, softcap > 0.f, st)
                               : launch_mass_form<__nv_bfloat16>(tq, tk, p, softcap > 0.f, st);
}
