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
// * A unit is 512 consecutive keys (four tiles) of one sequence and KV head, 256 where sequences
//   have few new tokens; its steps are the 128-row query tiles that see any of them. The
//   launch's line of (KV head, sequence, unit, step) is cut into equal parts, one per CTA; a unit
//   cut between CTAs leaves a partial sum per key each, joined by mass_join_kernel in CTA order
//   (the same bits on every run). One new token per sequence makes it a stream over K, each
//   tile reloaded as soon as its product is done; a whole chunk a stream over Q with K resident.
// * What bounds a chunk's step of 512 keys x 128 rows: its 65536 exponentials (4096 cycles of the
//   SM's MUFU, against 2048 of the tensor core), of which some run as a polynomial on the FMA
//   pipe, and the query tile's 32 KB from L2 (units of 256 keys read 6.3 TB/s of them on the
//   whole GPU and were bound by that). 2048 tokens over 30011: 482 us, 811 TFLOP/s, in a burst of
//   10 ms; repeated for seconds 516 us at the 1.84 GHz that the power cap leaves. Single tokens of 16
//   sequences over 1000 to 4095: 22 us, 3.3 TB/s (8 us of it start and drain).
// * Roles (640 threads): warps 0-15 = the sums, a warpgroup per key tile (one per warp scheduler
//   would show its latencies: eight warps took twice the time), warp 16 = TMA, warp 17 = UMMA
//   issue, warp 18 = the rows' lse (and slopes and positions) into shared memory, warp 19 =
//   scheduler, then zeros where no new token sees. Tensor memory: S of each key tile.
#include "chunk_common.cuh"

namespace fi {

constexpr int kMsThreads = 640;
constexpr int kMsTiles = 4;          // key tiles in shared memory, a warpgroup each
constexpr int kMsKeys = kMsTiles * kChunkTile;  // most keys of a unit
constexpr int kMsQ = 2;              // ring slots of query tiles
constexpr int kMsMaxBatch = 2048;
constexpr int kMsEmu = 2;            // of 16 columns, exp2 on the FMA pipe
constexpr int kMsRows = 4;           // ring slots of the rows' lse
constexpr int kMsSlots = 4;          // units that the scheduler is ahead

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
  uint64_t k_full[kMsTiles], k_empty[kMsTiles];
  uint64_t q_full[kMsQ], q_empty[kMsQ];
  uint64_t l_full[kMsRows], l_empty[kMsRows];
  uint64_t s_full[kMsTiles], s_empty[kMsTiles];
  uint64_t unit_full[kMsSlots], unit_empty[kMsSlots];
  uint64_t mma_done;
  uint64_t seq[kMsMaxBatch + 1];         // steps before each sequence
  uint64_t warp_sums[kMsThreads / 32];
  uint32_t tmem_base;
  MsUnit units[kMsSlots];
  alignas(16) float neg_lse[kMsRows][kChunkTile];  // -lse * log2(e), -inf: no such row
  alignas(16) float slope[kMsRows][kChunkTile];    // distance bias, log2 units
  alignas(16) float pos[kMsRows][kChunkTile];
};
constexpr int kMsSmemBytes =
    1024 + (kMsTiles + kMsQ) * kChunkTileBytes + (int)sizeof(MsBarriers);
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
  float* ws;     // [cta][first, last unit][kMsKeys]
  MsJoin* join;  // [cta]
  int tiles;     // key tiles of a unit: 4, or 2
  int* err;
};

// Query tiles [a, b) that see any key of unit u.
__device__ __forceinline__ void ms_steps(const ChunkBatch& p, const ChunkSeq& s, int keys, int u,
                                         int& a, int& b) {
  const int k0 = u * keys, k1 = min(k0 + keys, s.keys) - 1;
  int lo = 0, hi = s.n;
  if (k0 >= s.prefix) {
    lo = max(k0 - s.pos0, 0);
    if (p.window) hi = min(hi, k1 + p.window - s.pos0);
  }
  a = lo / p.tile_tokens;
  b = lo < hi ? (hi - 1) / p.tile_tokens + 1 : a;
}
__device__ __forceinline__ int ms_units(const ChunkSeq& s, int keys) {
  return (s.keys + keys - 1) / keys;
}

// Place in a ring of mbarriers: a slot and the parity of its current phase. The side that fills
// waits for parity ^ 1, which a fresh barrier has passed.
struct MsRing {
  int i = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int n) {
    if (++i == n) {
      i = 0;
      parity ^= 1;
    }
  }
};

// The scheduler (one warp): walks the CTA's part of the line and hands its units to the other
// roles through a ring in shared memory.
__device__ __forceinline__ void ms_schedule(const ChunkBatch& p, MsBarriers* m, int ktiles,
                                            int64_t cap, MsJoin* join_out, int* err) {
  const int ukeys = ktiles * kChunkTile;
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
    for (int base = 0; base < ms_units(s, ukeys); base += 32) {  // the unit of step r
      int a = 0, e = 0;
      if (base + lane < ms_units(s, ukeys)) ms_steps(p, s, ukeys, base + lane, a, e);
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
      int a = 0, e = 0;
      for (; u < ms_units(s, ukeys); ++u) {  // the line holds only units with steps
        ms_steps(p, s, ukeys, u, a, e);
        if (e > a) break;
      }
      const int n = max(e - a, 1);  // (1: lengths changed meanwhile; the walk ends all the same)
      e = a + n;
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
      if (lane < 2 * ktiles && (u * 2 * ktiles + lane) * kChunkPage < s.keys)
        pages_ok = chunk_page(p, b, s.keys, u * ktiles + (lane >> 1), lane & 1) != p.num_blocks;
      if (v.begins && !v.whole) {  // it goes on in the next CTA: the last one here
        const int64_t keys = min((int64_t)s.keys, cap);
        join.valid = 1;
        join.last_cta = (int)(((w + n) * active - 1) / total);
        join.keys = (int)min(keys - u * (int64_t)ukeys, (int64_t)ukeys);
        join.span = (int)min(cap - u * (int64_t)ukeys, (int64_t)ukeys);
        join.at = ((int64_t)b * p.hk + hk) * cap + u * (int64_t)ukeys;
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
  uint8_t* sK = smem;                                // [tile]
  uint8_t* sQ = smem + kMsTiles * kChunkTileBytes;   // [slot]
  MsBarriers* bars = reinterpret_cast<MsBarriers*>(sQ + kMsQ * kChunkTileBytes);
  const int ktiles = p.tiles, ukeys = ktiles * kChunkTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  const ChunkBatch& pb = p.b;
  const int tile_rows = pb.tile_tokens * pb.group;

  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < kMsTiles; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->s_full[s], 1);
      mbar_init(&bars->s_empty[s], 4);
    }
    for (int s = 0; s < kMsQ; ++s) {
      mbar_init(&bars->q_full[s], 1);
      mbar_init(&bars->q_empty[s], 1);
    }
    for (int s = 0; s < kMsRows; ++s) {
      mbar_init(&bars->l_full[s], 1);
      mbar_init(&bars->l_empty[s], 16);
    }
    for (int i = 0; i < kMsSlots; ++i) {
      mbar_init(&bars->unit_full[i], 1);
      mbar_init(&bars->unit_empty[i], 19);  // TMA, UMMA, warp 18, the 16 summing warps
    }
    mbar_init(&bars->mma_done, 1);
    fence_barrier_init();
  }
  // Query rows that TMA never writes: zeros, so that their columns hold 0 for every finite key.
#pragma unroll 1
  for (int i = threadIdx.x; i < kMsQ * 2 * (kChunkTile - tile_rows) * 8; i += kMsThreads) {
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
      for (int u = lane; u < ms_units(s, ukeys); u += 32) {
        int a, e;
        ms_steps(pb, s, ukeys, u, a, e);
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
      int tile = 0, next_unit = 0;  // key tiles loaded: tile i goes to slot i % kMsTiles
      uint32_t k_parity = 1;        // of the slots' current round
      MsRing qr;
      bool ok = true;
#pragma unroll 1
      for (const MsUnit* up; ok && (up = ms_next<false>(bars, next_unit, p.err)) != nullptr;
           ms_done<false>(bars, next_unit)) {
        const MsUnit& u = *up;
        const bool loads = ms_loads(u);
        auto load_q = [&](int q) {
          const int qs = qr.i;
          if (!(ok = mbar_wait(&bars->q_empty[qs], qr.parity ^ 1, p.err))) return;
          qr.next(kMsQ);
          const int token = u.start + q * pb.tile_tokens;
          uint8_t* dst = sQ + qs * kChunkTileBytes;
          mbar_arrive_expect_tx(&bars->q_full[qs], (uint32_t)(tile_rows * 256));
          tma_load_4d(dst, &tm_q, &bars->q_full[qs], 0, 0, u.hk, token);
          tma_load_4d(dst + kChunkHalf, &tm_q, &bars->q_full[qs], 64, 0, u.hk, token);
        };
#pragma unroll 1
        for (int t = 0; ok && t < ktiles; ++t) {
          int ph[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ph[i] = chunk_page(pb, u.b, u.keys, u.u * ktiles + t, i);
            if (ph[i] == pb.num_blocks && ((u.u * ktiles + t) * 2 + i) * kChunkPage < u.keys)
              set_error(p.err, FI_DEVERR_BAD_BLOCK);
          }
          const int slot = tile % kMsTiles;
          if (!(ok = mbar_wait(&bars->k_empty[slot], k_parity, p.err))) break;
          if (++tile % kMsTiles == 0) k_parity ^= 1;
          mbar_arrive_expect_tx(&bars->k_full[slot], kChunkTileBytes);
          uint8_t* dst = sK + slot * kChunkTileBytes;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            tma_load_4d(dst + i * (kChunkHalf / 2), &tm_k, &bars->k_full[slot], 0, u.hk, 0, ph[i]);
            tma_load_4d(dst + kChunkHalf + i * (kChunkHalf / 2), &tm_k, &bars->k_full[slot], 64,
                        u.hk, 0, ph[i]);
          }
          // the first query tile goes out behind the first key tile: the slots of the others may
          // have to wait for the unit before
          if (t == 0 && loads) load_q(u.q0);
        }
        if (!loads) continue;
#pragma unroll 1
        for (int q = u.q0 + 1; ok && q < u.q1; ++q) load_q(q);
      }
    }
  } else if (warp == 17) {
    if (lane == 0) {
      // ---------------------------------------------------------- UMMA issuer
      const uint32_t k_addr = smem_u32(sK), q_addr = smem_u32(sQ);
      int tile = 0, next_unit = 0, qs = 0;
      uint32_t k_parity = 0;
      uint32_t s_parity = (1u << kMsTiles) - 1;  // of each slot's s_empty
      MsRing qr;
      bool ok = true;
#pragma unroll 1
      for (const MsUnit* up; ok && (up = ms_next<false>(bars, next_unit, p.err)) != nullptr;
           ms_done<false>(bars, next_unit)) {
        const MsUnit& u = *up;
        const int slot0 = tile % kMsTiles;
#pragma unroll 1
        for (int q = u.q0; ok && q < u.q1; ++q) {
          if (ms_loads(u)) {
            qs = qr.i;
            if (!(ok = mbar_wait(&bars->q_full[qs], qr.parity, p.err))) break;
            qr.next(kMsQ);
          }
          const int rows = min(u.n - q * pb.tile_tokens, pb.tile_tokens) * pb.group;
          const uint32_t idesc = umma_idesc<T>(128, (uint32_t)(rows + 15) / 16 * 16, 0, 0);
          const uint64_t db = umma_desc_sw128(q_addr + qs * kChunkTileBytes, 16, 1024);
#pragma unroll 1
          for (int t = 0; ok && t < ktiles; ++t) {
            const int slot = slot0 + t;
            if (q == u.q0) ok = mbar_wait(&bars->k_full[slot], k_parity, p.err);
            ok = ok && mbar_wait(&bars->s_empty[slot], (s_parity >> slot) & 1, p.err);
            if (!ok) break;
            s_parity ^= 1u << slot;
            tc_fence_after();
            const uint64_t da = umma_desc_sw128(k_addr + slot * kChunkTileBytes, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t off = ((kk >> 2) * kChunkHalf + (kk & 3) * 32) >> 4;
              umma_ss(tmem + slot * 128, da + off, db + off, idesc, kk > 0);
            }
            umma_commit(&bars->s_full[slot]);
            if (q == u.q1 - 1) umma_commit(&bars->k_empty[slot]);
          }
          if (ok && ms_frees(u)) umma_commit(&bars->q_empty[qs]);
        }
        tile += ktiles;
        if (tile % kMsTiles == 0) k_parity ^= 1;
      }
      umma_commit(&bars->mma_done);
      mbar_wait(&bars->mma_done, 0, p.err);
    }
  } else if (warp == 18) {
    // -------------------------------------------------- the rows' lse, a column each
    int qc = 0, next_unit = 0;
    bool ok = true;
    int tok[4], head[4];  // of this lane's columns, -1: no row of a tile
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = lane + 32 * i;
      tok[i] = c < tile_rows ? c / pb.group : -1;
      head[i] = c % pb.group;
    }
#pragma unroll 1
    for (const MsUnit* up; ok && (up = ms_next<true>(bars, next_unit, p.err)) != nullptr;
         ms_done<true>(bars, next_unit)) {
      const MsUnit& u = *up;
      if (!ms_loads(u)) continue;
      const float* lse = p.lse + (int64_t)u.start * pb.hq + u.hk * pb.group;
      // a tile's values are read while the one before waits for its slot
      auto load = [&](int q, float* v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = q * pb.tile_tokens + tok[i];
          v[i] = -INFINITY;
          if (tok[i] >= 0 && q < u.q1 && k < u.n) v[i] = lse[(int64_t)k * pb.hq + head[i]];
        }
      };
      float now[4], next[4], sl[4];
      load(u.q0, now);
      if (kAlibi) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sl[i] = tok[i] >= 0 ? p.f.slopes[u.hk * pb.group + head[i]] * kLog2e : 0.f;
      }
#pragma unroll 1
      for (int q = u.q0; q < u.q1; ++q) {
        load(q + 1, next);
        const int ls = qc % kMsRows;
        if (qc >= kMsRows)
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&bars->l_empty[ls], ((qc / kMsRows) - 1) & 1, p.err));
        if (!ok) break;
        ++qc;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = lane + 32 * i;
          bars->neg_lse[ls][c] = now[i] == -INFINITY ? -INFINITY : -now[i] * kLog2e;
          if (kAlibi) {
            bars->slope[ls][c] = sl[i];
            bars->pos[ls][c] = (float)(q * pb.tile_tokens + tok[i]);  // from the first new token
          }
          now[i] = next[i];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->l_full[ls]);
      }
    }
  } else if (warp == 19) {
    ms_schedule(pb, bars, ktiles, p.cap, p.join + cta, p.err);
    // zeros where no new token sees (unless the call adds to mass)
    if (!p.accumulate) {
#pragma unroll 1
      for (int64_t r = cta; r < (int64_t)pb.batch * pb.hk; r += gridDim.x) {
        const ChunkSeq s = chunk_seq(pb, (int)(r / pb.hk));
        float* row = p.mass + r * p.cap;
#pragma unroll 1
        for (int64_t k0 = 0; k0 < p.cap; k0 += ukeys) {
          int a = 0, e = 0;
          if (s.n > 0 && k0 < s.keys) ms_steps(pb, s, ukeys, (int)(k0 / ukeys), a, e);
          if (e > a) continue;
          for (int64_t j = k0 + lane; j < k0 + ukeys && j < p.cap; j += 32) row[j] = 0.f;
        }
      }
    }
  } else {
    // ------------------------------------------------------------- sums, warps 0-15
    const int slot = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t tS = tmem + ((uint32_t)(quarter * 32) << 16) + slot * 128;
    int qc = 0, next_unit = 0;
    uint32_t s_parity = 0;
    // false once a wait ran out; the warp then goes on without waiting, its sums no longer count
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err));
    };
#pragma unroll 1
    for (const MsUnit* up; (up = ms_next<true>(bars, next_unit, p.err)) != nullptr;
         ms_done<true>(bars, next_unit)) {
      const MsUnit& u = *up;
      // units of two tiles take the slots in turn
      const int t = slot - (ktiles == 2 && (next_unit & 1) ? 2 : 0);
      const bool mine = t >= 0 && t < ktiles;
      const int tile0 = u.u * ukeys + t * kChunkTile, key = tile0 + row;
      const bool page_ok = u.pages_ok || !mine ||
                           chunk_page(pb, u.b, u.keys, u.u * ktiles + t, row >> 6) != pb.num_blocks;
      // tokens [open, shut) see every key of this tile
      int open = 0, shut = u.n;
      if (tile0 + kChunkTile > u.prefix) {
        open = tile0 + kChunkTile - 1 - u.pos0;
        if (pb.window) shut = min(u.n, tile0 + pb.window - u.pos0);
      }
      if (!u.pages_ok) shut = 0;
      const bool loads = ms_loads(u), frees = ms_frees(u);
      float acc = 0.f;
#pragma unroll 1
      for (int q = u.q0; q < u.q1; ++q) {
        if (loads) ++qc;
        const int ls = (qc - 1) % kMsRows;
        if (loads) wait(&bars->l_full[ls], ((qc - 1) / kMsRows) & 1);
        if (!mine) {  // another warpgroup's keys; the rows' slot is given back by all
          __syncwarp();
          if (lane == 0 && frees) mbar_arrive(&bars->l_empty[ls]);
          continue;
        }
        const int tok0 = q * pb.tile_tokens;
        bool mask = tok0 < open || tok0 + pb.tile_tokens > shut;
        int cols = tile_rows, c_lo = 0, c_hi = tile_rows;
        if (mask) {  // columns [c_lo, c_hi) see this key
          cols = c_hi = min(u.n - tok0, pb.tile_tokens) * pb.group;
          if (key >= u.prefix) {
            c_lo = min(max(key - u.pos0 - tok0, 0), kChunkTile) * pb.group;
            if (pb.window)
              c_hi = min(cols, min(max(key + pb.window - u.pos0 - tok0, 0), kChunkTile) * pb.group);
          }
          if (!page_ok) c_hi = 0;
        }
        wait(&bars->s_full[slot], s_parity);
        s_parity ^= 1;
        tc_fence_after();
        // (scalar arithmetic: packed pairs save issue slots on paper, but cost 1.5 moves a value)
        float sum;
        // Columns past the tile's rows hold products with zeros: NaN where the key is infinite. A step
        // whose sums show NaN runs again with those columns masked (masked in every step: 496 us for
        // 2048 tokens over 30011, this way 483).
#pragma unroll 1
        for (;; mask = true) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int cc = 0; cc < cols; cc += 16) {
            uint32_t raw[16];
            tmem_ld16(tS + cc, raw);
            float x[16];
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              const float4 v = *reinterpret_cast<const float4*>(&bars->neg_lse[ls][cc + c]);
              x[c] = v.x;
              x[c + 1] = v.y;
              x[c + 2] = v.z;
              x[c + 3] = v.w;
            }
            if constexpr (kAlibi) {
#pragma unroll
              for (int c = 0; c < 16; c += 4) {
                const float4 sl = *reinterpret_cast<const float4*>(&bars->slope[ls][cc + c]);
                const float4 ps = *reinterpret_cast<const float4*>(&bars->pos[ls][cc + c]);
                const float k = (float)(key - u.pos0);
                x[c] = fmaf(-sl.x, fabsf(k - ps.x), x[c]);
                x[c + 1] = fmaf(-sl.y, fabsf(k - ps.y), x[c + 1]);
                x[c + 2] = fmaf(-sl.z, fabsf(k - ps.z), x[c + 2]);
                x[c + 3] = fmaf(-sl.w, fabsf(k - ps.w), x[c + 3]);
              }
            }
            tmem_wait_ld();
            reg_fence<16>(raw);
            if constexpr (kCap) {
              float big = 0.f;
#pragma unroll
              for (int c = 0; c < 16; c += 2)
                big = fmax3f(big, fabsf(__uint_as_float(raw[c])), fabsf(__uint_as_float(raw[c + 1])));
              if (__all_sync(0xffffffffu, big <= p.f.tiny_max)) {  // (59 -> 50 us for 4 x 64 tokens)
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                  const uint64_t v = f32x2(__uint_as_float(raw[c]), __uint_as_float(raw[c + 1]));
                  f32x2_split(fma_f32x2(cap_tiny_x2(p.f, v), v, f32x2(x[c], x[c + 1])), x[c], x[c + 1]);
                }
              } else if (__all_sync(0xffffffffu, big * p.f.cap_in <= 1.f)) {
                // (in pairs: the polynomial is long enough to pay for the packing)
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                  const uint64_t v = mul_f32x2(
                      f32x2(__uint_as_float(raw[c]), __uint_as_float(raw[c + 1])),
                      f32x2(p.f.cap_in, p.f.cap_in));
                  f32x2_split(fma_f32x2(tanh_poly_x2(v), f32x2(p.f.cap_log2, p.f.cap_log2),
                                        f32x2(x[c], x[c + 1])), x[c], x[c + 1]);
                }
              } else {
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                  const float v = __uint_as_float(raw[c]) * p.f.cap_in;
                  x[c] = fmaf(fabsf(v) <= 1.f ? tanh_poly(v) : tanh_any(v), p.f.cap_log2, x[c]);
                }
              }
            } else {
#pragma unroll
              for (int c = 0; c < 16; ++c) x[c] = fmaf(__uint_as_float(raw[c]), p.f.scale_log2, x[c]);
            }
            if (mask) {
              const uint32_t vis = low_bits(c_hi - cc, 0) & ~low_bits(c_lo - cc, 0);
#pragma unroll
              for (int c = 0; c < 16; ++c)
                if (!((vis >> c) & 1u)) x[c] = -INFINITY;
            }
#pragma unroll
            for (int c = 0; c < 16; ++c)
              part[c & 3] = c < kMsEmu ? add_exp2_poly5(part[c & 3], x[c])
                                       : part[c & 3] + fast_exp2(x[c]);
          }
          sum = (part[0] + part[1]) + (part[2] + part[3]);
          if (mask || __all_sync(0xffffffffu, sum == sum)) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars->s_empty[slot]);
          if (frees) mbar_arrive(&bars->l_empty[ls]);
        }
        acc += sum;
      }
      if (!mine) continue;
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
  // No sequence has more than one query tile: every unit is one step, in one CTA (16 single tokens
  // over 1000 to 4095: 22 us, 23 with the join).
  if (p.b.total <= p.b.tile_tokens) return FI_OK;
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
  // Sequences of few tokens have one step a unit: smaller units even the CTAs' parts out.
  p.tiles = total_tokens > batch * p.b.tile_tokens ? 4 : 2;
  p.err = error_flag;
  return dtype == FI_DTYPE_F16 ? launch_mass_form<__half>(tq, tk, p, softcap > 0.f, st)
                               : launch_mass_form<__nv_bfloat16>(tq, tk, p, softcap > 0.f, st);
}
