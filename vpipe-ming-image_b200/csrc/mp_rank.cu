// Rank-space rows of a batch of requests on tcgen05, for requests of many rows:
//
//   v[t] = s_q F_a x[t]      row t of request q, F_a [rp][k] its adapter's factor
//
// (A in the forward pass, B^T in the backward pass). Bound by reading x once: 2 r
// operations for every two bytes.
//
// A unit is the rows of one request in one tile of 128 rows (64 where the blocks
// are that high). D[row][rank] = x F^T, both operands by TMA with the 128-byte
// swizzle, rows past the request's included: D's rows are independent, theirs are
// not used. As in mp_grad.cu an accumulator takes kChunk stages and is then added,
// in f32 with rounding to nearest, to sums in registers.
//
// With few units a cluster takes one, its CTAs share K and add their sums through
// distributed shared memory, in CTA order; with many, persistent CTAs walk them.
// (A few CTAs on the SMs that the projection beside them leaves idle would hide
// the whole launch, but one CTA needs 0.35 us a 64-wide stage, 65 cycles an MMA
// with 64 ranks, and the projection then waits for it: 4352 rows took 158 us, not
// 127.)
//
// The block is written whole (zeros in the rows of other requests and past rp):
// the projection kernel takes it as the appended K tiles' operand.
//
// Measured: 34 us for 16896 rows of 3840 with 64 ranks and 24 requests (130 MB, 3.8
// TB/s), 15.7 us for 4352 rows in 4 requests (2.1 TB/s; a cluster of 4 CTAs has 15
// stages, start and joining are half of its time).
#include <cuda_runtime.h>

#include "mp_device.cuh"
#include "mp_kernels.h"
#include "mp_launch.h"

namespace mp {

namespace {

constexpr int kTileRows = 128;  // MMA M
constexpr int kChunk = 4;       // 64-wide stages of an accumulator
constexpr uint32_t kXBytes = kTileRows * 128;
constexpr int kMaxStages = 10;
constexpr int kMaxRankSplits = 8;
constexpr int kSumWarp0 = 2;
constexpr int kRankThreads = 32 * (kSumWarp0 + 4);
constexpr uint32_t kAllBarrier = 1;

enum : uint32_t {
  kSiteRankFull = 0x3100u,
  kSiteRankEmpty = 0x3200u,
  kSiteRankSum = 0x3300u,
  kSiteRankTaken = 0x3400u,
  kSiteRankDone = 0x3500u,
};

struct RankGeo {
  int stages;
  uint32_t stage_bytes, smem;
};

// One CTA an SM with up to 128 ranks, two with up to 64.
__host__ __device__ inline RankGeo rank_geo(int rp) {
  RankGeo g;
  g.stage_bytes = kXBytes + (static_cast<uint32_t>(rp) * 128u + 1023u) / 1024u * 1024u;
  const uint32_t room = (rp <= 64 ? 104 : 224) * 1024;
  g.stages = static_cast<int>(room / g.stage_bytes);
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  const uint32_t tiles = g.stages * g.stage_bytes, exchange = kTileRows * (rp + 4) * 4;
  g.smem = (tiles > exchange ? tiles : exchange) + 1024 + 256;
  return g;
}

struct RankUnit {
  int unit;       // block of the plan at the units' level
  int row0;       // first row of x
  int lo, hi;     // the request's rows, from row0
  int adapter;
  bool work;      // of a live request
  bool clear;     // rows of v32 to clear: not of a live request
  int64_t out;    // row of vblk for row0
  int zero0, zero1, zero2, zero3;  // rows of vblk to clear besides: [zero0, zero1) and [zero2, zero3), from `out`
};

__device__ __forceinline__ int unit_level(const RankParams& p) { return p.lvl > 0 ? 1 : 0; }

// Unit i is block i of level 0 or 1 of the plan. The unit with the request's
// first (last) row in a block of 64 << lvl rows clears the block's rows before
// (after) its own 128, too.
__device__ __forceinline__ RankUnit rank_unit(const RankParams& p, int i) {
  const int ul = unit_level(p);
  RankUnit u;
  u.unit = i;
  const int4 ent = p.plan.block[ul][i];  // {tile, first row, row past the last, adapter}
  u.adapter = ent.w;
  u.work = ent.w >= 0;
  u.clear = ent.w < 0 && p.clear_v32 && ent.y < ent.z;
  u.row0 = ent.x << (6 + ul);
  u.lo = ent.y - u.row0;
  u.hi = ent.z - u.row0;
  u.zero0 = u.zero1 = u.zero2 = u.zero3 = 0;
  u.out = 0;
  if (u.work && p.vblk != nullptr) {
    const int tile = u.row0 >> (6 + p.lvl), blk = tile + (i - ent.x);  // i - ent.x: the request
    const int in = u.row0 - (tile << (6 + p.lvl));                     // the unit's place in the block
    u.out = (static_cast<int64_t>(blk) << (6 + p.lvl)) + in;
    if (p.lvl > 1) {
      const int4 whole = p.plan.block[p.lvl][blk];
      if (whole.y == ent.y) u.zero0 = -in;
      if (whole.z == ent.z) u.zero2 = kTileRows, u.zero3 = (64 << p.lvl) - in;
    }
  }
  return u;
}

// The request's strength; NaN with a factor that is not finite (it is stored as
// zeros, and its request's rows are NaN). And the adapter's own ranks: the columns
// past them are zeros.
struct UnitScale {
  float by;
  int ranks;
};
__device__ __forceinline__ UnitScale unit_scale(const RankParams& p, const RankUnit& u) {
  const AdapterInfo info = p.info[u.adapter];
  return {info.bad != 0 ? __int_as_float(0x7FC00000) : p.plan.block_s[unit_level(p)][u.unit], info.rank};
}

// The unit's rows of vblk outside its 128, or its rows of v32 if its request is
// not live, by threads `tid` of `threads`.
__device__ __forceinline__ void clear_rows(const RankParams& p, const RankUnit& u, int tid, int threads) {
  if (u.clear) {
    for (int e = tid; e < (u.hi - u.lo) * p.rp / 4; e += threads) {
      const int r = u.row0 + u.lo + e / (p.rp / 4), c = e % (p.rp / 4) * 4;
      *reinterpret_cast<float4*>(p.v32 + static_cast<int64_t>(r) * p.ld32 + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
  }
  if (!u.work || p.vblk == nullptr) return;
  const int per_row = p.ldb / 8;
  uint4* at = reinterpret_cast<uint4*>(p.vblk + u.out * p.ldb);
  for (int e = u.zero0 * per_row + tid; e < u.zero1 * per_row; e += threads) at[e] = make_uint4(0, 0, 0, 0);
  for (int e = u.zero2 * per_row + tid; e < u.zero3 * per_row; e += threads) at[e] = make_uint4(0, 0, 0, 0);
}

// COLS: rp rounded up to 32, 64 or 128, the sums a thread holds (one row each).
template <int COLS>
__global__ void __launch_bounds__(kRankThreads, COLS <= 64 ? 2 : 1) rank_tiles_kernel(const __grid_constant__ RankParams p) {
  extern __shared__ uint8_t rank_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = p.splits, rank = count > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit0 = static_cast<int>(blockIdx.x) / count, step = static_cast<int>(gridDim.x) / count;
  const int rows = 64 << unit_level(p);  // of a unit
  const RankGeo geo = rank_geo(p.rp);
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(rank_raw) + 1023u) & ~uintptr_t(1023u));
  const uint32_t tiles = smem_u32(base);
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + geo.smem - 1024 - 256);
  uint64_t *full = bars, *empty = bars + kMaxStages, *sum = bars + 2 * kMaxStages, *taken = sum + 2,
           *done = sum + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile uint32_t* abort = tmem_slot + 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < geo.stages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sum[b]), 1);
      mbar_init(smem_u32(&taken[b]), 4);
    }
    mbar_init(smem_u32(done), 1);
    *abort = 0u;
    fence_mbar_init();
    tma_prefetch_map(&p.tm_x);
    tma_prefetch_map(&p.tm_f);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 2 * COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_release();

  // K stages of this CTA
  const int all = (p.k + 63) / 64, per = (all + count - 1) / count;
  const int kt0 = min(rank * per, all), n_kt = min(kt0 + per, all) - kt0;

  if (warp == 0) {
    if (lane == 0) {
      RingPos at_stage;
      int sent = 0;
      bool ok = true;
      for (int unit = unit0; unit < p.units && ok; unit += step) {
        const RankUnit u = rank_unit(p, unit);
        if (!u.work) continue;
        for (int k = 0; k < n_kt; ++k, at_stage.next(geo.stages), ++sent) {
          const int s = at_stage.slot;
          if (at_stage.uses > 0)
            ok = mbar_wait<true>(smem_u32(&empty[s]), at_stage.phase ^ 1u, abort, kSiteRankEmpty | s, p.wait_limit_ns);
          if (!ok) break;
          const uint32_t bar = smem_u32(&full[s]), at = tiles + s * geo.stage_bytes;
          mbar_arrive_expect_tx(bar, kXBytes + static_cast<uint32_t>(p.rp) * 128u);
          tma_load_2d(at, &p.tm_x, bar, (kt0 + k) * 64, u.row0);
          tma_load_2d(at + kXBytes, &p.tm_f, bar, (kt0 + k) * 64, u.adapter * p.rp);
        }
      }
      if (*abort != 0u) {
        // copies in flight land (bounded) before the CTA leaves
        const uint64_t since = global_timer_ns();
        for (int j = max(0, sent - geo.stages); j < sent; ++j)
          while (!mbar_try_wait(smem_u32(&full[j % geo.stages]), (j / geo.stages) & 1u))
            if (global_timer_ns() - since > p.wait_limit_ns) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_bf16(kTileRows, p.rp);
      RingPos at_stage;
      int chunk = 0;
      bool ok = true;
      for (int unit = unit0; unit < p.units && ok; unit += step) {
        if (!rank_unit(p, unit).work) continue;
        for (int k = 0; k < n_kt; ++k, at_stage.next(geo.stages)) {
          const int s = at_stage.slot, b = chunk & 1;
          const bool first = k % kChunk == 0, last = k % kChunk == kChunk - 1 || k == n_kt - 1;
          if (first && chunk >= 2)
            ok = mbar_wait<true>(smem_u32(&taken[b]), ((chunk >> 1) - 1) & 1u, abort, kSiteRankTaken | b, p.wait_limit_ns);
          ok = ok && mbar_wait<true>(smem_u32(&full[s]), at_stage.phase, abort, kSiteRankFull | s, p.wait_limit_ns);
          if (!ok) break;
          tc_fence_after();
          const uint32_t xs = tiles + s * geo.stage_bytes, fs = xs + kXBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ss(tmem + b * COLS, make_sdesc_sw128(xs + kk * 32), make_sdesc_sw128(fs + kk * 32), idesc,
                    !first || kk > 0 ? 1u : 0u);
          umma_commit(smem_u32(&empty[s]));
          if (last) {
            umma_commit(smem_u32(&sum[b]));
            ++chunk;
          }
        }
      }
      umma_commit(smem_u32(done));
      const uint64_t since = global_timer_ns();
      while (!mbar_try_wait(smem_u32(done), 0))
        if (global_timer_ns() - since > p.wait_limit_ns) {
          atomicCAS(const_cast<uint32_t*>(abort), 0u, kSiteRankDone);
          break;
        }
    }
  } else {
    const int q = warp & 3, r = q * 32 + lane;  // this thread's row of a unit
    float sums[COLS];
    int chunk = 0;
    bool ok = true;
    for (int unit = unit0; unit < p.units && ok; unit += step) {
      const RankUnit u = rank_unit(p, unit);
      if (!u.work) {
        if (count == 1) clear_rows(p, u, threadIdx.x - 32 * kSumWarp0, 32 * 4);
        continue;
      }
#pragma unroll
      for (int c = 0; c < COLS; ++c) sums[c] = 0.0f;
      for (int k = 0; k < n_kt; k += kChunk, ++chunk) {
        const int b = chunk & 1;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait<true>(smem_u32(&sum[b]), (chunk >> 1) & 1u, abort, kSiteRankSum | b,
                                               p.wait_limit_ns)) != 0;
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < COLS; c += 16) {
          if (c >= p.rp) break;
          uint32_t v[16];
          MP_TMEM_LD_32X32B_X16(tmem + (static_cast<uint32_t>(q * 32) << 16) + b * COLS + c, v);
          MP_TMEM_WAIT_LD_REGS16(v);
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[c + j] += __uint_as_float(v[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&taken[b]));
      }
      if (count > 1 || !ok) break;  // a cluster has one unit
      clear_rows(p, u, threadIdx.x - 32 * kSumWarp0, 32 * 4);
      if (r >= rows) continue;
      const bool mine = r >= u.lo && r < u.hi;
      const UnitScale scale = unit_scale(p, u);
      const int ranks = mine ? scale.ranks : 0;
#pragma unroll
      for (int c = 0; c < COLS; ++c) sums[c] = c < ranks ? sums[c] * scale.by : 0.0f;
      if (mine && p.v32 != nullptr) {
        float* at = p.v32 + static_cast<int64_t>(u.row0 + r) * p.ld32;
#pragma unroll
        for (int c = 0; c < COLS; c += 4)
          if (c < p.rp) *reinterpret_cast<float4*>(at + c) = make_float4(sums[c], sums[c + 1], sums[c + 2], sums[c + 3]);
      }
      if (p.vblk != nullptr) {
        uint16_t* at = p.vblk + (u.out + r) * p.ldb;
#pragma unroll
        for (int c = 0; c < COLS; c += 8)
          *reinterpret_cast<uint4*>(at + c) =
              make_uint4(pack_bf16x2(sums[c], sums[c + 1]), pack_bf16x2(sums[c + 2], sums[c + 3]),
                         pack_bf16x2(sums[c + 4], sums[c + 5]), pack_bf16x2(sums[c + 6], sums[c + 7]));
        for (int c = COLS; c < p.ldb; c += 8) *reinterpret_cast<uint4*>(at + c) = make_uint4(0, 0, 0, 0);
      }
    }
    named_barrier(kAllBarrier, kRankThreads);  // copies landed, MMAs done: the stages' memory is free
    if (count > 1) {
      float* row = reinterpret_cast<float*>(base) + r * (p.rp + 4);
#pragma unroll
      for (int c = 0; c < COLS; c += 4)
        if (c < p.rp) *reinterpret_cast<float4*>(row + c) = make_float4(sums[c], sums[c + 1], sums[c + 2], sums[c + 3]);
    }
  }
  __syncwarp();
  if (warp < kSumWarp0) named_barrier(kAllBarrier, kRankThreads);
  const bool aborted = *abort != 0u;
  if (count > 1) {
    cluster_sync();
    if (!aborted) {
      // each CTA adds up and writes its share of the rows
      const RankUnit u = rank_unit(p, unit0);
      const UnitScale scale = u.work ? unit_scale(p, u) : UnitScale{0.0f, 0};
      clear_rows(p, u, rank * kRankThreads + threadIdx.x, count * kRankThreads);
      const int share = (rows + count - 1) / count, first = rank * share, last = min(first + share, rows);
      const int quads = (p.vblk != nullptr ? p.ldb : p.rp) / 4;
      const uint32_t ld = static_cast<uint32_t>(p.rp + 4) * 4u;
      for (int e = first * quads + threadIdx.x; u.work && e < last * quads; e += kRankThreads) {
        const int r = e / quads, c = e % quads * 4;
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r >= u.lo && r < u.hi && c < p.rp) {
          const uint32_t at = tiles + r * ld + c * 4u;
          float4 o[kMaxRankSplits];  // all in flight, then added in CTA order
#pragma unroll
          for (int z = 0; z < kMaxRankSplits; ++z)
            if (z < count) o[z] = ld_cluster_f4(mapa_shared(at, z));
          s = o[0];
#pragma unroll
          for (int z = 1; z < kMaxRankSplits; ++z)
            if (z < count) s.x += o[z].x, s.y += o[z].y, s.z += o[z].z, s.w += o[z].w;
          s.x = c < scale.ranks ? s.x * scale.by : 0.0f, s.y = c + 1 < scale.ranks ? s.y * scale.by : 0.0f;
          s.z = c + 2 < scale.ranks ? s.z * scale.by : 0.0f, s.w = c + 3 < scale.ranks ? s.w * scale.by : 0.0f;
          if (p.v32 != nullptr) *reinterpret_cast<float4*>(p.v32 + static_cast<int64_t>(u.row0 + r) * p.ld32 + c) = s;
        }
        if (p.vblk != nullptr)
          *reinterpret_cast<uint2*>(p.vblk + (u.out + r) * p.ldb + c) =
              make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
      }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 2 * COLS);
  if (threadIdx.x == 0 && aborted) atomicOr(p.err, kErrTimeout);
}

template <int COLS>
cudaError_t launch_cols(const RankParams& p, unsigned ctas, cudaStream_t stream) {
  const uint32_t smem = rank_geo(p.rp).smem;
  static SmemOptIn opted;
  cudaError_t e = opted.allow(reinterpret_cast<const void*>(rank_tiles_kernel<COLS>));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kRankThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, rank_tiles_kernel<COLS>, p);
}

}  // namespace

cudaError_t launch_rank_tiles(const RankParams& p, cudaStream_t stream) {
  RankParams q = p;
  q.units = plan_blocks(p.plan.m, p.plan.n_req, p.lvl > 0 ? 1 : 0);
  // K splits: until the units times the splits take most SMs, each with four stages. More cost more
  // than they bring: m 4352, k 3840 in one request takes 21.8 us with 8 splits,
  // 16.1 with 4.
  const int stages = (p.k + 63) / 64;
  q.splits = 1;
  while (q.splits < kMaxRankSplits && q.units * q.splits < 100 && stages >= 8 * q.splits) q.splits *= 2;
  const int room = 148 * (p.rp <= 64 ? 2 : 1);  // CTAs resident at once
  const unsigned ctas = q.splits > 1 ? static_cast<unsigned>(q.units) * q.splits
                                     : static_cast<unsigned>(q.units < room ? q.units : room);
  if (p.rp <= 32) return launch_cols<32>(q, ctas, stream);
  if (p.rp <= 64) return launch_cols<64>(q, ctas, stream);
  return launch_cols<128>(q, ctas, stream);
}

}  // namespace mp
