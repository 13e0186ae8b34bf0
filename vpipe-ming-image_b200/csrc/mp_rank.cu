// Rank-space rows of a batch of requests on tcgen05, for requests of many rows:
//
//   v[t] = s_q F_a x[t]      row t of request q, F_a [rp][k] its adapter's factor
//
// (A in the forward pass, B^T in the backward pass). Bound by reading x once: 2 r
// operations for every two bytes.
//
// A cluster takes up to 128 rows of one block of the plan (the rows of one
// request in one token tile); its CTAs share K and add their sums through
// distributed shared memory, in CTA order. D[row][rank] = x F^T, both operands by
// TMA with the 128-byte swizzle, rows past the request's included: D's rows are
// independent, theirs are not used. As in mp_grad.cu an accumulator takes kChunk
// stages and is then added, in f32 with rounding to nearest, to sums in registers.
//
// The block is written whole (zeros in the rows of other requests and past rp):
// the projection kernel takes it as the appended K tiles' operand.
#include <cuda_runtime.h>

#include "mp_device.cuh"
#include "mp_kernels.h"

namespace mp {

namespace {

constexpr int kTileRows = 128;  // MMA M
constexpr int kChunk = 4;       // 64-wide stages of an accumulator
constexpr uint32_t kXBytes = kTileRows * 128;
constexpr int kMaxStages = 8;
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
  const uint32_t room = rp <= 64 ? 104 * 1024 : 200 * 1024;
  g.stages = static_cast<int>(room / g.stage_bytes);
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  const uint32_t tiles = g.stages * g.stage_bytes, exchange = kTileRows * (rp + 4) * 4;
  g.smem = (tiles > exchange ? tiles : exchange) + 1024 + 256;
  return g;
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// COLS: rp rounded up to 32, 64 or 128, the sums a thread holds (one row each).
template <int COLS>
__global__ void __launch_bounds__(kRankThreads, COLS <= 64 ? 2 : 1) rank_tiles_kernel(const __grid_constant__ RankParams p) {
  extern __shared__ uint8_t rank_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank()), count = p.splits;
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

  // this cluster's rows: part `sub` of a block of 64 << lvl rows
  const int tile_rows = 64 << p.lvl, subs = tile_rows > kTileRows ? tile_rows / kTileRows : 1;
  const int unit = static_cast<int>(blockIdx.x) / count, blk = unit / subs, sub = unit % subs;
  const int4 ent = p.plan.block[p.lvl][blk];  // {tile, first row, row past the last, adapter}
  const bool used = ent.w >= 0;
  const int row0 = ent.x * tile_rows + sub * kTileRows, rows = min(kTileRows, tile_rows);
  const int lo = max(ent.y, row0) - row0, hi = min(ent.z, row0 + rows) - row0;  // the request's rows here
  const bool work = used && lo < hi;
  // K stages of this CTA
  const int all = (p.k + 63) / 64, per = (all + count - 1) / count;
  const int kt0 = min(rank * per, all), n_kt = work ? min(kt0 + per, all) - kt0 : 0;

  if (warp == 0) {
    if (lane == 0) {
      int sent = 0;
      for (int n = 0; n < n_kt; ++n) {
        const int s = n % geo.stages;
        if (n >= geo.stages && !mbar_wait(smem_u32(&empty[s]), ((n / geo.stages) & 1u) ^ 1u, abort,
                                          kSiteRankEmpty | s, p.wait_limit_ns))
          break;
        const uint32_t bar = smem_u32(&full[s]), at = tiles + s * geo.stage_bytes;
        mbar_arrive_expect_tx(bar, kXBytes + static_cast<uint32_t>(p.rp) * 128u);
        tma_load_2d(at, &p.tm_x, bar, (kt0 + n) * 64, row0);
        tma_load_2d(at + kXBytes, &p.tm_f, bar, (kt0 + n) * 64, ent.w * p.rp);
        sent = n + 1;
      }
      if (*abort != 0u) {
        // copies in flight land (bounded) before the CTA leaves
        const uint64_t since = global_timer_ns();
        for (int n = max(0, sent - geo.stages); n < sent; ++n)
          while (!mbar_try_wait(smem_u32(&full[n % geo.stages]), (n / geo.stages) & 1u))
            if (global_timer_ns() - since > p.wait_limit_ns) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && n_kt > 0) {
      const uint32_t idesc = make_idesc_bf16(kTileRows, p.rp);
      for (int n = 0; n < n_kt; ++n) {
        const int s = n % geo.stages, chunk = n / kChunk, b = chunk & 1;
        if (n % kChunk == 0 && chunk >= 2 &&
            !mbar_wait(smem_u32(&taken[b]), ((chunk >> 1) - 1) & 1u, abort, kSiteRankTaken | b, p.wait_limit_ns))
          break;
        if (!mbar_wait(smem_u32(&full[s]), (n / geo.stages) & 1u, abort, kSiteRankFull | s, p.wait_limit_ns)) break;
        tc_fence_after();
        const uint32_t xs = tiles + s * geo.stage_bytes, fs = xs + kXBytes;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_ss(tmem + b * COLS, make_sdesc_sw128(xs + kk * 32), make_sdesc_sw128(fs + kk * 32), idesc,
                  n % kChunk != 0 || kk > 0 ? 1u : 0u);
        umma_commit(smem_u32(&empty[s]));
        if (n % kChunk == kChunk - 1 || n == n_kt - 1) umma_commit(smem_u32(&sum[b]));
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
    const int q = warp & 3;
    float sums[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) sums[c] = 0.0f;
    for (int chunk = 0; chunk * kChunk < n_kt; ++chunk) {
      const int b = chunk & 1;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sum[b]), (chunk >> 1) & 1u, abort, kSiteRankSum | b,
                                             p.wait_limit_ns)))
        break;
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
    named_barrier(kAllBarrier, kRankThreads);  // copies landed, MMAs done: the stages' memory is free
    if (work) {
      float* row = reinterpret_cast<float*>(base) + (q * 32 + lane) * (p.rp + 4);
#pragma unroll
      for (int c = 0; c < COLS; c += 4)
        if (c < p.rp) *reinterpret_cast<float4*>(row + c) = make_float4(sums[c], sums[c + 1], sums[c + 2], sums[c + 3]);
    }
  }
  __syncwarp();
  if (warp < kSumWarp0) named_barrier(kAllBarrier, kRankThreads);
  const bool aborted = *abort != 0u;
  cluster_sync();
  if (used && !aborted) {
    // each CTA adds up and writes its share of the rows
    float scale = p.plan.block_s[p.lvl][blk];
    // a factor that is not finite is stored as zeros; its request's rows are NaN
    if (p.bad[ent.w] != 0) scale = __int_as_float(0x7FC00000);
    const int share = (rows + count - 1) / count, first = rank * share, last = min(first + share, rows);
    const int quads = (p.vblk != nullptr ? p.ldb : p.rp) / 4;
    const uint32_t ld = static_cast<uint32_t>(p.rp + 4) * 4u;
    for (int e = first * quads + threadIdx.x; e < last * quads; e += kRankThreads) {
      const int r = e / quads, c = e % quads * 4;
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const bool mine = work && r >= lo && r < hi && c < p.rp;
      if (mine) {
        const uint32_t at = tiles + r * ld + c * 4u;
        s = ld_cluster_f4(mapa_shared(at, 0));
        for (int z = 1; z < count; ++z) {
          const float4 o = ld_cluster_f4(mapa_shared(at, z));
          s.x += o.x, s.y += o.y, s.z += o.z, s.w += o.w;
        }
        s.x *= scale, s.y *= scale, s.z *= scale, s.w *= scale;
        if (p.v32 != nullptr) *reinterpret_cast<float4*>(p.v32 + static_cast<int64_t>(row0 + r) * p.ld32 + c) = s;
      }
      if (p.vblk != nullptr) {
        const int64_t at = static_cast<int64_t>(blk) * tile_rows + sub * kTileRows + r;
        *reinterpret_cast<uint2*>(p.vblk + at * p.ldb + c) =
            make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
      }
    }
  }
  cluster_sync();  // no CTA leaves while another reads its sums
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 2 * COLS);
  if (threadIdx.x == 0 && aborted) atomicOr(p.err, kErrTimeout);
}

template <int COLS>
cudaError_t launch_cols(const RankParams& p, unsigned clusters, cudaStream_t stream) {
  const uint32_t smem = rank_geo(p.rp).smem;
  cudaError_t e = cudaFuncSetAttribute(rank_tiles_kernel<COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * p.splits);
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
  const int blocks = plan_blocks(p.plan.m, p.plan.n_req, p.lvl), tile_rows = 64 << p.lvl;
  const int subs = tile_rows > kTileRows ? tile_rows / kTileRows : 1;
  if (blocks == 0) return cudaSuccess;
  // K splits: until the row parts with work (about one per 128 rows and one
  // more per request) times the splits fill the SMs, each with four stages
  const int parts = (p.plan.m + kTileRows - 1) / kTileRows + p.plan.n_req, stages = (p.k + 63) / 64;
  q.splits = 1;
  while (q.splits < 8 && parts * q.splits < 148 && stages >= 8 * q.splits) q.splits *= 2;
  const unsigned clusters = static_cast<unsigned>(blocks) * subs;
  if (p.rp <= 32) return launch_cols<32>(q, clusters, stream);
  if (p.rp <= 64) return launch_cols<64>(q, clusters, stream);
  return launch_cols<128>(q, clusters, stream);
}

}  // namespace mp
