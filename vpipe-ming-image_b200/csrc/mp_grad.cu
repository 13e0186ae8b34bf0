// Gradients of the factors of many adapters: matrix products grouped by
// adapter, over the ragged row ranges of its requests,
//
//   out[a] = sum over the rows t of adapter a of x[t]^T u[t],
//
// dA from x (bf16, or its 8-bit checkpoint) and u = s dy B, dB from dy and
// v = s x A^T. Bound by memory: x and dy are read once, 2 r operations for
// every byte or two of them.
//
// One cluster per adapter and 128 features; its CTAs take the adapter's rows
// 64 at a time in turn and add their sums through distributed shared memory, in
// CTA order. Per 64 rows: x by TMA, [64 rows][64 features] boxes that are the
// MN-major A operand of tcgen05 as they land (M = features, K = rows); u, f32 in
// memory, is cut by warps 2-9 into three bf16 parts of 8 bits each, side by
// side in the N of the B operand: the products are then those of the f32
// values, and cost no second pass over x.
//
// tcgen05 adds to its f32 accumulator without rounding to nearest: over a long
// run of rows the sums drift towards zero (2e-6 at 1000 rows). So an accumulator
// takes kChunk stages (256 rows) only; the last warps then add it, the three
// parts smallest first, to sums in registers, while the MMAs fill the other one.
//
// A checkpoint's codes are whole numbers of up to 8 bits, exact in bf16: warps
// 2-9 widen them, and the scale of a (row, 128 features) goes into u, in f32.
#include <cuda_runtime.h>

#include "mp_device.cuh"
#include "mp_kernels.h"

namespace mp {

namespace {

constexpr int kTileF = 128;   // features of a CTA (MMA M) and of a checkpoint scale
constexpr int kRows = 64;     // rows of a stage (four MMA K steps)
constexpr int kParts = 3;     // bf16 parts of an f32 value
static_assert(kTileF == kCkGroup, "one scale per row of a tile");

constexpr int kChunk = 4;     // stages of an accumulator

constexpr int kConvWarp0 = 2;
constexpr int kConvThreads = 256;
constexpr int kSumWarp0 = kConvWarp0 + kConvThreads / 32;
// Warps that add up the accumulators: 4 hold a feature row of up to 64 ranks a
// thread, 8 one of up to 128 in two halves (TASKS 4).
template <int TASKS>
constexpr int kSumWarps = TASKS == 4 ? 8 : 4;
template <int TASKS>
constexpr int kSumCols = TASKS == 1 ? 32 : 64;
template <int TASKS>
constexpr int kGradThreads = 32 * (kSumWarp0 + kSumWarps<TASKS>);
constexpr uint32_t kBoxBytes = kRows * 128;      // [64 rows][64 bf16]
constexpr uint32_t kXBytes = 2 * kBoxBytes;      // the A operand
constexpr uint32_t kCodeBytes = kRows * kTileF;  // a stage's codes
constexpr int kMaxGradStages = 6;
constexpr uint32_t kGradSmemMost = 220 * 1024;

constexpr uint32_t kAllBarrier = 1;  // named barrier of the whole CTA

enum : uint32_t {
  kSiteGradFull = 0x2100u,
  kSiteGradConv = 0x2200u,
  kSiteGradEmpty = 0x2300u,
  kSiteGradDone = 0x2400u,
  kSiteGradSum = 0x2500u,
  kSiteGradTaken = 0x2600u,
};

// Columns of the parts in the B operand and in TMEM: side by side while one
// MMA (N at most 256) takes all three, else the third from the next 64-column
// box on, with an MMA of its own.
struct PartCols {
  int n1, n2;     // N of the first and second MMA (0: none)
  int third;      // first column of the third part
  int boxes;      // 64-column boxes of the operand
  int cols;       // TMEM columns of one accumulator, a power of two
  int bufs;       // accumulators
};

__host__ __device__ inline PartCols part_cols(int rp) {
  PartCols c;
  const bool one = kParts * rp <= 256;
  c.third = one ? 2 * rp : (2 * rp + 63) / 64 * 64;
  c.n1 = one ? 3 * rp : 2 * rp;
  c.n2 = one ? 0 : rp;
  const int most = c.third + rp;
  c.boxes = (most + 63) / 64;
  c.cols = most <= 64 ? 64 : most <= 128 ? 128 : most <= 256 ? 256 : 512;
  c.bufs = c.cols <= 256 ? 2 : 1;
  return c;
}

// Floats between the sums of two ranks in the exchange buffer: dB is written
// rank fastest, and one more float puts consecutive ranks in different banks.
__host__ __device__ inline int exchange_ld(bool rank_major) { return rank_major ? kTileF : kTileF + 1; }

struct GradGeo {
  int stages;
  uint32_t stage_bytes, u_off, code_off;
  uint32_t smem;
};

__host__ __device__ inline GradGeo grad_geo(int rp, bool codes) {
  GradGeo g;
  g.u_off = kXBytes;
  g.code_off = kXBytes + part_cols(rp).boxes * kBoxBytes;
  g.stage_bytes = g.code_off + (codes ? kCodeBytes : 0);
  g.stages = static_cast<int>(kGradSmemMost / g.stage_bytes);
  if (g.stages > kMaxGradStages) g.stages = kMaxGradStages;
  const uint32_t tiles = g.stages * g.stage_bytes;
  const uint32_t exchange = rp * (kTileF + 1) * 4;
  g.smem = (tiles > exchange ? tiles : exchange) + 1024 + 256;
  return g;
}

// The row tiles of one adapter that fall to CTA `rank` of `count`: tile i of
// all its segments' tiles, i = rank, rank + count, ...
struct TileIter {
  const int2* seg;
  int left, i, count;
  int2 cur;
  __device__ TileIter(const RequestPlan& pl, int a, int rank, int count_) {
    const int b = pl.begin[a];
    seg = pl.seg + b;
    left = pl.begin[a + 1] - b;
    i = rank;
    count = count_;
    cur = left > 0 ? seg[0] : make_int2(0, 0);
  }
  // Tiles of this CTA in all.
  __device__ int total() const {
    int n = 0;
    for (int s = 0; s < left; ++s) n += (seg[s].y - seg[s].x + kRows - 1) / kRows;
    return n > i ? (n - i + count - 1) / count : 0;
  }
  // First row and rows of the next tile, or false.
  __device__ bool next(int& t0, int& rows) {
    while (left > 0) {
      const int n = (cur.y - cur.x + kRows - 1) / kRows;
      if (i < n) {
        t0 = cur.x + i * kRows;
        rows = min(kRows, cur.y - t0);
        i += count;
        return true;
      }
      i -= n;
      ++seg;
      if (--left > 0) cur = *seg;
    }
    return false;
  }
};

// MN-major operand of 64-row boxes, 128-byte swizzle: 64 features (128 bytes)
// by 8 rows are 1024 bytes, the next 8 rows follow (stride offset), the next 64
// features are a box further (leading offset); a 16-row step starts 2048 bytes on.
__device__ __forceinline__ uint64_t mn_desc(uint32_t tile, int kk) {
  uint64_t d = 0;
  const uint32_t a = tile + static_cast<uint32_t>(kk) * 2048u;
  d |= static_cast<uint64_t>((a & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kBoxBytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;  // descriptor version (sm_100)
  d |= static_cast<uint64_t>(2u) << 61;  // SWIZZLE_128B
  return d;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Eight values of row `row` of u from column c: zeros past the valid columns
// and for rows outside the segment.
__device__ __forceinline__ void load_u8(const float* u, int64_t ldu, int64_t row, int c, int cols, bool vec, bool ok,
                                        float (&f)[8]) {
  const float* at = u + row * ldu + c;
  if (ok && vec && c + 8 <= cols) {
    const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = ok && c + i < cols ? at[i] : 0.0f;
  }
}

// The next bf16 part of two values, which keep what is left of them. An
// infinity or NaN is all in its first part (inf - inf would be NaN).
__device__ __forceinline__ uint32_t take_part(float& a, float& b) {
  const uint32_t w = pack_bf16x2(a, b);
  const float ha = __uint_as_float(w << 16), hb = __uint_as_float(w & 0xFFFF0000u);
  a = fabsf(ha) <= 3.4e38f ? a - ha : 0.0f;
  b = fabsf(hb) <= 3.4e38f ? b - hb : 0.0f;
  return w;
}

struct GradSmem {
  uint32_t tiles;
  float* exchange;
  uint64_t *full, *conv, *empty;  // [stages]
  uint64_t *sum, *taken;          // [2] accumulator filled, and added up
  uint64_t* done;
  uint32_t* tmem_slot;
  volatile uint32_t* abort;
};

// TASKS: 8-value pieces of a 64-row stage of u per converting thread.
template <int TASKS, bool CODES>
__device__ void convert(const GradParams& p, const GradMember& mb, const GradSmem& sm, const GradGeo& geo,
                        const PartCols& pc, int a, int f_tile, int rank, int count) {
  const int tid = threadIdx.x - 32 * kConvWarp0, lane = threadIdx.x & 31;
  const int per_row = p.rp / 8, pieces = kRows * per_row;
  const bool vec = mb.ldu % 4 == 0 && (reinterpret_cast<uintptr_t>(mb.u) & 15) == 0;
  const float* scale = CODES ? mb.scale + static_cast<int64_t>(f_tile) * p.plan.m : nullptr;
  int row_of[TASKS], col_of[TASKS];
#pragma unroll
  for (int j = 0; j < TASKS; ++j) {
    const int e = tid + j * kConvThreads;
    row_of[j] = e < pieces ? e / per_row : kRows;  // kRows: no piece
    col_of[j] = e < pieces ? e % per_row * 8 : 0;
  }
  float f[TASKS][8], by[TASKS];
  auto load = [&](int t0, int rows) {
#pragma unroll
    for (int j = 0; j < TASKS; ++j) {
      const bool ok = row_of[j] < rows;
      load_u8(mb.u, mb.ldu, t0 + row_of[j], col_of[j], p.r, vec, ok, f[j]);
      if (CODES) by[j] = ok ? scale[t0 + row_of[j]] : 0.0f;
    }
  };
  // one answer for the warp, so that all of its lanes give up together
  auto wait_all = [&](uint32_t bar, uint32_t parity, uint32_t site) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, sm.abort, site, p.wait_limit_ns)) != 0;
  };
  TileIter it(p.plan, a, rank, count);
  int t0, rows;
  bool have = it.next(t0, rows);
  if (have) load(t0, rows);
  for (uint32_t n = 0; have; ++n) {
    const int s = static_cast<int>(n % geo.stages);
    const uint32_t ph = (n / geo.stages) & 1u;
    if (n >= static_cast<uint32_t>(geo.stages) &&
        !wait_all(smem_u32(&sm.empty[s]), ph ^ 1u, kSiteGradEmpty | s))
      return;
    const uint32_t xs = sm.tiles + s * geo.stage_bytes, us = xs + geo.u_off;
#pragma unroll
    for (int j = 0; j < TASKS; ++j) {
      if (row_of[j] >= kRows) continue;
      const uint32_t row = us + row_of[j] * 128u, sw = static_cast<uint32_t>(row_of[j] & 7);
      if (CODES) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] *= by[j];
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = take_part(f[j][2 * i], f[j][2 * i + 1]);
        const uint32_t col = col_of[j] + (part == 2 ? pc.third : part * p.rp);
        st_shared_v4(row + (col >> 6) * kBoxBytes + (((col >> 3 & 7u) ^ sw) << 4), w[0], w[1], w[2], w[3]);
      }
    }
    const int rows_now = rows;
    have = it.next(t0, rows);
    if (have) load(t0, rows);  // in flight until the next stage
    if (CODES) {
      if (!wait_all(smem_u32(&sm.full[s]), ph, kSiteGradFull | s)) return;
#pragma unroll
      for (int j = 0; j < kRows * kTileF / 16 / kConvThreads; ++j) {  // 16 codes of a row at a time
        const int e = tid + j * kConvThreads, row = e / (kTileF / 16), c = e % (kTileF / 16);
        uint4 q = ld_shared_v4(xs + geo.code_off + row * kTileF + c * 16);
        if (row >= rows_now) q = make_uint4(0, 0, 0, 0);
        const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // byte b + 128 as the float 32768 + (b + 128), less 32896: exact
          const uint32_t ofs = qw[i] ^ 0x80808080u;
          const float v0 = __uint_as_float(__byte_perm(ofs, 0x4700u, 0x5404u)) - 32896.0f;
          const float v1 = __uint_as_float(__byte_perm(ofs, 0x4700u, 0x5414u)) - 32896.0f;
          const float v2 = __uint_as_float(__byte_perm(ofs, 0x4700u, 0x5424u)) - 32896.0f;
          const float v3 = __uint_as_float(__byte_perm(ofs, 0x4700u, 0x5434u)) - 32896.0f;
          w[2 * i] = pack_bf16x2(v0, v1);
          w[2 * i + 1] = pack_bf16x2(v2, v3);
        }
        const uint32_t at = xs + (c >> 2) * kBoxBytes + row * 128u, ch = static_cast<uint32_t>(2 * (c & 3));
        const uint32_t sw = static_cast<uint32_t>(row & 7);
        st_shared_v4(at + ((ch ^ sw) << 4), w[0], w[1], w[2], w[3]);
        st_shared_v4(at + (((ch + 1) ^ sw) << 4), w[4], w[5], w[6], w[7]);
      }
    } else if (rows_now < kRows) {
      // the rows after the segment's last are another request's: zeros, since
      // an infinity or NaN there would come through a product with 0
      if (!wait_all(smem_u32(&sm.full[s]), ph, kSiteGradFull | s)) return;
      for (int e = rows_now * 8 + tid; e < kRows * 8; e += kConvThreads) {
        st_shared_v4(xs + e * 16, 0, 0, 0, 0);
        st_shared_v4(xs + kBoxBytes + e * 16, 0, 0, 0, 0);
      }
    }
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sm.conv[s]));
  }
}

template <int TASKS, bool CODES>
__device__ void grad_tile(const GradParams& p, const GradMember& mb, int a, int f_tile, uint8_t* raw) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank()), count = p.splits;
  const int col0 = warp >= kSumWarp0 + 4 ? kSumCols<TASKS> : 0;  // the adding warp's first rank
  const PartCols pc = part_cols(p.rp);
  const GradGeo geo = grad_geo(p.rp, CODES);
  GradSmem sm;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~uintptr_t(1023u));
  sm.tiles = smem_u32(base);
  sm.exchange = reinterpret_cast<float*>(base);
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + geo.smem - 1024 - 256);
  sm.full = bars;
  sm.conv = bars + kMaxGradStages;
  sm.empty = bars + 2 * kMaxGradStages;
  sm.sum = bars + 3 * kMaxGradStages;
  sm.taken = sm.sum + 2;
  sm.done = sm.taken + 2;
  sm.tmem_slot = reinterpret_cast<uint32_t*>(sm.done + 1);
  sm.abort = sm.tmem_slot + 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < geo.stages; ++s) {
      mbar_init(smem_u32(&sm.full[s]), 1);
      mbar_init(smem_u32(&sm.conv[s]), kConvThreads / 32);
      mbar_init(smem_u32(&sm.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sm.sum[b]), 1);
      mbar_init(smem_u32(&sm.taken[b]), kSumWarps<TASKS>);
    }
    mbar_init(smem_u32(sm.done), 1);
    *sm.abort = 0u;
    fence_mbar_init();
    tma_prefetch_map(&mb.tm_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(sm.tmem_slot), pc.cols * pc.bufs);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sm.tmem_slot;
  pdl_wait();
  pdl_release();

  const int tiles = TileIter(p.plan, a, rank, count).total();
  const int ld = exchange_ld(mb.rank_major != 0);
  if (warp == 0) {
    if (lane == 0) {
      TileIter it(p.plan, a, rank, count);
      int t0, rows;
      uint32_t n = 0, pend = 0;
      for (; it.next(t0, rows); ++n) {
        const int s = static_cast<int>(n % geo.stages);
        if (n >= static_cast<uint32_t>(geo.stages) &&
            !mbar_wait(smem_u32(&sm.empty[s]), ((n / geo.stages) & 1u) ^ 1u, sm.abort, kSiteGradEmpty | s,
                       p.wait_limit_ns))
          break;
        const uint32_t bar = smem_u32(&sm.full[s]), xs = sm.tiles + s * geo.stage_bytes;
        if (CODES) {
          mbar_arrive_expect_tx(bar, kCodeBytes);
          tma_load_2d(xs + geo.code_off, &mb.tm_x, bar, f_tile * kTileF, t0);
        } else {
          mbar_arrive_expect_tx(bar, kXBytes);
          tma_load_2d(xs, &mb.tm_x, bar, f_tile * kTileF, t0);
          tma_load_2d(xs + kBoxBytes, &mb.tm_x, bar, f_tile * kTileF + 64, t0);
        }
        pend = n + 1;
      }
      if (*sm.abort != 0u) {
        // copies in flight land (bounded) before the CTA leaves
        const uint64_t since = global_timer_ns();
        for (uint32_t j = pend > static_cast<uint32_t>(geo.stages) ? pend - geo.stages : 0; j < pend; ++j)
          while (!mbar_try_wait(smem_u32(&sm.full[j % geo.stages]), (j / geo.stages) & 1u))
            if (global_timer_ns() - since > p.wait_limit_ns) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && tiles > 0) {
      const uint32_t mn = (1u << 15) | (1u << 16);  // both operands MN-major
      const uint32_t id1 = make_idesc_bf16(kTileF, pc.n1) | mn, id2 = make_idesc_bf16(kTileF, pc.n2) | mn;
      for (int n = 0; n < tiles; ++n) {
        const int s = n % geo.stages, chunk = n / kChunk, b = chunk % pc.bufs, use = chunk / pc.bufs;
        const uint32_t ph = (n / geo.stages) & 1u;
        if (n % kChunk == 0 && use > 0 &&
            !mbar_wait(smem_u32(&sm.taken[b]), (use - 1) & 1u, sm.abort, kSiteGradTaken | b, p.wait_limit_ns))
          break;
        if (!mbar_wait(smem_u32(&sm.full[s]), ph, sm.abort, kSiteGradFull | s, p.wait_limit_ns) ||
            !mbar_wait(smem_u32(&sm.conv[s]), ph, sm.abort, kSiteGradConv | s, p.wait_limit_ns))
          break;
        tc_fence_after();
        const uint32_t xs = sm.tiles + s * geo.stage_bytes, us = xs + geo.u_off, d = tmem + b * pc.cols;
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk) {
          const uint32_t acc = n % kChunk != 0 || kk > 0 ? 1u : 0u;
          umma_ss(d, mn_desc(xs, kk), mn_desc(us, kk), id1, acc);
          if (pc.n2 > 0)
            umma_ss(d + pc.third, mn_desc(xs, kk), mn_desc(us + (pc.third >> 6) * kBoxBytes, kk), id2, acc);
        }
        umma_commit(smem_u32(&sm.empty[s]));
        if (n % kChunk == kChunk - 1 || n == tiles - 1) umma_commit(smem_u32(&sm.sum[b]));
      }
      umma_commit(smem_u32(sm.done));
      const uint64_t since = global_timer_ns();
      while (!mbar_try_wait(smem_u32(sm.done), 0))
        if (global_timer_ns() - since > p.wait_limit_ns) {
          atomicCAS(const_cast<uint32_t*>(sm.abort), 0u, kSiteGradDone);
          break;
        }
    }
  } else if (warp < kSumWarp0) {
    convert<TASKS, CODES>(p, mb, sm, geo, pc, a, f_tile, rank, count);
  } else {
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float sums[kSumCols<TASKS>];  // one feature, consecutive ranks
#pragma unroll
    for (int c = 0; c < kSumCols<TASKS>; ++c) sums[c] = 0.0f;
    for (int chunk = 0; chunk * kChunk < tiles; ++chunk) {
      const int b = chunk % pc.bufs;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sm.sum[b]), (chunk / pc.bufs) & 1u, sm.abort,
                                             kSiteGradSum | b, p.wait_limit_ns)))
        break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kSumCols<TASKS>; c += 16) {
        if (col0 + c >= p.rp) break;
        uint32_t v[16], w[16];
        const uint32_t at = tmem + lanes + b * pc.cols + col0 + c;
        MP_TMEM_LD_32X32B_X16(at + p.rp, v);
        MP_TMEM_LD_32X32B_X16(at + pc.third, w);
        MP_TMEM_WAIT_LD_REGS16(v);
        MP_TMEM_WAIT_LD_REGS16(w);
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(w[j]));
        MP_TMEM_LD_32X32B_X16(at, v);
        MP_TMEM_WAIT_LD_REGS16(v);
#pragma unroll
        for (int j = 0; j < 16; ++j) sums[c + j] += __uint_as_float(v[j]) + __uint_as_float(w[j]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.taken[b]));
    }
    // every copy has landed and every MMA is done (or the CTA gave up): the
    // stages' memory takes the sums
    named_barrier(kAllBarrier, kGradThreads<TASKS>);
    const int f = (warp & 3) * 32 + lane;
#pragma unroll
    for (int c = 0; c < kSumCols<TASKS>; ++c)
      if (col0 + c < p.rp) sm.exchange[(col0 + c) * ld + f] = sums[c];
  }
  __syncwarp();
  if (warp < kSumWarp0) named_barrier(kAllBarrier, kGradThreads<TASKS>);
  const bool aborted = *sm.abort != 0u;
  cluster_sync();
  // the CTAs share the adding up: each takes some ranks (dA) or features (dB)
  const int f0 = f_tile * kTileF, width = min(kTileF, mb.width - f0);
  float* out = mb.out + static_cast<int64_t>(a) * p.r * mb.width;
  const uint32_t ex = smem_u32(sm.exchange);
  auto sum_at = [&](int r, int f) {
    const uint32_t at = ex + static_cast<uint32_t>(r * ld + f) * 4u;
    float s = ld_cluster_f32(mapa_shared(at, 0));
    for (int z = 1; z < count; ++z) s += ld_cluster_f32(mapa_shared(at, z));
    return s;
  };
  if (!aborted) {
    if (mb.rank_major) {
      for (int e = threadIdx.x; e < p.r * kTileF; e += kGradThreads<TASKS>) {
        const int r = e / kTileF, f = e % kTileF;
        if (r % count == rank && f < width) out[static_cast<int64_t>(r) * mb.width + f0 + f] = sum_at(r, f);
      }
    } else {
      const int per = kTileF / count, lo = rank * per, hi = min(lo + per, width);
      for (int e = lo * p.r + threadIdx.x; e < hi * p.r; e += kGradThreads<TASKS>)
        out[static_cast<int64_t>(f0) * p.r + e] = sum_at(e % p.r, e / p.r);
    }
  }
  cluster_sync();  // no CTA leaves while another reads its sums
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, pc.cols * pc.bufs);
  if (threadIdx.x == 0 && aborted) atomicOr(p.err, kErrTimeout);
}

template <int TASKS>
__global__ void __launch_bounds__(kGradThreads<TASKS>, 1) adapter_grad_kernel(const __grid_constant__ GradParams p) {
  extern __shared__ uint8_t grad_raw[];
  int tile = static_cast<int>(blockIdx.x) / p.splits, mi = 0;
  if (p.n_mem > 1) {
    const int first = (p.mem[0].width + kTileF - 1) / kTileF;
    if (tile >= first) {
      mi = 1;
      tile -= first;
    }
  }
  const int a = blockIdx.y;
  if (p.mem[mi].scale != nullptr)
    grad_tile<TASKS, true>(p, p.mem[mi], a, tile, grad_raw);
  else
    grad_tile<TASKS, false>(p, p.mem[mi], a, tile, grad_raw);
}

template <int TASKS>
cudaError_t launch_tasks(const GradParams& p, uint32_t smem, dim3 grid, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(adapter_grad_kernel<TASKS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kGradThreads<TASKS>);
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
  return cudaLaunchKernelEx(&cfg, adapter_grad_kernel<TASKS>, p);
}

}  // namespace

cudaError_t launch_adapter_grad(const GradParams& p, cudaStream_t stream) {
  GradParams q = p;
  int tiles = 0;
  bool codes = false;
  for (int i = 0; i < p.n_mem; ++i) {
    tiles += (p.mem[i].width + kTileF - 1) / kTileF;
    codes = codes || p.mem[i].scale != nullptr;
  }
  // Row splits: while the CTAs of the adapters in use are fewer than the SMs
  // hold at once and each split keeps two stages of rows.
  const int used = p.plan.cap < p.plan.n_req ? p.plan.cap : (p.plan.n_req > 0 ? p.plan.n_req : 1);
  const int rows = (p.plan.m + used - 1) / used;
  q.splits = 1;
  while (q.splits < 8 && static_cast<long long>(tiles) * used * q.splits < 148 && rows > 2 * kRows * q.splits * 2)
    q.splits *= 2;
  uint32_t smem = grad_geo(p.rp, false).smem;
  if (codes) {
    const uint32_t s = grad_geo(p.rp, true).smem;
    smem = s > smem ? s : smem;
  }
  const dim3 grid(tiles * q.splits, p.plan.cap);
  if (p.rp <= 32) return launch_tasks<1>(q, smem, grid, stream);
  if (p.rp <= 64) return launch_tasks<2>(q, smem, grid, stream);
  return launch_tasks<4>(q, smem, grid, stream);
}

}  // namespace mp
