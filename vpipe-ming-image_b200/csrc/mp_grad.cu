// Gradients of the factors of many adapters: matrix products grouped by
// adapter, over the ragged row ranges of its requests,
//
//   out[a] = sum over the rows t of adapter a of x[t]^T u[t],
//
// dA from x (bf16, or its 8-bit checkpoint) and u = s dy B, dB from dy and
// v = s x A^T. Bound by memory: x and dy are read once, 2 r operations for
// every byte or two of them.
//
// An item is one adapter and 128 features. Per 64 of its rows: x by TMA, [64
// rows][64 features] boxes that are the MN-major A operand of tcgen05 as they land
// (M = features, K = rows); u, f32, by TMA too, is cut by warps 2-9 into three bf16
// parts of 8 bits each, side by side in the N of the B operand: the products are
// then those of the f32 values, and cost no second pass over x.
//
// tcgen05 adds to its f32 accumulator without rounding to nearest: over a long
// run of rows the sums drift towards zero (2e-6 at 1000 rows). So an accumulator
// takes kChunk stages (256 rows) only; the last warps then add it, the three
// parts smallest first, to sums in registers, while the MMAs fill the other one.
//
// With many items the CTAs are persistent: they walk the items, the loads of the
// next one running while the last warps write this one's sums. With few, a cluster
// takes one item, its CTAs the row tiles in turn, and they add their sums through
// distributed shared memory, in CTA order.
//
// A checkpoint's codes are whole numbers of up to 8 bits, exact in bf16: warps
// 2-9 widen them, and the scale of a (row, 128 features) goes into u, in f32.
//
// Measured: 88 us for 16896 rows 3840 x 3840, 24 requests, 16 adapters of up to 64
// ranks (x and dy once, 260 MB, at 3.0 TB/s), 129 with x in 8 bits; 24 us for 4352
// rows, 4 adapters of 16, x in 8 bits (2.1 TB/s). What bounds it is not HBM but
// cutting u: a stage's u is cut anew for each 128 features, 60 times here, and a CTA
// takes 0.6 us a stage for its chain of copies, parts, MMAs and sums.
#include <cuda_runtime.h>

#include <cmath>

#include "mp_device.cuh"
#include "mp_kernels.h"
#include "mp_launch.h"

namespace mp {

namespace {

constexpr int kTileF = 128;   // features of a CTA (MMA M) and of a checkpoint scale
constexpr int kRows = 64;     // rows of a stage (four MMA K steps)
constexpr int kParts = 3;     // bf16 parts of an f32 value
static_assert(kTileF == kCkGroup, "one scale per row of a tile");

constexpr int kChunk = 4;     // stages of an accumulator

constexpr int kConvWarp0 = 2;
constexpr int kConvThreads = 256;
constexpr int kConvGroups = 2;  // of four warps: the even slots' and the odd slots'
constexpr int kConvGroup = kConvThreads / kConvGroups;
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
constexpr int kMaxGradSplits = 8;
constexpr uint32_t kGradSmemMost = 226 * 1024;

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

// A cluster's sums in the exchange buffer, four next to one another as the output
// has them: dA [rank][feature]; dB [feature][rank], with four more floats that put
// the 16 bytes of eight features into different banks.
__host__ __device__ inline int exchange_ld(bool rank_major, int rp) { return rank_major ? kTileF : rp + 4; }

// A stage: x as the A operand | u's parts, the B operand | u, f32 | with a
// checkpoint its codes and the rows' scales.
struct GradGeo {
  int stages;
  uint32_t parts_off, u_off, code_off, scale_off, stage_bytes;
  uint32_t smem;
};

__host__ __device__ inline GradGeo grad_geo(int rp, bool codes) {
  GradGeo g;
  const PartCols pc = part_cols(rp);
  g.parts_off = kXBytes;
  g.u_off = g.parts_off + pc.boxes * kBoxBytes;
  g.code_off = g.u_off + kRows * rp * 4;
  g.scale_off = g.code_off + (codes ? kCodeBytes : 0);
  g.stage_bytes = (g.scale_off + (codes ? kRows * 4 : 0) + 1023) / 1024 * 1024;
  // two CTAs an SM with up to 32 ranks (their accumulators take half of TMEM each)
  const uint32_t half = 113 * 1024;
  const bool two = rp <= 32 && 2 * g.stage_bytes + 1280 <= half;
  g.stages = static_cast<int>(((two ? half : kGradSmemMost) - 1280) / g.stage_bytes);
  if (g.stages > kMaxGradStages) g.stages = kMaxGradStages;
  const uint32_t tiles = g.stages * g.stage_bytes;
  const uint32_t exchange = kTileF * (rp + 4) * 4;
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

// The next bf16 part of two values, which keep what is left of them. Parts are cut
// off towards zero, 8 bits each, and the rest is taken 2^-24 of the part too large:
// so all parts of a value that is not 0 have its sign and none is 0, and an infinity
// in x meets three that agree (0 would make it a NaN, the other sign inf - inf). In
// all they are the value and up to 2^-24 of it, half a unit in its last place.
__device__ __forceinline__ uint32_t take_part(float& a, float& b) {
  constexpr float kLess = -0.99999994f;  // 2^-24 - 1
  const uint32_t wa = __float_as_uint(a), wb = __float_as_uint(b);
  a = fmaf(__uint_as_float(wa & 0xFFFF0000u), kLess, a);
  b = fmaf(__uint_as_float(wb & 0xFFFF0000u), kLess, b);
  return __byte_perm(wa, wb, 0x7632);
}

// `f`, or with its sign f32's largest where it is an infinity. A NaN stays one.
__device__ __forceinline__ float no_infinity(float f) {
  float d;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(d) : "f"(f), "f"(3.4028235e38f));
  return d;
}

// 4 bytes, asynchronously; and their arrival on an mbarrier whose count has a
// place for this thread.
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
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

// An item: its adapter, member and feature tile. The adapters with the most rows
// come first.
struct Item {
  int a, f_tile;
  const GradMember* mb;
};

__device__ __forceinline__ Item item_of(const GradParams& p, int i) {
  Item it;
  const int place = i / p.tiles;
  it.a = p.plan.by_rows[place];
  int t = i - place * p.tiles;
  const int first = (p.mem[0].width + kTileF - 1) / kTileF;
  const bool second = p.n_mem > 1 && t >= first;
  it.mb = &p.mem[second ? 1 : 0];
  it.f_tile = second ? t - first : t;
  return it;
}

// The items of worker `w` of `workers`: one of each round, the rounds to and fro,
// so that whoever has the larger one of a round has the smaller one of the next
// (the rounds descend in rows). At 24 requests on 16 adapters the busiest of 148
// then has 8 % more rows than the average, 35 % more without.
struct ItemIter {
  int round, w, workers, items;
  __device__ ItemIter(const GradParams& p, int w_, int workers_) : round(0), w(w_), workers(workers_), items(p.items) {}
  // The next item, or -1.
  __device__ __forceinline__ int next() {
    const int first = round * workers, i = first + (round & 1 ? workers - 1 - w : w);
    ++round;
    return first < items && i < items ? i : -1;  // only the last round can be short
  }
};

// Warps 2-9, in two groups: a stage's work is a chain of latencies (its copies'
// arrival, shared memory, the conversions, the fence), so two stages are worked on
// at once. TASKS: 16-value pieces of a 64-row stage of u per thread. CODES: a
// member's x is a checkpoint (an instantiation of its own, so that the others do
// not carry its steps).
template <int TASKS, bool CODES>
__device__ void convert(const GradParams& p, const GradSmem& sm, const GradGeo& geo, const PartCols& pc, int item0,
                        int step, int rank, int count) {
  const int tid = (threadIdx.x - 32 * kConvWarp0) % kConvGroup, lane = threadIdx.x & 31;
  const int group = (threadIdx.x - 32 * kConvWarp0) / kConvGroup;
  const int per_row = p.rp / 8, pieces = kRows * per_row;
  constexpr int kPieces = TASKS * kConvGroups;
  int row_of[kPieces], col_of[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int e = tid + j * kConvGroup;
    row_of[j] = e < pieces ? e / per_row : kRows;  // kRows: no piece
    col_of[j] = e < pieces ? e % per_row * 8 : 0;
  }
  // one answer for the warp, so that all of its lanes give up together
  auto wait_all = [&](uint32_t bar, uint32_t parity, uint32_t site) {
    return __all_sync(0xFFFFFFFFu, mbar_wait<true>(bar, parity, sm.abort, site, p.wait_limit_ns)) != 0;
  };
  RingPos at_stage;
  ItemIter items(p, item0, step);
  for (int i = items.next(); i >= 0; i = items.next()) {
    const Item item = item_of(p, i);
    const bool codes = CODES && item.mb->scale != nullptr;
    TileIter it(p.plan, item.a, rank, count);
    int t0, rows;
    for (; it.next(t0, rows); at_stage.next(geo.stages)) {
      // A slot is one group's for good: it then waits for each of the slot's phases,
      // and none can pass without its arrival. (Stages in turn over an odd number
      // of slots would have a group wait for every second phase of a slot, which a
      // parity cannot tell from the one before.)
      if (at_stage.slot % kConvGroups != group) continue;
      const int s = at_stage.slot;
      const uint32_t ph = at_stage.phase;
      // the tile has landed (so the stage's last MMAs are done)
      if (!wait_all(smem_u32(&sm.full[s]), ph, kSiteGradFull | s)) return;
      const uint32_t xs = sm.tiles + s * geo.stage_bytes, parts = xs + geo.parts_off;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        if (row_of[j] >= kRows) continue;
        // rows past the segment's last are another request's: zeros
        float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (row_of[j] < rows) {
          const uint32_t at = xs + geo.u_off + (row_of[j] * p.rp + col_of[j]) * 4u;
          const float4 a = ld_shared_f4(at), b = ld_shared_f4(at + 16);
          f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
          f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        }
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
        if (codes && row_of[j] < rows) {
          float by;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(by) : "r"(xs + geo.scale_off + row_of[j] * 4u));
          // u times the scale. A product past f32's largest stays there: a code of 0
          // then gives 0, not the NaN of 0 and an infinity
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = no_infinity(f[e] * by);
        }
        const uint32_t row = parts + row_of[j] * 128u, sw = static_cast<uint32_t>(row_of[j] & 7);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = take_part(f[2 * e], f[2 * e + 1]);
          const uint32_t col = col_of[j] + (part == 2 ? pc.third : part * p.rp);
          st_shared_v4(row + (col >> 6) * kBoxBytes + (((col >> 3 & 7u) ^ sw) << 4), w[0], w[1], w[2], w[3]);
        }
        if (isinf(top)) {
          // all parts of an infinite u are what it is (inf - inf gave NaN)
#pragma unroll 1
          for (int e = col_of[j]; e < col_of[j] + 8; ++e) {
            float u, by = 1.0f;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(u) : "r"(xs + geo.u_off + (row_of[j] * p.rp + e) * 4u));
            if (!isinf(u)) continue;
            if (codes) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(by) : "r"(xs + geo.scale_off + row_of[j] * 4u));
            const uint16_t v = static_cast<uint16_t>(__float_as_uint(u * by) >> 16);
#pragma unroll 1
            for (int part = 0; part < kParts; ++part) {
              const uint32_t col = e + (part == 2 ? pc.third : part * p.rp);
              const uint32_t at = row + (col >> 6) * kBoxBytes + (((col >> 3 & 7u) ^ sw) << 4) + (col & 7u) * 2u;
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(v) : "memory");
            }
          }
        }
      }
      if (codes) {
#pragma unroll
        for (int j = 0; j < kRows * kTileF / 16 / kConvGroup; ++j) {  // 16 codes of a row at a time
          const int e = tid + j * kConvGroup, row = e / (kTileF / 16), c = e % (kTileF / 16);
          uint4 q = ld_shared_v4(xs + geo.code_off + row * kTileF + c * 16);
          if (row >= rows) q = make_uint4(0, 0, 0, 0);
          const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
          const uint64_t less = f32x2(-32896.0f, -32896.0f);
          uint32_t w[8];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            // byte b + 128 as the float 32768 + (b + 128), less 32896: exact
            const uint32_t ofs = qw[h] ^ 0x80808080u;
            auto code = [&](uint32_t sel) { return __uint_as_float(__byte_perm(ofs, 0x4700u, sel)); };
            w[2 * h] = f32x2_to_bf16x2(add_f32x2(f32x2(code(0x5404u), code(0x5414u)), less));
            w[2 * h + 1] = f32x2_to_bf16x2(add_f32x2(f32x2(code(0x5424u), code(0x5434u)), less));
          }
          const uint32_t at = xs + (c >> 2) * kBoxBytes + row * 128u, ch = static_cast<uint32_t>(2 * (c & 3));
          const uint32_t sw = static_cast<uint32_t>(row & 7);
          st_shared_v4(at + ((ch ^ sw) << 4), w[0], w[1], w[2], w[3]);
          st_shared_v4(at + (((ch + 1) ^ sw) << 4), w[4], w[5], w[6], w[7]);
        }
      } else if (rows < kRows) {
        // an infinity or NaN in the rows after the segment's last would come
        // through a product with 0
        for (int e = rows * 8 + tid; e < kRows * 8; e += kConvGroup) {
          st_shared_v4(xs + e * 16, 0, 0, 0, 0);
          st_shared_v4(xs + kBoxBytes + e * 16, 0, 0, 0, 0);
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.conv[s]));
    }
  }
}

// Registers: two CTAs an SM at up to 32 ranks leave 72 a thread, the 576 threads of
// more than 64 ranks 96; 72 and 132 bytes a thread spill, at 64 ranks none.
template <int TASKS, bool CODES>
__global__ void __launch_bounds__(kGradThreads<TASKS>, TASKS == 1 ? 2 : 1)
    adapter_grad_kernel(const __grid_constant__ GradParams p) {
  extern __shared__ uint8_t grad_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = p.splits, rank = count > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int item0 = static_cast<int>(blockIdx.x) / count, clusters = static_cast<int>(gridDim.x) / count;
  const int step = p.workers;
  const int col0 = warp >= kSumWarp0 + 4 ? kSumCols<TASKS> : 0;  // the adding warp's first rank
  const PartCols pc = part_cols(p.rp);
  const GradGeo geo = grad_geo(p.rp, CODES);
  GradSmem sm;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(grad_raw) + 1023u) & ~uintptr_t(1023u));
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
  // Zeros of item i (an adapter without rows) by this cluster's threads.
  auto clear_item = [&](int i) {
    const int tid = rank * kGradThreads<TASKS> + threadIdx.x, threads = count * kGradThreads<TASKS>;
    const Item item = item_of(p, i);
    const int f0 = item.f_tile * kTileF, width = min(kTileF, item.mb->width - f0);
    float* out = item.mb->out + static_cast<int64_t>(item.a) * p.r * item.mb->width;
    if (item.mb->rank_major) {
      out += f0;
      const bool quads = ((reinterpret_cast<uintptr_t>(out) | item.mb->width * 4u | width * 4u) & 15u) == 0;
      for (int r = tid >> 5; r < p.r; r += threads >> 5) {
        float* row = out + static_cast<int64_t>(r) * item.mb->width;
        if (quads) {
          if (lane * 4 < width) *reinterpret_cast<float4*>(row + lane * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        } else {
          for (int f = lane; f < width; f += 32) row[f] = 0.0f;
        }
      }
    } else {
      out += static_cast<int64_t>(f0) * p.r;
      const int n = width * p.r;
      if (((reinterpret_cast<uintptr_t>(out) | n * 4u) & 15u) == 0) {
        for (int e = tid * 4; e < n; e += threads * 4)
          *reinterpret_cast<float4*>(out + e) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      } else {
        for (int e = tid; e < n; e += threads) out[e] = 0.0f;
      }
    }
  };
  if (item0 >= p.workers) {
    // clusters of their own clear the adapters that are more than the requests
    pdl_wait();
    pdl_release();
    for (int i = p.items + item0 - p.workers; i < p.all_items; i += clusters - p.workers) clear_item(i);
    return;
  }
  if (count > 1) {
    // clusters of adapters without rows leave before any set-up
    pdl_wait();
    const Item item = item_of(p, item0);
    if (p.plan.begin[item.a] == p.plan.begin[item.a + 1]) {
      pdl_release();
      clear_item(item0);
      return;
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < geo.stages; ++s) {
      mbar_init(smem_u32(&sm.full[s]), 33);  // the producer's lane 0 with the copies' bytes, and every lane
      mbar_init(smem_u32(&sm.conv[s]), kConvGroup / 32);
      mbar_init(smem_u32(&sm.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sm.sum[b]), 1);
      mbar_init(smem_u32(&sm.taken[b]), kSumWarps<TASKS>);
    }
    mbar_init(smem_u32(sm.done), 1);
    *sm.abort = 0u;
    fence_mbar_init();
    for (int i = 0; i < p.n_mem; ++i) {
      tma_prefetch_map(&p.mem[i].tm_x);
      tma_prefetch_map(&p.mem[i].tm_u);
    }
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

  if (warp == 0) {
    RingPos at_stage;
    int sent = 0;
    bool ok = true;
    ItemIter items(p, item0, step);
    for (int i = items.next(); i >= 0 && ok; i = items.next()) {
      const Item item = item_of(p, i);
      const GradMember& mb = *item.mb;
      const bool codes = CODES && mb.scale != nullptr;
      TileIter it(p.plan, item.a, rank, count);
      int t0, rows;
      for (; ok && it.next(t0, rows); at_stage.next(geo.stages), ++sent) {
        const int s = at_stage.slot;
        if (at_stage.uses > 0)
          ok = __all_sync(0xFFFFFFFFu, mbar_wait<true>(smem_u32(&sm.empty[s]), at_stage.phase ^ 1u, sm.abort,
                                                       kSiteGradEmpty | s, p.wait_limit_ns)) != 0;
        if (!ok) break;
        const uint32_t bar = smem_u32(&sm.full[s]), xs = sm.tiles + s * geo.stage_bytes;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, kRows * p.rp * 4 + (codes ? kCodeBytes : kXBytes));
          tma_load_2d(xs + geo.u_off, &mb.tm_u, bar, 0, t0);
          if (codes) {
            tma_load_2d(xs + geo.code_off, &mb.tm_x, bar, item.f_tile * kTileF, t0);
          } else {
            tma_load_2d(xs, &mb.tm_x, bar, item.f_tile * kTileF, t0);
            tma_load_2d(xs + kBoxBytes, &mb.tm_x, bar, item.f_tile * kTileF + 64, t0);
          }
        }
        if (codes) {
          const float* scale = mb.scale + static_cast<int64_t>(item.f_tile) * p.plan.m + t0;
          for (int r = lane; r < rows; r += 32) cp_async_4(xs + geo.scale_off + r * 4u, scale + r);
        }
        cp_async_arrive(bar);
      }
    }
    if (*sm.abort != 0u && lane == 0) {
      // copies in flight land (bounded) before the CTA leaves
      const uint64_t since = global_timer_ns();
      for (int j = max(0, sent - geo.stages); j < sent; ++j)
        while (!mbar_try_wait(smem_u32(&sm.full[j % geo.stages]), (j / geo.stages) & 1u))
          if (global_timer_ns() - since > p.wait_limit_ns) break;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t mn = (1u << 15) | (1u << 16);  // both operands MN-major
      const uint32_t id1 = make_idesc_bf16(kTileF, pc.n1) | mn, id2 = make_idesc_bf16(kTileF, pc.n2) | mn;
      RingPos at_stage, at_acc;  // stages and accumulators filled
      bool ok = true;
      ItemIter items(p, item0, step);
      for (int i = items.next(); i >= 0 && ok; i = items.next()) {
        const int tiles = TileIter(p.plan, item_of(p, i).a, rank, count).total();
        for (int k = 0; k < tiles; ++k, at_stage.next(geo.stages)) {
          const int s = at_stage.slot, b = at_acc.slot;
          const uint32_t ph = at_stage.phase;
          const bool first = k % kChunk == 0, last = k % kChunk == kChunk - 1 || k == tiles - 1;
          if (first && at_acc.uses > 0)
            ok = mbar_wait<true>(smem_u32(&sm.taken[b]), at_acc.phase ^ 1u, sm.abort, kSiteGradTaken | b, p.wait_limit_ns);
          // the converting warps arrive after the tile has landed
          ok = ok && mbar_wait<true>(smem_u32(&sm.full[s]), ph, sm.abort, kSiteGradFull | s, p.wait_limit_ns) &&
               mbar_wait<true>(smem_u32(&sm.conv[s]), ph, sm.abort, kSiteGradConv | s, p.wait_limit_ns);
          if (!ok) break;
          tc_fence_after();
          const uint32_t xs = sm.tiles + s * geo.stage_bytes, us = xs + geo.parts_off, d = tmem + b * pc.cols;
#pragma unroll
          for (int kk = 0; kk < kRows / 16; ++kk) {
            const uint32_t acc = !first || kk > 0 ? 1u : 0u;
            umma_ss(d, mn_desc(xs, kk), mn_desc(us, kk), id1, acc);
            if (pc.n2 > 0)
              umma_ss(d + pc.third, mn_desc(xs, kk), mn_desc(us + (pc.third >> 6) * kBoxBytes, kk), id2, acc);
          }
          umma_commit(smem_u32(&sm.empty[s]));
          if (last) {
            umma_commit(smem_u32(&sm.sum[b]));
            at_acc.next(pc.bufs);
          }
        }
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
    convert<TASKS, CODES>(p, sm, geo, pc, item0, step, rank, count);
  } else {
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int f = (warp & 3) * 32 + lane;
    float sums[kSumCols<TASKS>];  // one feature, consecutive ranks
    RingPos at_acc;
    bool ok = true;
    ItemIter items(p, item0, step);
    for (int i = items.next(); i >= 0 && ok; i = items.next()) {
      const Item item = item_of(p, i);
      const int tiles = TileIter(p.plan, item.a, rank, count).total();
#pragma unroll
      for (int c = 0; c < kSumCols<TASKS>; ++c) sums[c] = 0.0f;
      for (int k = 0; k < tiles; k += kChunk, at_acc.next(pc.bufs)) {
        const int b = at_acc.slot;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait<true>(smem_u32(&sm.sum[b]), at_acc.phase, sm.abort, kSiteGradSum | b,
                                                     p.wait_limit_ns)) != 0;
        if (!ok) break;
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
      bool nan = false;
#pragma unroll
      for (int c = 0; c < kSumCols<TASKS>; ++c) nan = nan || sums[c] != sums[c];
      if (nan) {
        // past the adapter's own ranks u is 0: so are the sums, whatever x held
        const int own = p.info[item.a].rank;
#pragma unroll
        for (int c = 0; c < kSumCols<TASKS>; ++c) sums[c] = col0 + c < own ? sums[c] : 0.0f;
      }
      if (count > 1 || !ok) break;  // a cluster has one item
      const int ff = item.f_tile * kTileF + f;
      if (ff < item.mb->width) {
        float* out = item.mb->out + static_cast<int64_t>(item.a) * p.r * item.mb->width;
        if (item.mb->rank_major) {
#pragma unroll
          for (int c = 0; c < kSumCols<TASKS>; ++c)
            if (col0 + c < p.r) out[static_cast<int64_t>(col0 + c) * item.mb->width + ff] = sums[c];
        } else {
          float* row = out + static_cast<int64_t>(ff) * p.r + col0;
          if (p.r % 4 == 0) {  // whole 16-byte pieces (the output is 16-byte aligned)
#pragma unroll
            for (int c = 0; c < kSumCols<TASKS>; c += 4)
              if (col0 + c < p.r)
                *reinterpret_cast<float4*>(row + c) = make_float4(sums[c], sums[c + 1], sums[c + 2], sums[c + 3]);
          } else {
#pragma unroll
            for (int c = 0; c < kSumCols<TASKS>; ++c)
              if (col0 + c < p.r) row[c] = sums[c];
          }
        }
      }
    }
    // every copy has landed and every MMA is done (or the CTA gave up): the
    // stages' memory takes a cluster's sums
    named_barrier(kAllBarrier, kGradThreads<TASKS>);
    if (count > 1) {
      const bool rank_major = item_of(p, item0).mb->rank_major != 0;
      const int ld = exchange_ld(rank_major, p.rp);
#pragma unroll
      for (int c = 0; c < kSumCols<TASKS>; c += 4) {
        if (col0 + c >= p.rp) break;
        if (rank_major) {
#pragma unroll
          for (int j = 0; j < 4; ++j) sm.exchange[(col0 + c + j) * ld + f] = sums[c + j];
        } else {
          *reinterpret_cast<float4*>(sm.exchange + f * ld + col0 + c) =
              make_float4(sums[c], sums[c + 1], sums[c + 2], sums[c + 3]);
        }
      }
    }
  }
  __syncwarp();
  if (warp < kSumWarp0) named_barrier(kAllBarrier, kGradThreads<TASKS>);
  const bool aborted = *sm.abort != 0u;
  if (count > 1) {
    cluster_sync();
    if (!aborted) {
      // the CTAs share the adding up: each takes some ranks (dA) or features (dB)
      const Item item = item_of(p, item0);
      const GradMember& mb = *item.mb;
      const int ld = exchange_ld(mb.rank_major != 0, p.rp);
      const int f0 = item.f_tile * kTileF, width = min(kTileF, mb.width - f0);
      float* out = mb.out + static_cast<int64_t>(item.a) * p.r * mb.width;
      const uint32_t ex = smem_u32(sm.exchange);
      auto sums_at = [&](int e) {
        const uint32_t at = ex + static_cast<uint32_t>(e) * 4u;
        float4 o[kMaxGradSplits];  // all in flight, then added in CTA order
#pragma unroll
        for (int z = 0; z < kMaxGradSplits; ++z)
          if (z < count) o[z] = ld_cluster_f4(mapa_shared(at, z));
        float4 s = o[0];
#pragma unroll
        for (int z = 1; z < kMaxGradSplits; ++z)
          if (z < count) s.x += o[z].x, s.y += o[z].y, s.z += o[z].z, s.w += o[z].w;
        return s;
      };
      // the `n` first of four sums, 16 bytes at once where they all are and may be
      auto put = [&](float* to, float4 s, int n) {
        if (n >= 4 && (reinterpret_cast<uintptr_t>(to) & 15u) == 0) {
          *reinterpret_cast<float4*>(to) = s;
        } else {
          if (n > 0) to[0] = s.x;
          if (n > 1) to[1] = s.y;
          if (n > 2) to[2] = s.z;
          if (n > 3) to[3] = s.w;
        }
      };
      if (mb.rank_major) {
        for (int e = threadIdx.x; (e >> 5) * count + rank < p.r; e += kGradThreads<TASKS>) {
          const int r = (e >> 5) * count + rank, f = (e & 31) * 4;
          if (f < width) put(out + static_cast<int64_t>(r) * mb.width + f0 + f, sums_at(r * ld + f), width - f);
        }
      } else {
        const int quads = (p.r + 3) / 4, per = kTileF / count, lo = rank * per, hi = min(lo + per, width);
        for (int e = threadIdx.x; e < (hi - lo) * quads; e += kGradThreads<TASKS>) {
          const int f = lo + e / quads, r = e % quads * 4;
          put(out + static_cast<int64_t>(f0 + f) * p.r + r, sums_at(f * ld + r), p.r - r);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, pc.cols * pc.bufs);
  if (threadIdx.x == 0 && aborted) atomicOr(p.err, kErrTimeout);
}

template <int TASKS, bool CODES>
cudaError_t launch_tasks(const GradParams& p, uint32_t smem, unsigned grid, cudaStream_t stream) {
  static SmemOptIn opted;
  cudaError_t e = opted.allow(reinterpret_cast<const void*>(adapter_grad_kernel<TASKS, CODES>));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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
  return cudaLaunchKernelEx(&cfg, adapter_grad_kernel<TASKS, CODES>, p);
}

// CTAs that share an adapter's rows: the least of rounds x (9 us a CTA and 0.6 us a
// stage) and 1.5 us + 0.15 us a CTA for a cluster's joining. An SM takes `per_sm`
// CTAs, the GPU 148, 74, 33, 15 clusters of 1, 2, 4, 8 of them; the `rest` items that
// are only cleared count for half a CTA each. What the host does not know is put at
// what it is for requests that pick their adapters at random: how many adapters
// have rows, and that the one with the most has 1.7 times the average. With 1, 2,
// 4, 8 CTAs the launch takes 85, 49, 31, 21 us at 7713 rows 440 x 576, 2 adapters of
// 56 ranks; 135, 75, 44, 52 at 13705 rows 288 x 2880, 2 of 48; 36, 24, 31, 52 at 4352
// rows 3840 x 3840, 4 of 16 (8 bit); 16, 25, 40, 75 at 1954 rows 832 x 1600, 6 of 52.
int choose_splits(const RequestPlan& pl, int tiles, int rest, int per_sm) {
  const double live = pl.cap * (1.0 - std::pow(1.0 - 1.0 / pl.cap, pl.n_req > 0 ? pl.n_req : 1));
  const double stages = std::fmax((1.7 - 0.7 / live) * pl.m / (live * kRows), pl.n_req / live);
  int best = 1;
  double best_us = 1e300;
  for (int s = 1; s <= kMaxGradSplits; s *= 2) {
    const double room = per_sm * s * (s == 1 ? 148 : s == 2 ? 74 : s == 4 ? 33 : 15);
    const double ctas = tiles * live * s + 0.5 * std::fmin(148.0, static_cast<double>(rest) * s);
    const double us = std::fmax(1.0, ctas / room) * (9.0 + 0.6 * stages / s) + (s > 1 ? 1.5 + 0.15 * s : 0.0);
    if (us < best_us) {
      best_us = us;
      best = s;
    }
  }
  return best;
}

}  // namespace

cudaError_t launch_adapter_grad(const GradParams& p, cudaStream_t stream) {
  GradParams q = p;
  q.tiles = 0;
  q.codes = 0;
  for (int i = 0; i < p.n_mem; ++i) {
    q.tiles += (p.mem[i].width + kTileF - 1) / kTileF;
    if (p.mem[i].scale != nullptr) q.codes = 1;
  }
  const long long all_items = static_cast<long long>(q.tiles) * p.plan.cap;
  if (all_items > (1 << 30)) return cudaErrorInvalidValue;
  // Adapters come in the order of their rows, so those past the number of
  // requests have none: their gradients are cleared by the way.
  const int used = p.plan.cap < p.plan.n_req ? p.plan.cap : (p.plan.n_req > 0 ? p.plan.n_req : 1);
  q.all_items = static_cast<int>(all_items);
  q.items = q.tiles * used;
  const GradGeo geo = grad_geo(p.rp, q.codes != 0);
  const int per_sm = geo.smem <= 113 * 1024 ? 2 : 1, room = 148 * per_sm, rest = q.all_items - q.items;
  q.splits = choose_splits(p.plan, q.tiles, rest, per_sm);
  q.workers = q.splits > 1 ? q.items : (q.items < room ? q.items : room);
  // Clusters of their own clear, beside those at work: with 10 of 12 adapters of
  // 3672 x 192 and 64 ranks to clear, the working CTAs doing it took the launch
  // from 10.6 to 26 us.
  const int most = (148 + q.splits - 1) / q.splits;
  const unsigned grid = static_cast<unsigned>(q.workers + (rest < most ? rest : most)) * q.splits;
  if (q.codes != 0) {
    if (p.rp <= 32) return launch_tasks<1, true>(q, geo.smem, grid, stream);
    if (p.rp <= 64) return launch_tasks<2, true>(q, geo.smem, grid, stream);
    return launch_tasks<4, true>(q, geo.smem, grid, stream);
  }
  if (p.rp <= 32) return launch_tasks<1, false>(q, geo.smem, grid, stream);
  if (p.rp <= 64) return launch_tasks<2, false>(q, geo.smem, grid, stream);
  return launch_tasks<4, false>(q, geo.smem, grid, stream);
}

}  // namespace mp
