// Adapters by request: the plan of a batch, the adapter bank's layout, and the
// rank-space rows of a batch whose requests each have an adapter of their own.
//
//   y[t] = W x[t] + s_q B_a (A_a x[t])      row t of request q, adapter a = a_q
//
// The product with W and the one with B_a are one pass of the projection
// kernel (mp_proj.cu), which takes each token tile's adapters as appended K
// tiles; what is here computes v[t] = s_q A_a x[t] for it and, in the backward
// pass, u[t] = s_q B_a^T dy[t] (the same kernel on the transposed factors).
#include <cuda_runtime.h>

#include "mp_device.cuh"
#include "mp_kernels.h"

namespace mp {

namespace {

// ---- plan --------------------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int kPerThread = kMaxRequests / kPlanThreads;

// Exclusive prefix sum over the block of each thread's kPerThread values, in place.
__device__ void scan_block(int (&v)[kPerThread], int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) sum += v[i];
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xFFFFFFFFu, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int w = warp_sums[lane];
    int wi = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, wi, d);
      if (lane >= d) wi += o;
    }
    warp_sums[lane] = wi - w;
  }
  __syncthreads();
  int at = warp_sums[warp] + inc - sum;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int x = v[i];
    v[i] = at;
    at += x;
  }
  __syncthreads();
}

// Largest q with start[q] <= row, over start[0 .. n] (start[0] = 0).
__device__ __forceinline__ int last_at(const int* start, int n, int row) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= row)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Bound by the latency of its scans and of the writes between them: 9 us for one
// request, 20 us for 15 over 12346 rows, once a batch for all projections.
// One block: lengths are clamped to [0, what is left of m] and adapters
// outside [-1, cap) dropped (kErrRequests then tells the host). All outputs
// are integers in a fixed order, the same for the same inputs.
__global__ void __launch_bounds__(kPlanThreads) plan_requests_kernel(const __grid_constant__ PlanParams p) {
  __shared__ int start[kMaxRequests + 1];
  __shared__ int adapter[kMaxRequests];
  __shared__ uint16_t tiles_of[kMaxAdapters];  // tiles of 64 rows (at most 2^13 + kMaxRequests)
  __shared__ int warp_sums[32];
  const RequestPlan& pl = p.plan;
  const int n = pl.n_req, tid = threadIdx.x;
  pdl_wait();
  pdl_release();

  int len[kPerThread], at[kPerThread];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int q = tid * kPerThread + i;
    int l = q < n ? p.lengths[q] : 0;
    if (l < 0 || l > pl.m) {
      bad = true;
      l = l < 0 ? 0 : pl.m;
    }
    len[i] = at[i] = l;
  }
  // lengths are at most m < 2^31 / kMaxRequests, so their sum fits
  scan_block(at, warp_sums);
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int q = tid * kPerThread + i;
    if (at[i] + len[i] > pl.m) bad = true;
    if (q < n) start[q] = min(at[i], pl.m);
    if (q == n - 1) start[n] = min(at[i] + len[i], pl.m);
  }
  if (n == 0 && tid == 0) start[0] = 0;
  __syncthreads();
  int chunks[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int q = tid * kPerThread + i;
    chunks[i] = 0;
    if (q >= n) continue;
    int a = p.adapters[q];
    if (a < -1 || a >= pl.cap) {
      bad = true;
      a = -1;
    }
    const int rows = start[q + 1] - start[q];
    if (rows == 0 || (p.strengths != nullptr && p.strengths[q] == 0.0f)) a = -1;
    adapter[q] = a;
    if (a >= 0) chunks[i] = (rows + kChunkRows - 1) / kChunkRows;
  }
  if (bad) atomicOr(p.err, kErrRequests);
  __syncthreads();

  // chunks of the live requests' rows
  const int n_chunk = plan_chunks(pl.m, n);
  int chunk_at[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) chunk_at[i] = chunks[i];
  scan_block(chunk_at, warp_sums);
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int q = tid * kPerThread + i;
    if (q >= n) continue;
    const float s = p.strengths != nullptr ? p.strengths[q] : 1.0f;
    for (int c = 0; c < chunks[i]; ++c) {
      const int r0 = start[q] + c * kChunkRows;
      const int rows = min(kChunkRows, start[q + 1] - r0);
      pl.chunk[chunk_at[i] + c] = make_int4(r0, rows | (q << 8), adapter[q], __float_as_int(s));
    }
  }
  if (tid == kPlanThreads - 1) warp_sums[0] = chunk_at[kPerThread - 1] + chunks[kPerThread - 1];
  __syncthreads();
  for (int i = warp_sums[0] + tid; i < n_chunk; i += kPlanThreads) pl.chunk[i] = make_int4(0, 0, -1, 0);

  // row ranges by adapter: a live request's place is the number of live ones
  // that have a lower adapter, or the same one and come before it
  for (int q = tid; q < n; q += kPlanThreads) {
    const int a = adapter[q];
    if (a < 0) continue;
    int place = 0;
    for (int j = 0; j < n; ++j) {
      const int b = adapter[j];
      place += (b >= 0 && (b < a || (b == a && j < q))) ? 1 : 0;
    }
    pl.seg[place] = make_int2(start[q], start[q + 1]);
  }
  for (int a = tid; a <= pl.cap; a += kPlanThreads) {
    int below = 0, tiles = 0;
    for (int j = 0; j < n; ++j) {
      below += (adapter[j] >= 0 && adapter[j] < a) ? 1 : 0;
      if (adapter[j] == a) tiles += (start[j + 1] - start[j] + 63) / 64;
    }
    pl.begin[a] = below;
    if (a < pl.cap) tiles_of[a] = static_cast<uint16_t>(tiles);
  }
  __syncthreads();
  for (int a = tid; a < pl.cap; a += kPlanThreads) {
    const int mine = tiles_of[a];
    int place = 0;
    for (int b = 0; b < pl.cap; ++b) place += (tiles_of[b] > mine || (tiles_of[b] == mine && b < a)) ? 1 : 0;
    pl.by_rows[place] = a;
  }

  for (int r = tid; r < min(pl.m, kFewRows); r += kPlanThreads)
    pl.row_adapter[r] = r < start[n] ? adapter[last_at(start, n, r)] : -1;

  // blocks and lists of every level's token tiles
  for (int l = 0; l < kPlanLevels; ++l) {
    const int tile = 64 << l, tiles = plan_tiles(pl.m, l), blocks = plan_blocks(pl.m, n, l);
    for (int b = tid; b < blocks; b += kPlanThreads) pl.block[l][b] = make_int4(-1, 0, 0, -1);
    __syncthreads();
    for (int t = tid; t < tiles; t += kPlanThreads) {
      const int row0 = t * tile, row1 = min(row0 + tile, pl.m);
      int live = 0, first = 0;
      if (row0 < start[n]) {
        const int q0 = last_at(start, n, row0);
        first = t + q0;
        for (int q = q0; q < n && start[q] < row1; ++q) {
          const int lo = max(start[q], row0), hi = min(start[q + 1], row1);
          if (lo >= hi) continue;
          pl.block[l][t + q] = make_int4(t, lo, hi, adapter[q]);
          if (adapter[q] < 0) continue;
          pl.block_s[l][t + q] = p.strengths != nullptr ? p.strengths[q] : 1.0f;
          pl.list[l][first + live] = make_int2(t + q, adapter[q]);
          ++live;
        }
      }
      if (row1 > start[n]) pl.block[l][t + n] = make_int4(t, max(start[n], row0), row1, -1);
      pl.first[l][t] = first;
      pl.live[l][t] = live;
    }
  }
}

// ---- adapter bank -------------------------------------------------------------

__device__ __forceinline__ bool finite_bf16(uint16_t v) { return (v & 0x7F80u) != 0x7F80u; }

// 32 x 32 tiles over [rows][cols]: `src` (pitch ld) in place, zeros past
// (rows_ok, cols_ok) and for values that are not finite; the transposed tile
// into `dst` ([cols_t][rows], pitch ld_t) when it is not null.
__device__ void finish_tile(uint16_t* src, int ld, uint16_t* dst, int ld_t, int rows, int cols, int rows_ok,
                            int cols_ok, int cols_t, int r0, int c0, int32_t* bad, uint16_t (&sm)[32][33]) {
  const int c = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < 32; r += 8) {
    uint16_t v = 0;
    if (r0 + r < rows && c0 + c < cols) {
      uint16_t* at = src + static_cast<size_t>(r0 + r) * ld + c0 + c;
      if (r0 + r < rows_ok && c0 + c < cols_ok) v = *at;
      if (!finite_bf16(v)) {
        v = 0;
        *bad = 1;
      }
      *at = v;
    }
    sm[r][c] = v;
  }
  __syncthreads();
  if (dst != nullptr) {
    for (int r = threadIdx.x >> 5; r < 32; r += 8)
      if (c0 + r < cols_t && r0 + c < rows) dst[static_cast<size_t>(c0 + r) * ld_t + r0 + c] = sm[c][r];
  }
}

__global__ void __launch_bounds__(256) bank_set_kernel(const __grid_constant__ BankSetParams p) {
  __shared__ uint16_t sm[32][33];
  const int rt = (p.rp + 31) / 32, kt = (p.kp + 31) / 32, nt = (p.n + 31) / 32;
  int i = blockIdx.x;
  if (i == 0 && threadIdx.x == 0) p.info->rank = p.rank;
  if (i < rt * kt) {  // A [rp][kp], transposed [k][rp]
    finish_tile(p.a, p.kp, p.at, p.rp, p.rp, p.kp, p.rank, p.k, p.k, i / kt * 32, i % kt * 32, &p.info->bad, sm);
  } else {  // B [n][rp], transposed [rp][np]
    i -= rt * kt;
    if (i < rt * nt)
      finish_tile(p.b, p.rp, p.bt, p.np, p.n, p.rp, p.n, p.rank, p.rp, i / rt * 32, i % rt * 32, &p.info->bad, sm);
  }
}

// ---- rank-space rows, few at a time --------------------------------------------

// D[16][8] += A[16][16] B[16][8]: bf16 in, f32 out (the warp-wide fragments of mma.sync).
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D = A B (no accumulator to start from).
__device__ __forceinline__ void mma_16x8x16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// 16 bf16 values of a row from column c (a multiple of 16; the row is 16-byte
// aligned), zeros from column k on and where !ok: nothing past the k-th value
// is read.
__device__ __forceinline__ void load16(const uint16_t* row, int c, int k, bool ok, uint32_t (&w)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = c + 8 * h;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (ok && at + 8 <= k) {
      v = *reinterpret_cast<const uint4*>(row + at);
    } else if (ok && at < k) {
      uint16_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = at + j < k ? row[at + j] : static_cast<uint16_t>(0);
      v = make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16));
    }
    w[4 * h] = v.x;
    w[4 * h + 1] = v.y;
    w[4 * h + 2] = v.z;
    w[4 * h + 3] = v.w;
  }
}

constexpr int kRankWarps = 16;
constexpr int kRankBatch = 4;  // K groups a warp has in flight

// What no chunk writes of the plan's block `blk`: for a live request its block of
// vblk but for the request's rows and ranks, otherwise the rows of v32.
__device__ void clear_block(const RankParams& p, int blk, int tid, int threads) {
  const int4 ent = p.plan.block[p.lvl][blk];
  if (ent.w >= 0 && p.vblk != nullptr) {
    const int rows = 64 << p.lvl, row0 = ent.x << (6 + p.lvl), quads = p.ldb / 8, own = p.rp / 8;
    uint4* at = reinterpret_cast<uint4*>(p.vblk + (static_cast<int64_t>(blk) << (6 + p.lvl)) * p.ldb);
    for (int e = tid; e < rows * quads; e += threads) {
      const int r = row0 + e / quads;
      if (r < ent.y || r >= ent.z || e % quads >= own) at[e] = make_uint4(0, 0, 0, 0);
    }
  } else if (ent.w < 0 && p.clear_v32) {
    for (int e = tid; e < (ent.z - ent.y) * p.rp / 4; e += threads) {
      const int r = ent.y + e / (p.rp / 4), c = e % (p.rp / 4) * 4;
      *reinterpret_cast<float4*>(p.v32 + static_cast<int64_t>(r) * p.ld32 + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
  }
}

// One block: 16 ranks of one chunk (at most 8 rows of one request); its warps
// take the 64-wide K groups in turn and their sums are added in warp order. The
// blocks after the chunks' clear what no chunk writes.
// Within a group lane (g, j) (g = lane / 4, j = lane % 4) holds columns
// 16 j .. 16 j + 15 of ranks g and g + 8 and of row g: both operands of the
// four MMAs of a group then come from two 16-byte loads each, the K columns
// taken in the same order in both. With few rows a block or two have to fetch
// the whole factor, so what counts is the bytes each keeps in flight: 16 warps
// of four groups.
// Measured: 5 us for 16 requests of one row (3840 features, 32 ranks), 9.1 us for 1024
// rows in 4 requests; beyond, 0.022 us for every block more, of which 0.014 are left
// at 256 features: its start and the adding up.
__global__ void __launch_bounds__(32 * kRankWarps) rank_rows_kernel(const __grid_constant__ RankParams p) {
  __shared__ float part[kRankWarps][16][kChunkRows];
  pdl_wait();
  pdl_release();
  const int chunks = plan_chunks(p.plan.m, p.plan.n_req);
  if (static_cast<int>(blockIdx.x) >= chunks) {
    if (blockIdx.y == 0) clear_block(p, static_cast<int>(blockIdx.x) - chunks, threadIdx.x, 32 * kRankWarps);
    return;
  }
  const int4 ch = p.plan.chunk[blockIdx.x];
  const int rows = ch.y & 0xFF;
  if (rows == 0) return;
  const int req = ch.y >> 8, adapter = ch.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int r0 = blockIdx.y * 16;
  const uint16_t* fa = p.f + (static_cast<size_t>(adapter) * p.rp + r0 + g) * p.fp;
  const uint16_t* fb = fa + static_cast<size_t>(8) * p.fp;
  const uint16_t* xr = p.x + static_cast<int64_t>(ch.x + min(g, rows - 1)) * p.ldx;
  float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int groups = (p.k + 63) / 64;
  for (int i0 = warp; i0 < groups; i0 += kRankWarps * kRankBatch) {
    uint32_t wa[kRankBatch][8], wb[kRankBatch][8], wx[kRankBatch][8];
#pragma unroll
    for (int b = 0; b < kRankBatch; ++b) {
      const int i = i0 + b * kRankWarps, c = 64 * i + 16 * j;
      load16(fa, c, p.k, i < groups, wa[b]);
      load16(fb, c, p.k, i < groups, wb[b]);
      load16(xr, c, p.k, i < groups && g < rows, wx[b]);
    }
#pragma unroll
    for (int b = 0; b < kRankBatch; ++b)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        mma_16x8x16(d, wa[b][2 * s], wb[b][2 * s], wa[b][2 * s + 1], wb[b][2 * s + 1], wx[b][2 * s], wx[b][2 * s + 1]);
  }
  part[warp][g][2 * j] = d[0];
  part[warp][g][2 * j + 1] = d[1];
  part[warp][g + 8][2 * j] = d[2];
  part[warp][g + 8][2 * j + 1] = d[3];
  __syncthreads();
  const int r = threadIdx.x & 15, row = threadIdx.x >> 4;
  if (row >= rows) return;
  float sum = part[0][r][row];
#pragma unroll
  for (int w = 1; w < kRankWarps; ++w) sum += part[w][r][row];
  sum *= __int_as_float(ch.w);
  const AdapterInfo info = p.info[adapter];
  // a factor that is not finite is stored as zeros; its request's rows are NaN
  if (info.bad != 0) sum = __int_as_float(0x7FC00000);
  if (r0 + r >= info.rank) sum = 0.0f;
  const int t = ch.x + row;
  if (p.v32 != nullptr) p.v32[static_cast<int64_t>(t) * p.ld32 + r0 + r] = sum;
  if (p.vblk != nullptr) {
    const int tile = t >> (6 + p.lvl);
    const int64_t at = (static_cast<int64_t>(tile + req) << (6 + p.lvl)) + (t & ((64 << p.lvl) - 1));
    p.vblk[at * p.ldb + r0 + r] = __bfloat16_as_ushort(__float2bfloat16_rn(sum));
  }
}

// ---- the whole projection, few rows ------------------------------------------------

// The 16 weights of one row that a lane holds of a 64-wide K group, as loaded.
template <int BITS>
struct FewCodes {
  static constexpr int kWords = BITS == 0 ? 8 : BITS == 8 ? 4 : 2;
  uint32_t w[kWords];
};

// Bytes of a 64-wide group of a row, and of a lane's share of it.
template <int BITS>
constexpr int kGroupBytes = BITS == 0 ? 128 : 8 * BITS;

template <int BITS>
__device__ __forceinline__ void few_load(const uint8_t* at, int col, int k, FewCodes<BITS>& c) {
  if constexpr (BITS == 0) {  // `at`: the lane's column `col`; zeros from column k on
    load16(reinterpret_cast<const uint16_t*>(at) - col, col, k, true, c.w);
  } else if constexpr (BITS == 8) {
    const uint4 v = ld_global_nc_v4(at);
    c.w[0] = v.x, c.w[1] = v.y, c.w[2] = v.z, c.w[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
    c.w[0] = v.x, c.w[1] = v.y;
  }
}

// The lane's 16 weights as eight bf16 pairs, in MMA order: pairs 2 s and 2 s + 1
// are K step s. Packed codes come out as whole numbers, exact in bf16: w8 as q
// (0 .. 255) in order; w4 as 128 + q, the code put into the low mantissa bits of
// 128, two at a time where they lie 16 bits apart: pair i of a word is (i, i + 4).
template <int BITS>
__device__ __forceinline__ void few_pairs(const FewCodes<BITS>& c, uint32_t code_xor, uint32_t (&p)[8]) {
  if constexpr (BITS == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = c.w[i];
  } else if constexpr (BITS == 8) {
    const uint64_t less = f32x2(-32768.0f, -32768.0f);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t w = c.w[s] ^ code_xor;
      auto code = [&](uint32_t sel) { return __uint_as_float(__byte_perm(w, 0x4700u, sel)); };  // 32768 + q
      p[2 * s] = f32x2_to_bf16x2(add_f32x2(f32x2(code(0x5404u), code(0x5414u)), less));
      p[2 * s + 1] = f32x2_to_bf16x2(add_f32x2(f32x2(code(0x5424u), code(0x5434u)), less));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (c.w[i >> 2] >> (4 * (i & 3)) & 0x000F000Fu) | 0x43004300u;
  }
}

// The lane's 16 values of x in the same order.
template <int BITS>
__device__ __forceinline__ void few_x(const uint16_t* at, int col, int k, uint32_t (&x)[8]) {
  if constexpr (BITS == 0) {
    load16(at - col, col, k, true, x);
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(at)), b = __ldg(reinterpret_cast<const uint4*>(at) + 1);
    if constexpr (BITS == 8) {
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
      x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      x[0] = __byte_perm(a.x, a.z, 0x5410), x[1] = __byte_perm(a.x, a.z, 0x7632);
      x[2] = __byte_perm(a.y, a.w, 0x5410), x[3] = __byte_perm(a.y, a.w, 0x7632);
      x[4] = __byte_perm(b.x, b.z, 0x5410), x[5] = __byte_perm(b.x, b.z, 0x7632);
      x[6] = __byte_perm(b.y, b.w, 0x5410), x[7] = __byte_perm(b.y, b.w, 0x7632);
    }
  }
}

// W x of one feature and row of a packed weight, weight by weight, for a sum that
// the codes' arithmetic does not hold: scale sum_k q x and offset sum_k x are of
// opposite signs and up to 255 times x, so an infinity in x came out as inf - inf,
// and x beyond 1e36 overflowed where W x does not. Rare, and never inlined: the
// kernel's loop keeps its registers. Ends at a NaN, which stays one. A thread does
// a whole sum: a call of one such row takes 60 us (w4 10240x3840), of 16 such rows
// 247. A warp a row took 33 and 206, but a barrier or a larger function behind the
// loop cost every call of up to 8 rows 1.1 us of 11.
template <int BITS>
__device__ __noinline__ float few_dot(const FewParams& p, int n, int t) {
  const uint8_t* w = p.w + static_cast<size_t>(n) * p.w_pitch;
  const uint32_t* sb = p.sb + static_cast<size_t>(n) * p.sb_stride;
  const uint16_t* x = p.x + static_cast<int64_t>(t) * p.ldx;
  float sum = 0.0f;
#pragma unroll 1
  for (int c = 0; c < p.k && sum == sum; c += 64) {  // k is a multiple of 64
    const uint32_t z = sb[c / 64];
    const float scale = bf16_bits_to_f32(z & 0xFFFFu), bias = bf16_bits_to_f32(z >> 16);
#pragma unroll 4
    for (int h = 0; h < 64; h += 8) {
      const uint4 xv = *reinterpret_cast<const uint4*>(x + c + h);
      const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
      uint32_t q[2];
      if constexpr (BITS == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(w + c + h);
        q[0] = v.x ^ p.code_xor, q[1] = v.y ^ p.code_xor;
      } else {
        q[0] = *reinterpret_cast<const uint32_t*>(w + (c + h) / 2);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float code = BITS == 8 ? static_cast<float>(q[i / 4] >> (8 * (i % 4)) & 0xFFu) - p.zero
                                     : static_cast<float>(q[0] >> (4 * i) & 0xFu);
        sum = fmaf(fmaf(code, scale, bias), __uint_as_float(i % 2 == 0 ? xw[i / 2] << 16 : xw[i / 2] & 0xFFFF0000u), sum);
      }
    }
  }
  return sum;
}

// Blocks an SM that the registers are cut to. With 17 to 32 rows and bf16 two
// blocks of 8 warps, not one, take 3840x3840 from 23.0 to 16.8 us; the codes of
// packed weights do not fit beside four tiles of x then.
template <int BITS, int NT, int WARPS>
constexpr int kFewBlocks = NT > 2 ? (WARPS == 4 ? 3 : BITS == 0 ? 2 : 1)
                                  : (WARPS == 4 ? 5 : NT == 1 && BITS == 4 ? 3 : 2);

// y[t] = W x[t] + B_a v[t] for up to 8 NT rows: bound by reading W once. A
// block takes 16 features, its WARPS warps the 64-wide K groups in turn, lanes as in
// rank_rows_kernel. Packed weights are not dequantized: a group's MMAs run on
// the codes, and with the sum of the group's x (one more MMA, against ones)
//   sum_k W x = scale sum_k q x + (bias - scale zero) sum_k x
// in f32, exact codes and one scale per group. The kernel starts beside
// rank_rows_kernel (it reads x and W, which are complete when that one runs) and
// waits for it before the adapters' part. Rows past m repeat the last one: the
// MMA's columns are independent, theirs are not stored.
// Measured, a call in a row of calls (weight in L2 in part): 1 row of w8 3840x3840
// 10.6 us, of bf16 10240x3840 18.6 us (4.2 TB/s of weight); 16 rows of w4 10240x3840
// with 16 adapters of 32 ranks 22 us (29 MB; a third of the issue slots: codes to
// bf16 and the wait for each group's loads).
template <int BITS, int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, kFewBlocks<BITS, NT, WARPS>)
    few_rows_kernel(const __grid_constant__ FewParams p) {
  // K groups a warp loads at a time, one batch ahead: 128 bytes a lane in flight;
  // up to 8 rows of w4 half of that from 24 warps an SM, not 16 (10240x3840, one
  // row: 13.8 -> 11.1 us; at 16 rows and w8 the registers do not stretch so far)
  constexpr int kBatch = BITS == 4 ? (NT == 1 ? 2 : 4) : BITS == 8 ? 2 : 1;
  __shared__ float part[WARPS][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int f0 = blockIdx.x * 16;
  // The lane's place in the warp's first group, stepped from batch to batch: the
  // groups of a batch are constant offsets from it.
  constexpr int kGroup = kGroupBytes<BITS>, kStep = WARPS * kBatch;
  const uint8_t* wp[2];
  const uint32_t* sp[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = min(f0 + 8 * h + g, p.n - 1);  // rows past n repeat the last
    wp[h] = p.w + static_cast<size_t>(n) * p.w_pitch + warp * kGroup + j * (kGroup / 4);
    sp[h] = p.sb + static_cast<size_t>(n) * p.sb_stride + warp;
  }
  const uint16_t* xp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) xp[t] = p.x + static_cast<int64_t>(min(8 * t + g, p.m - 1)) * p.ldx + 64 * warp + 16 * j;
  const int groups = (p.k + 63) / 64;

  FewCodes<BITS> codes[2][kBatch][2];
  uint32_t sb[2][kBatch][2];
  auto load = [&](int i0, int buf) {  // and steps on
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (i0 + b * WARPS < groups) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          few_load<BITS>(wp[h] + b * WARPS * kGroup, 64 * (i0 + b * WARPS) + 16 * j, p.k, codes[buf][b][h]);
          if constexpr (BITS != 0) sb[buf][b][h] = __ldg(sp[h] + b * WARPS);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      wp[h] += kStep * kGroup;
      sp[h] += kStep;
    }
  };
  load(warp, 0);
  float y[NT][4];
#pragma unroll
  for (int e = 0; e < 4 * NT; ++e) y[e / 4][e % 4] = 0.0f;
  const uint32_t ones = 0x3F803F80u;
  // whole pairs of batches, so that the buffers' indices are constants
  for (int i0 = warp; i0 < groups; i0 += 2 * kStep) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int ih = i0 + half * kStep;
      if (ih >= groups) break;
      load(ih + kStep, half ^ 1);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int i = ih + b * WARPS;
        if (i >= groups) break;
        uint32_t x[NT][8];
#pragma unroll
        for (int t = 0; t < NT; ++t) few_x<BITS>(xp[t] + b * WARPS * 64, 64 * i + 16 * j, p.k, x[t]);
        uint32_t lo[8], hi[8];
        few_pairs<BITS>(codes[half][b][0], p.code_xor, lo);
        few_pairs<BITS>(codes[half][b][1], p.code_xor, hi);
        if constexpr (BITS == 0) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int s = 0; s < 4; ++s)
              mma_16x8x16(y[t], lo[2 * s], hi[2 * s], lo[2 * s + 1], hi[2 * s + 1], x[t][2 * s], x[t][2 * s + 1]);
        } else {
          // scale, and bias less scale * zero, of rows g and g + 8
          const uint32_t z0 = sb[half][b][0], z1 = sb[half][b][1];
          const float s0 = bf16_bits_to_f32(z0 & 0xFFFFu), s1 = bf16_bits_to_f32(z1 & 0xFFFFu);
          const float o0 = fmaf(-p.zero, s0, bf16_bits_to_f32(z0 >> 16));
          const float o1 = fmaf(-p.zero, s1, bf16_bits_to_f32(z1 >> 16));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float d[4], e[4];  // e: the sums of x, the same in every row
            mma_16x8x16_first(e, ones, ones, ones, ones, x[t][0], x[t][1]);
            mma_16x8x16_first(d, lo[0], hi[0], lo[1], hi[1], x[t][0], x[t][1]);
#pragma unroll
            for (int s = 1; s < 4; ++s) {
              mma_16x8x16(e, ones, ones, ones, ones, x[t][2 * s], x[t][2 * s + 1]);
              mma_16x8x16(d, lo[2 * s], hi[2 * s], lo[2 * s + 1], hi[2 * s + 1], x[t][2 * s], x[t][2 * s + 1]);
            }
            y[t][0] = fmaf(s0, d[0], fmaf(o0, e[0], y[t][0]));
            y[t][1] = fmaf(s0, d[1], fmaf(o0, e[1], y[t][1]));
            y[t][2] = fmaf(s1, d[2], fmaf(o1, e[0], y[t][2]));
            y[t][3] = fmaf(s1, d[3], fmaf(o1, e[1], y[t][3]));
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) xp[t] += kStep * 64;
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) part[warp][g + 8 * (q >> 1)][8 * t + 2 * j + (q & 1)] = y[t][q];
  __syncthreads();
  pdl_wait();  // v is complete; y may be written
  pdl_release();
  const int f = threadIdx.x & 15;
  if (f0 + f >= p.n) return;
  for (int t = threadIdx.x >> 4; t < p.m; t += 2 * WARPS) {
    float sum = part[0][f][t];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) sum += part[w][f][t];
    if constexpr (BITS != 0) {
      if (!isfinite(sum)) sum = few_dot<BITS>(p, f0 + f, t);
    }
    const int a = p.row_adapter[t];
    if (a >= 0) {
      const uint16_t* br = p.b + (static_cast<size_t>(a) * p.n + f0 + f) * p.rp;
      const float* v = p.v + static_cast<int64_t>(t) * p.ldv;
      float low = 0.0f;
      for (int r = 0; r < p.rp; r += 8) {
        const uint4 bw = *reinterpret_cast<const uint4*>(br + r);
        const float4 v0 = *reinterpret_cast<const float4*>(v + r), v1 = *reinterpret_cast<const float4*>(v + r + 4);
        low = fmaf(__uint_as_float(bw.x << 16), v0.x, low);
        low = fmaf(__uint_as_float(bw.x & 0xFFFF0000u), v0.y, low);
        low = fmaf(__uint_as_float(bw.y << 16), v0.z, low);
        low = fmaf(__uint_as_float(bw.y & 0xFFFF0000u), v0.w, low);
        low = fmaf(__uint_as_float(bw.z << 16), v1.x, low);
        low = fmaf(__uint_as_float(bw.z & 0xFFFF0000u), v1.y, low);
        low = fmaf(__uint_as_float(bw.w << 16), v1.z, low);
        low = fmaf(__uint_as_float(bw.w & 0xFFFF0000u), v1.w, low);
      }
      sum += low;
    }
    p.y[static_cast<int64_t>(t) * p.ldy + f0 + f] = __bfloat16_as_ushort(__float2bfloat16_rn(sum));
  }
}

// ---- dense transpose of a projection weight -------------------------------------

// dst[k][n] (pitch np) = bf16 weight [n][k]: the values the projection kernel
// multiplies with (packed codes dequantized with its arithmetic and rounding).
__global__ void __launch_bounds__(256) weight_transpose_kernel(const uint8_t* w, const uint32_t* sb, int sb_stride,
                                                               int n, int k, int kp, int bits, uint32_t code_xor,
                                                               float code_offset, uint16_t* dst, int np) {
  __shared__ uint16_t sm[32][33];
  const int c = threadIdx.x & 31, n0 = blockIdx.y * 32, k0 = blockIdx.x * 32;
  for (int r = threadIdx.x >> 5; r < 32; r += 8) {
    uint16_t v = 0;
    if (n0 + r < n && k0 + c < k) {
      const size_t row = n0 + r;
      const int col = k0 + c;
      if (bits == 0) {
        v = reinterpret_cast<const uint16_t*>(w)[row * kp + col];
      } else {
        const uint32_t word = sb[row * sb_stride + (col >> 6)];
        const float sc = bf16_bits_to_f32(word & 0xFFFFu), bi = bf16_bits_to_f32(word >> 16);
        const float bf = fmaf(-sc, code_offset, bi);
        uint32_t q;
        if (bits == 8)
          q = w[row * k + col] ^ (code_xor & 0xFFu);
        else
          q = (w[row * (k / 2) + (col >> 1)] >> (4 * (col & 1))) & 0xFu;
        v = __bfloat16_as_ushort(__float2bfloat16_rn(fmaf(32768.0f + static_cast<float>(q), sc, bf)));
      }
    }
    sm[r][c] = v;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < 32; r += 8)
    if (k0 + r < k && n0 + c < np) dst[static_cast<size_t>(k0 + r) * np + n0 + c] = sm[c][r];
}

// A launch that may begin its set-up while the one before it on the stream ends.
template <class P>
cudaError_t launch_overlapped(void (*kernel)(P), dim3 grid, dim3 block, const P& p, cudaStream_t stream,
                              bool overlap = true) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = overlap ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_plan_requests(const PlanParams& p, cudaStream_t stream) {
  return launch_overlapped(plan_requests_kernel, dim3(1), dim3(kPlanThreads), p, stream);
}

cudaError_t launch_bank_set(const BankSetParams& p, cudaStream_t stream) {
  const int rt = (p.rp + 31) / 32, kt = (p.kp + 31) / 32, nt = (p.n + 31) / 32;
  bank_set_kernel<<<rt * (kt + nt), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_rank_rows(const RankParams& p, cudaStream_t stream) {
  const bool clear = p.vblk != nullptr || p.clear_v32;
  const int blocks = clear ? plan_blocks(p.plan.m, p.plan.n_req, p.lvl) : 0;
  const dim3 grid(plan_chunks(p.plan.m, p.plan.n_req) + blocks, p.rp / 16);
  if (grid.x == 0) return cudaSuccess;  // no request
  return launch_overlapped(rank_rows_kernel, grid, dim3(32 * kRankWarps), p, stream);
}

namespace {

template <int BITS, int NT>
cudaError_t launch_few(const FewParams& p, cudaStream_t stream) {
  const dim3 grid((p.n + 15) / 16);
  // it may start beside rank_rows_kernel, never beside what comes before that
  const bool over = p.chunks > 0;
  // Blocks of 8 warps, or of 4 with more of them on an SM where that takes the
  // features in fewer rounds: a second round of a few blocks costs as much as the
  // first. 8 / 4 warps at 10240x3840: 1 row w4 11.2 / 10.9 us, w8 17.9 / 13.9, bf16
  // 19.9 / 18.5; 16 rows w4 21.9 / 23.2, w8 23.6 / 28.0 (the registers of five
  // blocks do not hold the codes beside two tiles of x), bf16 30.7 / 24.0; 32 rows w4
  // 39.7 / 33.9, w8 42.6 / 32.7, bf16 39.1 / 41.2. Up to 16 rows five blocks of 4
  // an SM have to take all (1 row, w4 12288x3840: 13.5 / 15.8), and below three
  // they leave SMs short of loads (5120x3840: 1 row bf16 11.5 / 15.5; but 32 rows w4
  // 23.0 / 17.7).
  constexpr bool kPays = NT == 4 ? BITS != 0 : NT == 1 || BITS == 0;
  if constexpr (kPays) {
    if (p.n > 16 * 148 * (NT == 4 ? 2 : 3) && (NT == 4 || p.n <= 16 * 148 * 5))
      return launch_overlapped(few_rows_kernel<BITS, NT, 4>, grid, dim3(128), p, stream, over);
  }
  return launch_overlapped(few_rows_kernel<BITS, NT, 8>, grid, dim3(256), p, stream, over);
}

template <int BITS>
cudaError_t launch_few(const FewParams& p, cudaStream_t stream) {
  if (p.m <= 8) return launch_few<BITS, 1>(p, stream);
  if (p.m <= 16) return launch_few<BITS, 2>(p, stream);
  if (p.m <= kFewRows) return launch_few<BITS, 4>(p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_few_rows(const FewParams& p, int bits, cudaStream_t stream) {
  switch (bits) {
    case 0: return launch_few<0>(p, stream);
    case 8: return launch_few<8>(p, stream);
    case 4: return launch_few<4>(p, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_weight_transpose(const void* w, const uint32_t* sb, int sb_stride, int n, int k, int kp, int bits,
                                    uint32_t code_xor, float code_offset, uint16_t* dst, int np,
                                    cudaStream_t stream) {
  const dim3 grid((k + 31) / 32, (np + 31) / 32);
  weight_transpose_kernel<<<grid, 256, 0, stream>>>(static_cast<const uint8_t*>(w), sb, sb_stride, n, k, kp, bits,
                                                    code_xor, code_offset, dst, np);
  return cudaGetLastError();
}

}  // namespace mp
