// Gradients of the factors of many adapters: matrix products grouped by
// adapter, over the ragged row ranges of its requests,
//
//   out[a] = sum over the rows t of adapter a of u[t] (outer) x[t],
//
// dA from x and u = s dy B, dB from dy and v = s x A^T. Sums in f32.
#include <cuda_runtime.h>

#include "mp_device.cuh"
#include "mp_kernels.h"

namespace mp {

namespace {

constexpr int kTileF = 64;   // features of a block
constexpr int kRows = 32;    // rows staged at a time
constexpr int kGradThreads = 256;

// One block: 64 features of one adapter, all ranks; rows are staged through
// shared memory in f32 and every thread owns one feature and every fourth rank.
__global__ void __launch_bounds__(kGradThreads) adapter_grad_kernel(const __grid_constant__ GradParams p) {
  __shared__ float sx[kRows][kTileF];
  __shared__ float su[kRows][kMaxAdapterRank];
  int i = blockIdx.x;
  int mi = 0;
  if (p.n_mem > 1) {
    const int first = (p.mem[0].width + kTileF - 1) / kTileF;
    if (i >= first) {
      mi = 1;
      i -= first;
    }
  }
  const GradMember& mb = p.mem[mi];
  const int a = blockIdx.y, f0 = i * kTileF;
  const int f = threadIdx.x % kTileF, rg = threadIdx.x / kTileF;  // 4 rank groups
  float acc[kMaxAdapterRank / 4];
#pragma unroll
  for (int r = 0; r < kMaxAdapterRank / 4; ++r) acc[r] = 0.0f;
  for (int s = p.plan.begin[a]; s < p.plan.begin[a + 1]; ++s) {
    const int2 seg = p.plan.seg[s];
    for (int t0 = seg.x; t0 < seg.y; t0 += kRows) {
      const int rows = min(kRows, seg.y - t0);
      __syncthreads();
      for (int e = threadIdx.x; e < kRows * kTileF; e += kGradThreads) {
        const int t = e / kTileF, c = f0 + e % kTileF;
        float v = 0.0f;
        if (t < rows && c < mb.width) {
          const int64_t row = t0 + t;
          v = mb.x != nullptr ? bf16_bits_to_f32(mb.x[row * mb.ldx + c])
                              : mb.q[row * mb.ldq + c] * mb.scale[static_cast<int64_t>(c / kCkGroup) * p.plan.m + row];
        }
        sx[t][e % kTileF] = v;
      }
      for (int e = threadIdx.x; e < kRows * p.r; e += kGradThreads) {
        const int t = e / p.r, c = e % p.r;
        su[t][c] = t < rows ? mb.u[static_cast<int64_t>(t0 + t) * mb.ldu + c] : 0.0f;
      }
      __syncthreads();
      for (int t = 0; t < rows; ++t) {
        const float x = sx[t][f];
#pragma unroll
        for (int r = 0; r < kMaxAdapterRank / 4; ++r)
          if (rg + 4 * r < p.r) acc[r] = fmaf(su[t][rg + 4 * r], x, acc[r]);
      }
    }
  }
  if (f0 + f >= mb.width) return;
  float* out = mb.out + static_cast<int64_t>(a) * p.r * mb.width;
#pragma unroll
  for (int r = 0; r < kMaxAdapterRank / 4; ++r) {
    const int rank = rg + 4 * r;
    if (rank >= p.r) break;
    out[mb.rank_major ? static_cast<int64_t>(rank) * mb.width + f0 + f
                      : static_cast<int64_t>(f0 + f) * p.r + rank] = acc[r];
  }
}

}  // namespace

cudaError_t launch_adapter_grad(const GradParams& p, cudaStream_t stream) {
  int tiles = 0;
  for (int i = 0; i < p.n_mem; ++i) tiles += (p.mem[i].width + kTileF - 1) / kTileF;
  adapter_grad_kernel<<<dim3(tiles, p.plan.cap), kGradThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace mp
