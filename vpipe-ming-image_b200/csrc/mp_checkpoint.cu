// Activation checkpoints in 8 bits: the bf16 rows a backward pass needs, kept
// as one signed byte a value and one f32 scale for every 128 features of a row,
//
//   scale = max|x| / 127,   q = rint(x * (127 * (1 / max|x|))),   x' = q * scale,
//
// every operation rounded to f32.
//
// Both kernels are one pass, bound by memory: 3 bytes a value. Each of 16
// lanes holds 8 consecutive features of a group (one 16-byte load), the group's
// maximum goes round them by shuffles. A thread takes the same features of
// kCkRows rows: four loads in flight each, and the four scales of a group land
// in one 32-byte sector. The bf16 rows are read and written with a streaming
// hint, which leaves L2 to the codes: the restore that follows finds some there.
#include <cuda_runtime.h>

#include "mp_device.cuh"
#include "mp_kernels.h"

namespace mp {

namespace {

constexpr int kCkThreads = 256;
constexpr int kPerLane = 8;                         // features of a lane
constexpr int kGroupLanes = kCkGroup / kPerLane;    // 16

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

constexpr int kCkRows = 4;

// Block (x, y): rows [4 x, 4 x + 4), groups [16 y, 16 y + 16), one per half-warp.
__global__ void __launch_bounds__(kCkThreads) checkpoint_kernel(const __grid_constant__ CheckpointParams p) {
  const int row0 = blockIdx.x * kCkRows;
  const int group = blockIdx.y * (kCkThreads / kGroupLanes) + threadIdx.x / kGroupLanes;
  const int c = group * kCkGroup + (threadIdx.x % kGroupLanes) * kPerLane;
  pdl_wait();
  pdl_release();
  uint4 raw[kCkRows];
#pragma unroll
  for (int r = 0; r < kCkRows; ++r) {
    raw[r] = make_uint4(0, 0, 0, 0);
    const uint16_t* x = p.x + static_cast<int64_t>(row0 + r) * p.ldx + c;
    if (row0 + r >= p.m) continue;
    if (c + kPerLane <= p.k) {
      raw[r] = __ldcs(reinterpret_cast<const uint4*>(x));
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (c + i < p.k) w[i >> 1] |= static_cast<uint32_t>(x[i]) << (16 * (i & 1));
      raw[r] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
#pragma unroll
  for (int r = 0; r < kCkRows; ++r) {
    float f[8];
    unpack8(raw[r], f);
    float top = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      top = fmaxf(top, fabsf(f[i]));
      finite = finite && fabsf(f[i]) <= 3.3895314e38f;  // false for NaN
    }
    if (!finite) top = __int_as_float(0x7F800000);  // fmaxf drops a NaN
#pragma unroll
    for (int d = 1; d < kGroupLanes; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    finite = top <= 3.3895314e38f;
    if (c >= p.k || row0 + r >= p.m) continue;
    const bool live = finite && top >= kCkTiny;
    const float inv = live ? __fmul_rn(127.0f, __frcp_rn(top)) : 0.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      // |x| inv <= 127 (1 + 2^-24)^3: rounds to 127 at most
      const int q = live ? __float2int_rn(__fmul_rn(f[i], inv)) : 0;
      w[i >> 2] |= (static_cast<uint32_t>(q) & 0xFFu) << (8 * (i & 3));
    }
    int8_t* out = p.q + static_cast<int64_t>(row0 + r) * p.ldq + c;  // the pitch is a multiple of 16
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    if (threadIdx.x % kGroupLanes == 0) {
      // a group with an infinity or a NaN is NaN throughout
      const float s = finite ? (live ? __fdiv_rn(top, 127.0f) : 0.0f) : __int_as_float(0x7FC00000);
      p.scale[static_cast<int64_t>(group) * p.m + row0 + r] = s;
    }
  }
}

__global__ void __launch_bounds__(kCkThreads) restore_kernel(const __grid_constant__ CheckpointParams p) {
  const int row0 = blockIdx.x * kCkRows;
  const int c = (blockIdx.y * kCkThreads + threadIdx.x) * kPerLane;
  pdl_wait();
  pdl_release();
  if (c >= p.k) return;
  uint2 w[kCkRows];
  float s[kCkRows];
#pragma unroll
  for (int r = 0; r < kCkRows; ++r) {
    const int row = min(row0 + r, p.m - 1);
    w[r] = *reinterpret_cast<const uint2*>(p.q + static_cast<int64_t>(row) * p.ldq + c);
    s[r] = p.scale[static_cast<int64_t>(c / kCkGroup) * p.m + row];
  }
#pragma unroll
  for (int r = 0; r < kCkRows; ++r) {
    if (row0 + r >= p.m) return;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? w[r].x : w[r].y) >> (8 * (i & 3)))) * s[r];
    uint16_t* y = p.y + static_cast<int64_t>(row0 + r) * p.ldx + c;
    if (c + kPerLane <= p.k) {
      __stcs(reinterpret_cast<uint4*>(y), make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                     pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])));
    } else {
      for (int i = 0; c + i < p.k; ++i) y[i] = __bfloat16_as_ushort(__float2bfloat16_rn(f[i]));
    }
  }
}

cudaError_t launch(void (*kernel)(CheckpointParams), dim3 grid, const CheckpointParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kCkThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_checkpoint(const CheckpointParams& p, cudaStream_t stream) {
  const int per_block = kCkThreads * kPerLane;
  return launch(checkpoint_kernel, dim3((p.m + kCkRows - 1) / kCkRows, (p.k + per_block - 1) / per_block), p, stream);
}

cudaError_t launch_restore(const CheckpointParams& p, cudaStream_t stream) {
  const int per_block = kCkThreads * kPerLane;
  return launch(restore_kernel, dim3((p.m + kCkRows - 1) / kCkRows, (p.k + per_block - 1) / per_block), p, stream);
}

}  // namespace mp
