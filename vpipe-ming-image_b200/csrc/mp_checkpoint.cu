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
// kCkRows rows: four loads in flight each, one reciprocal for four rows, and the
// four scales of a group land in one 32-byte sector. The bf16 rows are read and
// written with a streaming hint, which leaves L2 to the codes: the restore that
// follows finds some there. Measured at 16896 x 10240: 84 us to keep (525 MB, 6.2
// TB/s, 79 % of the issue slots), 78 us to restore (6.7 TB/s, part of the codes from L2).
#include <cuda_runtime.h>

#include "mp_device.cuh"
#include "mp_kernels.h"

namespace mp {

namespace {

constexpr int kCkThreads = 256;
constexpr int kPerLane = 8;                         // features of a lane
constexpr int kGroupLanes = kCkGroup / kPerLane;    // 16

constexpr int kCkRows = 4;

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

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
  // max|x| on the bf16 patterns, two at a time: without the sign they order like
  // the values, infinities and NaNs last
  uint32_t top2[kCkRows];
#pragma unroll
  for (int r = 0; r < kCkRows; ++r)
    top2[r] = max_u16x2(max_u16x2(raw[r].x & 0x7FFF7FFFu, raw[r].y & 0x7FFF7FFFu),
                        max_u16x2(raw[r].z & 0x7FFF7FFFu, raw[r].w & 0x7FFF7FFFu));
  // The group's lanes share the four rows' maxima out as they reduce them: after
  // two exchanges lane (8 b3 + 4 b2 + ..) holds row 2 b3 + b2 alone, so that the
  // reciprocal and the division are done once a lane, not once a row.
  const int lane = threadIdx.x % kGroupLanes;
  const bool b3 = (lane & 8) != 0, b2 = (lane & 4) != 0;
  const uint32_t s0 = __shfl_xor_sync(0xFFFFFFFFu, b3 ? top2[0] : top2[2], 8);
  const uint32_t s1 = __shfl_xor_sync(0xFFFFFFFFu, b3 ? top2[1] : top2[3], 8);
  const uint32_t k0 = max_u16x2(b3 ? top2[2] : top2[0], s0), k1 = max_u16x2(b3 ? top2[3] : top2[1], s1);
  uint32_t mine = max_u16x2(b2 ? k1 : k0, __shfl_xor_sync(0xFFFFFFFFu, b2 ? k0 : k1, 4));
  mine = max_u16x2(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, 2));
  mine = max_u16x2(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, 1));
  const uint32_t top_bits = max(mine & 0xFFFFu, mine >> 16);
  const float top = bf16_bits_to_f32(top_bits);
  const bool finite = top_bits < 0x7F80u, live = finite && top >= kCkTiny;
  const float my_inv = live ? __fmul_rn(127.0f, __frcp_rn(top)) : 0.0f;
  const int my_row = row0 + (lane >> 2);
  if ((lane & 3) == 0 && group * kCkGroup < p.k && my_row < p.m) {
    // a group with an infinity or a NaN is NaN throughout
    p.scale[static_cast<int64_t>(group) * p.m + my_row] =
        live ? __fdiv_rn(top, 127.0f) : finite ? 0.0f : __int_as_float(0x7FC00000);
  }
#pragma unroll
  for (int r = 0; r < kCkRows; ++r) {
    const float inv = __shfl_sync(0xFFFFFFFFu, my_inv, 4 * r, kGroupLanes);
    if (c >= p.k || row0 + r >= p.m) continue;
    // x inv, then the nearest whole number (ties to even) in the low mantissa
    // bits of 1.5 2^23; |x| inv <= 127 (1 + 2^-24)^3 rounds to 127 at most. The
    // two roundings are the definition's, so never one FMA (packed f32x2 products
    // and sums were joined into one: a code in 1400 moved).
    auto code = [&](uint32_t pattern) {
      return __float_as_uint(__fadd_rn(__fmul_rn(__uint_as_float(pattern), inv), 12582912.0f));
    };
    const uint32_t v[4] = {raw[r].x, raw[r].y, raw[r].z, raw[r].w};
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t a = v[2 * h], b = v[2 * h + 1];
      const uint32_t lo = __byte_perm(code(a << 16), code(a & 0xFFFF0000u), 0x0040);
      const uint32_t hi = __byte_perm(code(b << 16), code(b & 0xFFFF0000u), 0x0040);
      w[h] = inv != 0.0f ? __byte_perm(lo, hi, 0x5410) : 0u;
    }
    int8_t* out = p.q + static_cast<int64_t>(row0 + r) * p.ldq + c;  // the pitch is a multiple of 16
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
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
