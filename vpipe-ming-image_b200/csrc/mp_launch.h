// Host-side helper of the kernels' launch functions.
#pragma once

#include <cuda_runtime.h>

namespace mp {

// Opts a kernel in to all the shared memory a block may have, once per device (the
// driver call costs half a microsecond of every launch otherwise). A second host
// thread that comes between does the same again.
struct SmemOptIn {
  bool done[64] = {};
  cudaError_t allow(const void* kernel) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (done[dev]) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e == cudaSuccess) done[dev] = true;
    return e;
  }
};

}  // namespace mp
