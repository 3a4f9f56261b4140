// A kernel's dynamic shared memory above 48 KB, and with `carveout` all that an SM can give for it: asked for once a device, of which a process may use several.
#pragma once
#include <cuda_runtime.h>

static inline int smem_limit(const void* kernel, int bytes, bool carveout, bool (&ready)[64]) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess || (device >= 0 && device < 64 && ready[device])) return (int)e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && carveout) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  if (e == cudaSuccess && device >= 0 && device < 64) ready[device] = true;
  return (int)e;
}
