// Host-side launch helpers.
#pragma once
#include <cuda_runtime.h>

namespace carekv {

// SMs of the current device (148 where it cannot be asked).
inline int sm_count() {
  static thread_local int count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (count[dev] == 0 && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return count[dev];
}

// Lets `kernel` use BYTES of dynamic shared memory on the current device;
// asked of the runtime once per host thread, kernel and device (0.5 us).
template <int BYTES, typename K>
cudaError_t allow_smem(K* kernel) {
  static thread_local const void* known[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const void* id = reinterpret_cast<const void*>(kernel);
  if (dev >= 0 && dev < 64 && known[dev] == id) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  if (e == cudaSuccess && dev >= 0 && dev < 64) known[dev] = id;
  return e;
}

}  // namespace carekv
