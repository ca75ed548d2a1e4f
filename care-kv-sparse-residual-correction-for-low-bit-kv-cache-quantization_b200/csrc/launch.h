// Host-side launch helpers.
#pragma once
#include <cuda.h>
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

// cuTensorMapEncodeTiled, found through the runtime (no link against the
// driver library); null where the driver has none.
using TensorMapEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                     const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                     CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline TensorMapEncode tensor_map_encode() {
  static const TensorMapEncode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<TensorMapEncode>(f);
  }();
  return encode;
}

}  // namespace carekv
