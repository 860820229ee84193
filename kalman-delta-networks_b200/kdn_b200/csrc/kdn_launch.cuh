// Shared memory beyond a launch's default, asked for once per kernel and device.
#pragma once

#include <atomic>

#include "kdn_common.cuh"

namespace kdn {

// Lets Kernel take up to `most` bytes of dynamic shared memory on the current
// device.  `most` has to be the same in every call for a kernel.
template <auto Kernel>
int allow_smem(size_t most, const char* what) {
  static std::atomic<uint64_t> done{0};  // a bit per device
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (err == cudaSuccess && (done.load(std::memory_order_relaxed) & bit)) return KDN_OK;
  if (err == cudaSuccess) err = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return set_error(KDN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return KDN_OK;
}

}  // namespace kdn
