// Workgroups with more than 64 KB of LDS.
#pragma once

#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstdint>

namespace rr::kern {

// Lets a kernel have `bytes` of dynamic LDS on the current device: asked for once a device (a
// second thread's call in between asks for the same again), which `allowed` notes.
inline hipError_t allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>* allowed) {
  int device = 0;
  hipError_t error = hipGetDevice(&device);
  if (error != hipSuccess) return error;
  const uint64_t bit = device < 64 ? uint64_t{1} << device : 0;
  if ((allowed->load(std::memory_order_relaxed) & bit) != 0) return hipSuccess;
  error = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (error == hipSuccess) allowed->fetch_or(bit, std::memory_order_relaxed);
  return error;
}

}  // namespace rr::kern
