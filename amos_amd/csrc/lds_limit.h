// Workgroups that want more than 64 KB of dynamic LDS: the kernel is told so once on every device it runs on.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>

#include "mapper.h"

namespace amos {

constexpr int kLdsMaxDevices = 64;

// `done`: a static of the caller's, one bit a device.  `no_scratch`: kernels that count their own outstanding copies
// must not have been built with register spills, whose traffic would be counted among them.
inline int allow_lds(const void* fn, int bytes, bool no_scratch, const char* what, std::atomic<uint64_t>& done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess && dev < kLdsMaxDevices && (done.load(std::memory_order_relaxed) >> dev & 1)) return 0;
  if (e == hipSuccess) e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess && no_scratch) {
    hipFuncAttributes fa;
    e = hipFuncGetAttributes(&fa, fn);
    if (e == hipSuccess && fa.localSizeBytes)
      return set_error(AMOS_ERR_INFEASIBLE, "%s was built with %d bytes of scratch memory per lane", what, (int)fa.localSizeBytes);
  }
  if (e != hipSuccess) return set_error(AMOS_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  if (dev < kLdsMaxDevices) done.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  return 0;
}

}  // namespace amos
