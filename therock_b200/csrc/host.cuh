// Host-side helpers shared by the entry points: device selection, error return, NVTX ranges.
#pragma once

#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include "../../include/fused_moe_c.h"
#include "plan.hpp"

namespace fmoe {

// Makes the device that owns `ptr` current for the lifetime of the object and puts the
// caller's device back afterwards: the entry points leave no trace in the calling thread.
class DeviceGuard {
 public:
  explicit DeviceGuard(const void* ptr) {
    cudaPointerAttributes attr;
    if (ptr == nullptr || cudaPointerGetAttributes(&attr, ptr) != cudaSuccess) {
      cudaGetLastError();   // not fatal: stay on the calling thread's device
      return;
    }
    if (attr.type != cudaMemoryTypeDevice) return;
    int cur = -1;
    if (cudaGetDevice(&cur) != cudaSuccess || cur == attr.device) return;
    if (cudaSetDevice(attr.device) != cudaSuccess) {
      rc_ = fail(FMOE_ERR_CUDA, "cudaSetDevice(%d) failed", attr.device);
      return;
    }
    prev_ = cur;
  }
  ~DeviceGuard() {
    if (prev_ >= 0) cudaSetDevice(prev_);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  int rc() const { return rc_; }

 private:
  int prev_ = -1;
  int rc_ = FMOE_OK;
};

// NVTX range around one stage of an operator (a no-op unless a profiler is attached).
struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
};

#define FMOE_CUDA(expr)                                                                    \
  do {                                                                                     \
    cudaError_t e__ = (expr);                                                              \
    if (e__ != cudaSuccess)                                                                \
      return fmoe::fail(FMOE_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e__));   \
  } while (0)

}  // namespace fmoe
