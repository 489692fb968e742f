// Host-side helpers of the stand-alone ops that live in their own translation units.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/dfssm.h"

int dfssm_fail(int code, const char* fmt, ...);  // sets the thread's last-error message (dfssm_capi.cu)

#define DFSSM_CU(call)                                                                                    \
  do {                                                                                                    \
    const cudaError_t _e = (call);                                                                        \
    if (_e != cudaSuccess)                                                                                \
      return dfssm_fail(DFSSM_ERR_CUDA, "%s failed: %s (%d) at %s:%d", #call, cudaGetErrorString(_e), (int)_e, \
                        __FILE__, __LINE__);                                                              \
  } while (0)

namespace dfssm {

// Dynamic shared memory limit of one kernel, raised once per device (the runtime call costs
// microseconds, which a one-token op would otherwise pay at every launch).  One object per kernel
// instance, `static` where the kernel is launched; two threads may both make the call, which is harmless.
struct SmemLimit {
  static constexpr int kDevices = 64;
  std::atomic<int> have[kDevices];
  SmemLimit() {
    for (auto& h : have) h.store(0, std::memory_order_relaxed);
  }
  cudaError_t raise(const void* fn, int bytes) {
    int dev = 0;
    cudaError_t ce = cudaGetDevice(&dev);
    if (ce != cudaSuccess) return ce;
    const bool known = dev < kDevices;
    if (known && have[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    ce = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (ce == cudaSuccess && known) have[dev].store(bytes, std::memory_order_relaxed);
    return ce;
  }
};

}  // namespace dfssm
