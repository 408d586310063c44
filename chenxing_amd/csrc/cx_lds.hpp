// cx_lds.hpp -- the dynamic-LDS limits of kernels that take more than the default.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>
#include <mutex>

namespace cx {

// A kernel's limit is kept by device and only ever raised.  raise() sets it on the
// current device and returns 0, or the HIP error; a failure is not remembered, so the
// next call tries again.
class LdsLimit {
 public:
  int raise(const void* kernel, int bytes) {
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return (int)e;
    if (dev < DEVICES && set_[dev].load(std::memory_order_acquire) >= bytes) return 0;
    std::lock_guard<std::mutex> g(mu_);        // a later, smaller call must not lower it
    if (dev < DEVICES && set_[dev].load(std::memory_order_relaxed) >= bytes) return 0;
    if (hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        e != hipSuccess)
      return (int)e;
    if (dev < DEVICES) set_[dev].store(bytes, std::memory_order_release);
    return 0;
  }

 private:
  static constexpr int DEVICES = 64;
  std::mutex mu_;
  std::atomic<int> set_[DEVICES] = {};
};

}  // namespace cx
