// dyn_lds.h -- how much dynamic LDS a kernel may be launched with, kept per device.
// Host code alone: the runtime holds the limit of a kernel for the current device.
#pragma once

#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstddef>
#include <mutex>

namespace ojx {

// What a kernel's limit was raised to, by device.  Static, one for each kernel.
struct DynLds {
    static constexpr int kDevices = 64;              // past them the limit is set at every call
    std::atomic<size_t> granted[kDevices];
};

// The current device's limit of kernel fn, at least `bytes` from here on.
inline hipError_t raise_dyn_lds(const void *fn, size_t bytes, DynLds *lds) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const bool kept = dev >= 0 && dev < DynLds::kDevices;
    if (kept && bytes <= lds->granted[dev].load(std::memory_order_acquire)) return hipSuccess;
    static std::mutex one;                           // a smaller limit must not follow a larger one
    std::lock_guard<std::mutex> hold(one);
    if (kept && bytes <= lds->granted[dev].load(std::memory_order_relaxed)) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == hipSuccess && kept) lds->granted[dev].store(bytes, std::memory_order_release);
    return e;
}

}  // namespace ojx
