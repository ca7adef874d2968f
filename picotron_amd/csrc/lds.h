// Dynamic LDS beyond 64 KB for the kernels that use it.
#pragma once
#include <atomic>

#include "common.h"

// lets a kernel have `bytes` of dynamic LDS; asked once per device
template <auto KERNEL>
static inline hipError_t allow_lds(int bytes) {
    static std::atomic<uint64_t> allowed{0};
    int device = 0;
    const hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (allowed.load(std::memory_order_relaxed) & bit) return hipSuccess;
    const hipError_t set = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (set == hipSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
    return set;
}
