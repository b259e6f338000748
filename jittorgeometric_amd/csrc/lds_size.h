// Kernels with more than 64 KB of dynamic LDS.
#pragma once
#include <atomic>

#include "common.h"

namespace jg {

// Allows `bytes` of dynamic LDS for a kernel, once on each device: the attribute belongs to the
// function as the current device holds it, not to the call.  Two threads at once set it twice.
template <auto Kernel> static void raise_lds(size_t bytes)
{
    static std::atomic<uint64_t> raised{0};
    int device = 0;
    (void)hipGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (raised.load(std::memory_order_acquire) & bit) return;
    (void)hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    raised.fetch_or(bit, std::memory_order_release);
}

}  // namespace jg
