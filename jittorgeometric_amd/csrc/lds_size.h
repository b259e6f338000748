// Kernels with more than 64 KB of dynamic LDS.
#pragma once
#include <mutex>

#include "common.h"

namespace jg {

// allows `bytes` of dynamic LDS for a kernel: once per kernel, whichever thread gets here first (the
// attribute belongs to the function, not to the call)
template <auto Kernel> static void raise_lds(size_t bytes)
{
    static std::once_flag raised;
    std::call_once(raised, [&] {
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    });
}

}  // namespace jg
