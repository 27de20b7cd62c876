// ggq_launch.hpp -- launch helpers of the row, integer-product and expert kernels (not part of the C ABI).
#pragma once

#include "ggq_host.hpp"

#include <atomic>
#include <cstdint>

namespace ggq {

// Lets kernel `fn` take `bytes` of dynamic LDS on the current device; `raised` (one per kernel) remembers the devices it was done on.
inline hipError_t allow_lds(const void* fn, int bytes, std::atomic<uint64_t>& raised)
{
    int dev = 0;
    const hipError_t got = hipGetDevice(&dev);
    if (got != hipSuccess) return got;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (raised.load(std::memory_order_relaxed) & bit) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) raised.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

}  // namespace ggq
