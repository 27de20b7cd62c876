// ggq_launch.hpp -- launch helpers of the row, integer-product and expert kernels (not part of the C ABI).
#pragma once

#include "ggq_host.hpp"

#include <atomic>
#include <cstdint>

namespace ggq {

// HIP takes fewer than 2^32 threads in one dimension of a launch.
inline bool launchable(uint64_t blocks, uint32_t threads) { return blocks < (1ull << 32) / threads; }

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
