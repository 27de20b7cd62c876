// ggq_int8.hip -- C ABI over ggq_int8.hpp: the product of 8-bit integers with a scale per row of x and per row of w.
#include "ggq_int8.hpp"
#include "ggq_launch.hpp"
#include "../../include/ggq.h"

namespace {

using namespace ggq;

constexpr uint32_t MAX_K = 131071;                 // 128 * 128 * k stays below 2^31

template <int DT, int TM, int TN, int WM, int WN, int KS, int NB>
hipError_t launch_tile(I8Args a, hipStream_t s)
{
    constexpr uint32_t lds = NB * (TM + TN) * I8_BK;
    static std::atomic<uint64_t> raised{0};
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(&linear_i8_tile<DT, TM, TN, WM, WN, KS, NB>), (int)lds, raised);
    if (e != hipSuccess) return e;
    a.tiles_m = (a.m + TM - 1) / TM;
    a.tiles_n = (a.n + TN - 1) / TN;
    hipLaunchKernelGGL((linear_i8_tile<DT, TM, TN, WM, WN, KS, NB>), dim3(a.tiles_m * a.tiles_n), dim3(WM * WN * KS * 64), lds, s, a);
    return hipGetLastError();
}

template <int DT, bool FEW>
hipError_t launch_rows16(const I8Args& a, hipStream_t s)
{
    const uint32_t lds = FEW ? a.m * ((a.k + 63u) / 64u * 64u + 16u) : 0u;                  // <= 16384 + 16 x 79 bytes
    hipLaunchKernelGGL((linear_i8_rows<DT, FEW>), dim3((a.n + 15u) / 16u), dim3(I8_ROW_WAVES * 64), lds, s, a);
    return hipGetLastError();
}

template <int DT>
hipError_t launch(const I8Args& a, hipStream_t s)
{
    if (a.m <= 16 && launchable((a.n + 15u) / 16u, I8_ROW_WAVES * 64)) return launch_rows16<DT, false>(a, s);
    // The tile that finishes first: rounds of workgroups over the chip times what a step of 128 k takes, in ns.  Measured at 256 x 4096 x 4096 (a part of
    // the chip), 512 x 10240 x 4096 and 4608 x 10240 x 4096 (all of it, at the clock it holds then): 256 x 256 (128 KiB of LDS: one workgroup per CU) 1330 ...
    // 1450 in one round, 1850 in several; 128 x 128 670 alone on a CU, 1050 for two; 64 x 64 350 alone, 420 for two.  A list of tiles that is too long for
    // one launch does not finish.
    auto tiles = [&](uint64_t t) { return ((a.m + t - 1) / t) * ((a.n + t - 1) / t); };
    const uint64_t t256 = tiles(256), t128 = tiles(128), t64 = tiles(64), never = ~0ull;
    const uint64_t big = !launchable(t256, 512) ? never : t256 <= 256 ? 1450 : (t256 + 255) / 256 * 1850;
    const uint64_t mid = !launchable(t128, 256) ? never : t128 <= 256 ? 670 : (t128 + 511) / 512 * 1050;
    const uint64_t small = !launchable(t64, 256) ? never : t64 <= 256 ? 350 : (t64 + 511) / 512 * 420;
    if (small <= mid && small <= big) return launch_tile<DT, 64, 64, 1, 2, 2, 4>(a, s);
    if (mid < big) return launch_tile<DT, 128, 128, 2, 2, 1, 2>(a, s);
    return launch_tile<DT, 256, 256, 2, 4, 1, 2>(a, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool unaligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == GGQ_F32 ? 3u : 1u)) != 0; }

}  // namespace

extern "C" int ggq_linear_int8(const void* xq, uint64_t x_stride, const float* x_scale, uint32_t m, const void* wq, uint64_t w_stride, const float* w_scale, uint32_t n,
                               uint32_t k, const void* bias, void* y, int dtype, void* hip_stream)
{
    if (dtype < 0 || dtype > 2 || k == 0 || k > MAX_K) return GGQ_ERR_ARG;
    if (m == 0 || n == 0) return GGQ_OK;
    if (m >= 1u << 31 || n >= 1u << 31 || !launchable(((uint64_t)m + 255) / 256 * (((uint64_t)n + 255) / 256), 512)) return GGQ_ERR_ARG;      // workgroups of the largest tile
    const uint64_t k16 = (k + 15u) & ~15u;
    if (!xq || !x_scale || !wq || !w_scale || !y || x_stride % 16 != 0 || w_stride % 16 != 0 || x_stride < k16 || w_stride < k16) return GGQ_ERR_ARG;
    if (!aligned16(xq) || !aligned16(wq) || unaligned(y, dtype) || unaligned(bias, dtype) || unaligned(x_scale, GGQ_F32) || unaligned(w_scale, GGQ_F32)) return GGQ_ERR_ALIGN;
    const I8Args a{static_cast<const uint8_t*>(xq), static_cast<const uint8_t*>(wq), x_scale, w_scale, static_cast<const uint8_t*>(bias), static_cast<uint8_t*>(y),
                   x_stride, w_stride, m, n, k, 0, 0};
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = dtype == GGQ_F16 ? launch<OUT_F16>(a, s) : (dtype == GGQ_BF16 ? launch<OUT_BF16>(a, s) : launch<OUT_F32>(a, s));
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}

extern "C" int ggq_linear_int8_few(const void* x, uint32_t m, const void* wq, uint64_t w_stride, const float* w_scale, uint32_t n, uint32_t k, const void* bias, void* y,
                                   int dtype, void* hip_stream)
{
    if (dtype < 0 || dtype > 2 || m > 16 || k == 0 || k % 8u != 0 || (uint64_t)m * k > (uint64_t)I8_FEW || !launchable(n / 16u + 1u, I8_ROW_WAVES * 64)) return GGQ_ERR_ARG;
    if (m == 0 || n == 0) return GGQ_OK;
    if (!x || !wq || !w_scale || !y || w_stride % 16 != 0 || w_stride < ((k + 15u) & ~15u)) return GGQ_ERR_ARG;
    if (!aligned16(x) || !aligned16(wq) || unaligned(y, dtype) || unaligned(bias, dtype) || unaligned(w_scale, GGQ_F32)) return GGQ_ERR_ALIGN;
    const I8Args a{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(wq), nullptr, w_scale, static_cast<const uint8_t*>(bias), static_cast<uint8_t*>(y), 0, w_stride, m, n, k, 0, 0};
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = dtype == GGQ_F16 ? launch_rows16<OUT_F16, true>(a, s) : (dtype == GGQ_BF16 ? launch_rows16<OUT_BF16, true>(a, s) : launch_rows16<OUT_F32, true>(a, s));
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}
