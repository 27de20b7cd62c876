// ggq_moe.hip -- C ABI over ggq_moe.hpp: router and expert products of a mixture-of-experts layer for a few tokens.
#include "ggq_moe.hpp"
#include "ggq_launch.hpp"
#include "../../include/ggq.h"

namespace {

using namespace ggq;

typedef hipError_t (*moe_fn)(const MoeArgs&, hipStream_t);

template <class F, int OUT, int MB>
hipError_t launch_up(const MoeArgs& a, hipStream_t s)
{
    const uint32_t pairs = a.tokens * a.top_k, experts = pairs < a.experts ? pairs : a.experts;      // at most so many are chosen
    hipLaunchKernelGGL((moe_up<F, OUT, MB>), dim3(a.ff / 16u, experts), dim3(MOE_UP_WAVES * 64), 0, s, a);
    return hipGetLastError();
}

template <class F, int OUT, int MB>
hipError_t launch_down(const MoeArgs& a, hipStream_t s)
{
    const uint32_t lds = MOE_DOWN_WAVES * a.tokens * 64u;                                             // <= 32 KiB, beside up to 41 KiB of static LDS
    static std::atomic<uint64_t> raised{0};
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(&moe_down<F, OUT, MB>), MOE_DOWN_WAVES * MOE_MAX_TOKENS * 64, raised);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((moe_down<F, OUT, MB>), dim3(a.dim / 16u), dim3(MOE_DOWN_WAVES * 64), lds, s, a);
    return hipGetLastError();
}

struct MoeEntry { int qtype, block_size; moe_fn up[2][2], down[2][2]; };                              // [dtype f16 / bf16][MB 1 / 2]
#define GGQ_MOE_ROW(FN, F, OUT) {FN<F, OUT, 1>, FN<F, OUT, 2>}
#define GGQ_MOE(F) MoeEntry { F::ID, F::BS, {GGQ_MOE_ROW(launch_up, F, OUT_F16), GGQ_MOE_ROW(launch_up, F, OUT_BF16)}, \
                              {GGQ_MOE_ROW(launch_down, F, OUT_F16), GGQ_MOE_ROW(launch_down, F, OUT_BF16)} }
const MoeEntry MOE[] = {
    GGQ_MOE(FmtQ4_0), GGQ_MOE(FmtQ4_1), GGQ_MOE(FmtQ5_0), GGQ_MOE(FmtQ5_1), GGQ_MOE(FmtQ8_0),
    GGQ_MOE(FmtQ2_K), GGQ_MOE(FmtQ3_K), GGQ_MOE(FmtQ4_K), GGQ_MOE(FmtQ5_K), GGQ_MOE(FmtQ6_K),
    GGQ_MOE(FmtIQ4_NL), GGQ_MOE(FmtIQ4_XS),
};

const MoeEntry* entry(int qtype)
{
    for (const MoeEntry& e : MOE)
        if (e.qtype == qtype) return &e;
    return nullptr;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

extern "C" int ggq_moe_route(const void* x, const void* router, uint32_t tokens, uint32_t dim, uint32_t experts, uint32_t top_k, int renormalize, int32_t* ids,
                             float* weights, int dtype, int router_dtype, void* hip_stream)
{
    if ((dtype != GGQ_F16 && dtype != GGQ_BF16) || (router_dtype != dtype && router_dtype != GGQ_F32) || dim == 0 || dim % 8u != 0 || experts == 0 || experts > (uint32_t)MOE_MAX_EXPERTS || top_k == 0 ||
        top_k > (uint32_t)MOE_MAX_TOPK || top_k > experts || tokens > 0x7FFFFFFFu / MOE_MAX_TOPK) return GGQ_ERR_ARG;
    if (tokens == 0) return GGQ_OK;
    if (!x || !router || !ids || !weights) return GGQ_ERR_ARG;
    if (!aligned16(x) || !aligned16(router) || !aligned4(ids) || !aligned4(weights)) return GGQ_ERR_ALIGN;
    typedef void (*route_fn)(const uint8_t*, const uint8_t*, uint32_t, uint32_t, uint32_t, int, int32_t*, float*);
    static const route_fn ROUTE[2][2] = {{moe_route<OUT_F16, OUT_F16>, moe_route<OUT_F16, OUT_F32>}, {moe_route<OUT_BF16, OUT_BF16>, moe_route<OUT_BF16, OUT_F32>}};
    hipLaunchKernelGGL(ROUTE[dtype][router_dtype == GGQ_F32 ? 1 : 0], dim3(tokens), dim3(MOE_ROUTE_THREADS), 0, static_cast<hipStream_t>(hip_stream),
                       static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(router), dim, experts, top_k, renormalize, ids, weights);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}

extern "C" uint64_t ggq_moe_workspace(uint32_t tokens, uint32_t top_k, uint32_t ff) { return (uint64_t)tokens * top_k * ff * 4u; }

extern "C" int ggq_moe_experts(const ggq_moe_desc* d, void* hip_stream)
{
    if (!d) return GGQ_ERR_ARG;
    const MoeEntry *up = entry(d->up_qtype), *down = entry(d->down_qtype);
    if (!up || !down) return GGQ_ERR_QTYPE;
    auto whole = [](const MoeEntry* e, uint32_t k) { return k != 0 && k % (e->block_size == 32 ? 64u : 256u) == 0; };
    if ((d->dtype != GGQ_F16 && d->dtype != GGQ_BF16) || (d->act != 0 && d->act != 1) || !whole(up, d->dim) || !whole(down, d->ff) || d->dim % 16u != 0 || d->ff % 16u != 0 ||
        d->experts == 0 || d->experts > (uint32_t)MOE_MAX_EXPERTS || d->top_k == 0 || d->top_k > (uint32_t)MOE_MAX_TOPK || d->tokens > (uint32_t)MOE_MAX_TOKENS) return GGQ_ERR_ARG;
    if (d->tokens == 0) return GGQ_OK;
    if (!d->x || !d->ids || !d->weights || !d->gate || !d->up || !d->down || !d->y || !d->workspace || d->workspace_bytes < ggq_moe_workspace(d->tokens, d->top_k, d->ff))
        return GGQ_ERR_ARG;
    if (!aligned16(d->x) || !aligned16(d->gate) || !aligned16(d->up) || !aligned16(d->down) || !aligned16(d->workspace) || !aligned4(d->ids) || !aligned4(d->weights) ||
        (reinterpret_cast<uintptr_t>(d->y) & 1u)) return GGQ_ERR_ALIGN;
    const MoeArgs a{static_cast<const uint8_t*>(d->x), d->ids, d->weights, static_cast<const uint8_t*>(d->gate), static_cast<const uint8_t*>(d->up),
                    static_cast<const uint8_t*>(d->down), static_cast<uint8_t*>(d->y), static_cast<uint8_t*>(d->workspace), d->tokens, d->top_k, d->experts, d->dim, d->ff, d->act};
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    hipError_t e = up->up[d->dtype][d->tokens > 16 ? 1 : 0](a, s);
    if (e == hipSuccess) e = down->down[d->dtype][d->tokens > 8 ? 1 : 0](a, s);
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}
