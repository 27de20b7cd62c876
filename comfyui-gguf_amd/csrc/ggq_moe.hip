// ggq_moe.hip -- C ABI over ggq_moe.hpp: router and expert products of a mixture-of-experts layer for a few tokens.
#include "ggq_moe.hpp"
#include "ggq_launch.hpp"
#include "../../include/ggq.h"

namespace {

using namespace ggq;

typedef hipError_t (*moe_fn)(MoeArgs, hipStream_t);

constexpr uint32_t HALF_LDS = 80u * 1024u, ALL_LDS = 160u * 1024u;

template <class F, int OUT, int MB>
hipError_t launch_up(MoeArgs a, hipStream_t s)
{
    constexpr uint32_t fixed = sizeof(MoeTable) + MOE_WAVES * MOE_MAX_TOKENS * 4 + 2 * MB * MOE_WAVES * 1024 + 64, mats = MB == 1 ? 1 : 2;
    const uint32_t pairs = a.tokens * a.top_k, most = (pairs < a.experts ? pairs : a.experts) * (a.ff / 16u);      // tiles, if every pair chose another expert
    const uint32_t blocks = (a.tokens + 15u) / 16u;
    a.spare = blocks > (uint32_t)MB ? blocks - MB : 0u;
    const uint32_t lds = MOE_WAVES * (mats * a.spare * 1024u + MOE_RING * Mf16Geom<F>::SLICE);
    if (fixed + lds > ALL_LDS) return hipErrorInvalidConfiguration;
    static std::atomic<uint64_t> raised{0};
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(&moe_up<F, OUT, MB>), (int)(ALL_LDS - fixed), raised);
    if (e != hipSuccess) return e;
    // as many workgroups as the chip holds (MB > 1: their registers leave one per CU), dealt the same number of tiles
    const uint32_t fit = MB == 1 && fixed + lds <= HALF_LDS ? 512u : 256u;
    hipLaunchKernelGGL((moe_up<F, OUT, MB>), dim3(most < fit ? most : fit), dim3(MOE_WAVES * 64), lds, s, a);
    return hipGetLastError();
}

// Workgroups of `waves` waves that share the (expert, span) list of moe_down's 16 rows: so many that every CU gets 16 waves.
uint32_t down_parts(uint32_t dim, uint32_t waves)
{
    const uint32_t tiles = dim / 16u, want = 256u * (16u / waves);
    return tiles >= want ? 1u : (want / tiles < 8u ? want / tiles : 8u);
}

template <class F, int OUT, int MB, int W>
hipError_t launch_down_w(MoeArgs a, hipStream_t s, bool& fits)
{
    constexpr uint32_t fixed = sizeof(MoeTable) + MOE_MAX_TOKENS * MOE_MAX_TOPK * 4 + 2 * W * MOE_MAX_TOKENS * 4 + 64;
    const uint32_t blocks = (2u * a.tokens + 15u) / 16u;
    a.spare = blocks > (uint32_t)MB ? blocks - MB : 0u;
    const uint32_t sums = W * (a.tokens * 64u + a.spare * 1024u);
    const uint32_t lds = sums + W * MOE_RING * Mf16Geom<F>::SLICE;
    fits = fixed + lds <= ALL_LDS;
    if (!fits) return hipSuccess;
    static std::atomic<uint64_t> raised{0};
    hipError_t e = allow_lds(reinterpret_cast<const void*>(&moe_down<F, OUT, MB, W>), (int)(ALL_LDS - fixed), raised);
    if (e != hipSuccess) return e;
    a.parts = down_parts(a.dim, W);
    hipLaunchKernelGGL((moe_down<F, OUT, MB, W>), dim3(a.dim / 16u, a.parts), dim3(W * 64), lds, s, a);
    e = hipGetLastError();
    if (e != hipSuccess || a.parts == 1) return e;
    const uint32_t quads = a.tokens * a.dim / 4u;
    hipLaunchKernelGGL((moe_combine<OUT>), dim3((quads + 255u) / 256u), dim3(256), 0, s, a.part, a.y, a.parts, quads);
    return hipGetLastError();
}

// One block of columns: 16 waves per workgroup, so that from 4096 rows of y on no second pass over parts is needed (it is 4 us); else 8, for the registers.
template <class F, int OUT, int MB>
hipError_t launch_down(MoeArgs a, hipStream_t s)
{
    bool fits = false;
    if constexpr (MB == 1) {
        const hipError_t e = launch_down_w<F, OUT, 1, 16>(a, s, fits);
        if (e != hipSuccess || fits) return e;
    }
    const hipError_t e = launch_down_w<F, OUT, MB, 8>(a, s, fits);
    return e != hipSuccess || fits ? e : hipErrorInvalidConfiguration;
}

struct MoeEntry { int qtype, block_size; moe_fn up[2][3], down[2][3]; };                              // [dtype f16 / bf16][blocks of 16 columns 1 / 2 / 4]
#define GGQ_MOE_ROW(FN, F, OUT) {FN<F, OUT, 1>, FN<F, OUT, 2>, FN<F, OUT, 4>}
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

// Blocks of 16 columns for `per_token` columns of each token of an expert: room for three standard deviations above the mean of evenly spread choices (more
// tokens than that on one expert are multiplied block by block, with their sums in LDS).
int column_blocks(uint32_t tokens, uint32_t top_k, uint32_t experts, uint32_t per_token)
{
    const double mean = (double)tokens * top_k / experts, most = mean + 3.0 * __builtin_sqrt(mean);
    if (per_token == 2 && tokens > 32) return 2;                    // the sums of what may overflow have to fit the LDS
    const double cols = (most < tokens ? most : (double)tokens) * per_token;
    return cols <= 16.0 ? 0 : (cols <= 32.0 ? 1 : 2);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

extern "C" uint64_t ggq_moe_route_workspace(uint32_t tokens, uint32_t experts) { return experts > (uint32_t)MOE_ROUTE_WAVES ? (uint64_t)tokens * experts * 8u : 0u; }

extern "C" int ggq_moe_route(const void* x, const void* router, uint32_t tokens, uint32_t dim, uint32_t experts, uint32_t top_k, int renormalize, int32_t* ids,
                             float* weights, int dtype, int router_dtype, void* workspace, uint64_t workspace_bytes, void* hip_stream)
{
    if ((dtype != GGQ_F16 && dtype != GGQ_BF16) || (router_dtype != dtype && router_dtype != GGQ_F32) || dim == 0 || dim % 8u != 0 || experts == 0 ||
        experts > (uint32_t)MOE_MAX_EXPERTS || top_k == 0 || top_k > (uint32_t)MOE_MAX_TOPK || top_k > experts || tokens > 65535u) return GGQ_ERR_ARG;
    if (tokens == 0) return GGQ_OK;
    const uint64_t need = ggq_moe_route_workspace(tokens, experts);
    if (!x || !router || !ids || !weights || (need && !workspace) || workspace_bytes < need) return GGQ_ERR_ARG;
    if (!aligned16(x) || !aligned16(router) || !aligned4(ids) || !aligned4(weights) || (reinterpret_cast<uintptr_t>(workspace) & 7u)) return GGQ_ERR_ALIGN;
    const uint8_t *xb = static_cast<const uint8_t*>(x), *rb = static_cast<const uint8_t*>(router);
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const int wide = router_dtype == GGQ_F32 ? 1 : 0;
    if (need == 0) {
        typedef void (*route_fn)(const uint8_t*, const uint8_t*, uint32_t, uint32_t, uint32_t, int, int32_t*, float*);
        static const route_fn ROUTE[2][2] = {{moe_route<OUT_F16, OUT_F16>, moe_route<OUT_F16, OUT_F32>}, {moe_route<OUT_BF16, OUT_BF16>, moe_route<OUT_BF16, OUT_F32>}};
        hipLaunchKernelGGL(ROUTE[dtype][wide], dim3(tokens), dim3(MOE_ROUTE_WAVES * 64), 0, s, xb, rb, dim, experts, top_k, renormalize, ids, weights);
    } else {
        typedef void (*scores_fn)(const uint8_t*, const uint8_t*, uint32_t, uint32_t, double*);
        static const scores_fn SCORES[2][2] = {{moe_scores<OUT_F16, OUT_F16>, moe_scores<OUT_F16, OUT_F32>}, {moe_scores<OUT_BF16, OUT_BF16>, moe_scores<OUT_BF16, OUT_F32>}};
        hipLaunchKernelGGL(SCORES[dtype][wide], dim3((experts + 3u) / 4u, tokens), dim3(256), 0, s, xb, rb, dim, experts, static_cast<double*>(workspace));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return hip_fail(e);
        hipLaunchKernelGGL(moe_pick, dim3(tokens), dim3(MOE_MAX_EXPERTS), 0, s, static_cast<const double*>(workspace), experts, top_k, renormalize, ids, weights);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}

extern "C" uint64_t ggq_moe_workspace(uint32_t tokens, uint32_t top_k, uint32_t dim, uint32_t ff)
{
    const uint64_t hidden = ((uint64_t)tokens * top_k * ff * 4u + 15u) & ~15ull;
    return dim < 16u ? hidden : hidden + (uint64_t)down_parts(dim, 8) * tokens * dim * 4u;              // 8 waves: the most parts
}

extern "C" int ggq_moe_experts(const ggq_moe_desc* d, void* hip_stream)
{
    if (!d) return GGQ_ERR_ARG;
    const MoeEntry *up = entry(d->up_qtype), *down = entry(d->down_qtype);
    if (!up || !down) return GGQ_ERR_QTYPE;
    auto whole = [](const MoeEntry* e, uint32_t k) { return k != 0 && k % (e->block_size == 32 ? 64u : 256u) == 0; };
    if ((d->dtype != GGQ_F16 && d->dtype != GGQ_BF16) || (d->act != 0 && d->act != 1) || !whole(up, d->dim) || !whole(down, d->ff) || d->dim % 16u != 0 || d->ff % 16u != 0 || d->dim > (1u << 24) || d->ff > (1u << 24) ||
        d->experts == 0 || d->experts > (uint32_t)MOE_MAX_EXPERTS || d->top_k == 0 || d->top_k > (uint32_t)MOE_MAX_TOPK || d->tokens > (uint32_t)MOE_MAX_TOKENS) return GGQ_ERR_ARG;
    if (d->tokens == 0) return GGQ_OK;
    if (!d->x || !d->ids || !d->weights || !d->gate || !d->up || !d->down || !d->y || !d->workspace || d->workspace_bytes < ggq_moe_workspace(d->tokens, d->top_k, d->dim, d->ff))
        return GGQ_ERR_ARG;
    if (!aligned16(d->x) || !aligned16(d->gate) || !aligned16(d->up) || !aligned16(d->down) || !aligned16(d->workspace) || !aligned4(d->ids) || !aligned4(d->weights) ||
        (reinterpret_cast<uintptr_t>(d->y) & 7u)) return GGQ_ERR_ALIGN;
    MoeArgs a{static_cast<const uint8_t*>(d->x), d->ids, d->weights, static_cast<const uint8_t*>(d->gate), static_cast<const uint8_t*>(d->up),
              static_cast<const uint8_t*>(d->down), static_cast<uint8_t*>(d->y), static_cast<uint8_t*>(d->workspace), nullptr, d->tokens, d->top_k, d->experts, d->dim, d->ff, d->act, 1, 0};
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(d->workspace) + (((uint64_t)a.tokens * a.top_k * a.ff * 4u + 15u) & ~15ull));
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    hipError_t e = up->up[d->dtype][column_blocks(a.tokens, a.top_k, a.experts, 1)](a, s);
    if (e == hipSuccess) e = down->down[d->dtype][column_blocks(a.tokens, a.top_k, a.experts, 2)](a, s);
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}
