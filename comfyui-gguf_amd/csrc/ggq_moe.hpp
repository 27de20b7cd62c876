// ggq_moe.hpp -- gfx950 device code: a mixture-of-experts layer for a few tokens, straight from packed GGUF expert weights.
//
// Mathematics, per token x:  l = Wr x;  p = softmax(l);  the top_k largest p (equal ones to the lower index), divided by their sum if asked;
//     y = sum_s p_s Wd[e_s] (act(Wg[e_s] x) * (Wu[e_s] x)).
//
// Three kernels: the router (moe_route, a workgroup per token), the gate and up projections with the activation (moe_up), the down projection with the
// weighted sum over experts (moe_down).  What bounds them is reading the packed bytes of the chosen experts, each ONCE for all tokens that chose it:
//   * moe_up: a workgroup owns 16 rows of Wg and the same 16 rows of Wu of one chosen expert; half of its waves contract the gate rows, half the up
//     rows, each a part of k; the tokens of that expert are the 16 columns of v_mfma_f32_16x16x32 (A = 16 rows of decoded weights).
//   * moe_down: a workgroup owns 16 rows of the output for ALL tokens and walks every chosen expert, so the sum over a token's experts needs no second
//     pass and no atomics; its waves take equal, contiguous parts of the (expert, piece of k) list.
//   * the list of chosen experts and the tokens of each are found by every workgroup itself from the ids (at most 64 x 16 of them).
// A weight is the reference's value bit for bit (ggq_device.hpp: same decode, same fp16 operations, then the rounding to the activations' type).
// The hidden vector act(g) * u is kept in two parts of the activations' type -- its rounded value and the rounded rest -- which ride as two columns of
// the down product: about 16 (bf16) or 22 (fp16) bits, for no more weight traffic.  The fp16 rest is kept times 2^11, out of the subnormals.
// Sums: fp32 in the MFMA's order, k-parts in wave order, experts in ascending order within a wave: the result does not depend on timing.
#pragma once

#include "ggq_mfma16.hpp"
#include "ggq_rows.hpp"

namespace ggq {

constexpr int MOE_MAX_TOKENS = 64, MOE_MAX_TOPK = 16, MOE_MAX_EXPERTS = 512;
constexpr int MOE_WORDS = MOE_MAX_EXPERTS / 32;

// ---- the router: a workgroup per token, a wave per expert in turn

// Eight products, formed and added in fp64: which of two close scores is larger decides which experts run.  RT: the router's type, fp32 in GGUF files.
template <int OUT, int RT> GGQ_DEV double moe_dot8(const uint8_t* x, const uint8_t* w)
{
    float u[8], v[8];
    row_load8<OUT>(x, 0, 8, u);
    row_load8<RT>(w, 0, 8, v);
    double s[4];
#pragma unroll
    for (int k = 0; k < 4; k++) s[k] = (double)u[2 * k] * (double)v[2 * k] + (double)u[2 * k + 1] * (double)v[2 * k + 1];
    return (s[0] + s[1]) + (s[2] + s[3]);
}

constexpr int MOE_ROUTE_THREADS = 512;

template <int OUT, int RT>
__global__ __launch_bounds__(MOE_ROUTE_THREADS) void moe_route(const uint8_t* __restrict__ x_, const uint8_t* __restrict__ router_, uint32_t dim, uint32_t experts,
                                                              uint32_t top_k, int renormalize, int32_t* __restrict__ ids, float* __restrict__ weights)
{
    __shared__ double score[MOE_MAX_EXPERTS];
    __shared__ double chosen[MOE_MAX_TOPK];
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint8_t* x = x_ + (uint64_t)blockIdx.x * dim * 2;
    for (uint32_t e = wave; e < experts; e += MOE_ROUTE_THREADS / 64) {
        constexpr uint32_t RB = RT == OUT_F32 ? 4 : 2;
        const uint8_t* w = router_ + (uint64_t)e * dim * RB;
        double acc = 0.0;
        for (uint32_t i = lane * 8u; i < dim; i += 512u)
            acc += moe_dot8<OUT, RT>(x + (uint64_t)i * 2, w + (uint64_t)i * RB);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
        if (lane == 0) score[e] = acc;
    }
    __syncthreads();
    // rank of an expert = how many come before it; a NaN comes last (its weight is NaN all the same)
    const bool mine = t < experts;
    uint32_t rank = ~0u;
    if (mine) {
        const double own = score[t];
        rank = 0;
        for (uint32_t e = 0; e < experts; e++) {
            const double o = score[e];
            rank += (o > own || (o == own && e < t) || (own != own && (o == o || e < t))) ? 1u : 0u;
        }
        if (rank < top_k) {
            chosen[rank] = own;
            ids[(uint64_t)blockIdx.x * top_k + rank] = (int32_t)t;
        }
    }
    __syncthreads();
    if (rank < top_k) {
        const double top = chosen[0];
        float sum = 0.0f;
        if (renormalize) for (uint32_t s = 0; s < top_k; s++) sum += __expf((float)(chosen[s] - top));
        else for (uint32_t e = 0; e < experts; e++) sum += __expf((float)(score[e] - top));
        weights[(uint64_t)blockIdx.x * top_k + rank] = __expf((float)(score[t] - top)) * __builtin_amdgcn_rcpf(sum);
    }
}

// ---- which experts were chosen, and by whom

// bit e of words[]: some token chose expert e.  Called by the whole workgroup; ends with a barrier.
GGQ_DEV void moe_mark(uint32_t* words, const int32_t* __restrict__ ids, uint32_t pairs, uint32_t experts)
{
    if (threadIdx.x < MOE_WORDS) words[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < pairs; p += blockDim.x) {
        const uint32_t e = (uint32_t)ids[p];
        if (e < experts) atomicOr(&words[e >> 5], 1u << (e & 31u));
    }
    __syncthreads();
}

// the `a`-th chosen expert in ascending order, or -1 (wave-uniform)
GGQ_DEV int moe_nth(const uint32_t* words, uint32_t a)
{
    for (int w = 0; w < MOE_WORDS; w++) {
        uint32_t b = words[w];
        const uint32_t n = (uint32_t)__builtin_popcount(b);
        if (a >= n) { a -= n; continue; }
        for (; a > 0; a--) b &= b - 1u;
        return 32 * w + __builtin_ctz(b);
    }
    return -1;
}

// The tokens that chose `expert`: lane t looks at token t.  `slot`: its first place in ids, `weight`: the sum over its places (the same expert twice
// counts twice).  Returns the mask of tokens.
GGQ_DEV uint64_t moe_tokens(const int32_t* __restrict__ ids, const float* __restrict__ weights, uint32_t tokens, uint32_t top_k, int expert, uint32_t& slot, float& weight)
{
    const uint32_t t = threadIdx.x & 63u;
    bool has = false;
    slot = 0;
    weight = 0.0f;
    if (t < tokens)
        for (uint32_t s = top_k; s-- > 0;)
            if (ids[t * top_k + s] == expert) {
                has = true;
                slot = t * top_k + s;
                weight += weights[t * top_k + s];
            }
    return __ballot(has);
}

GGQ_DEV float moe_act(float g, int act)
{
    if (act == 0) return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g));                                    // silu
    const float u = 0.7978845608028654f * (g + 0.044715f * g * g * g);                                     // gelu, tanh form: g / (1 + exp(-2u))
    return g * __builtin_amdgcn_rcpf(1.0f + __expf(-2.0f * u));
}

// one 256-element span of 16 rows, packed bytes to registers: as in linear_mfma16 (a short last span only in the 32-element formats)
template <class F> GGQ_DEV void moe_fetch(gcptr rows, uint64_t row_bytes, uint32_t span, uint32_t n_spans, uint32_t tail_len, u32x4 (&pf)[Mf16Geom<F>::NUW])
{
    using G = Mf16Geom<F>;
    const int lane = (int)(threadIdx.x & 63u);
    const bool tail = F::BS == 32 && span + 1 == n_spans && tail_len != (uint32_t)MF_SPAN;                 // wave-uniform
    const uint32_t span_bytes = (tail ? tail_len : (uint32_t)MF_SPAN) / (uint32_t)F::BS * (uint32_t)F::TS;
#pragma unroll
    for (int u = 0; u < G::NUW; u++) {
        const uint32_t unit = (uint32_t)(lane + 64 * u), ur = unit / (uint32_t)G::U, uu = unit % (uint32_t)G::U;
        const gcptr at = rows + (uint64_t)(ur < 16u ? ur : 0u) * row_bytes + (uint64_t)span * G::SPAN_BYTES;
        const uint32_t a = G::SKEW ? ((uint32_t)(uintptr_t)at & 15u) : 0u;
        // loads start 16-byte aligned: what they read past the span lies in a unit that also holds bytes of the tensor
        pf[u] = (ur < 16u && uu * 16u < a + span_bytes) ? gload16<true>(at - a + uu * 16u) : u32x4{0, 0, 0, 0};
        if (tail) {                                                                                        // blocks past the end decode to zeros
            const int32_t valid = (int32_t)(a + span_bytes) - (int32_t)(uu * 16u);
            uint32_t d[4] = {pf[u].x, pf[u].y, pf[u].z, pf[u].w};
#pragma unroll
            for (int i = 0; i < 4; i++) d[i] &= valid >= 4 * i + 4 ? 0xFFFFFFFFu : (valid == 4 * i + 2 ? 0x0000FFFFu : 0u);
            pf[u] = u32x4{d[0], d[1], d[2], d[3]};
        }
    }
}

template <class F> GGQ_DEV void moe_stash(uint8_t* slice, const u32x4 (&pf)[Mf16Geom<F>::NUW])
{
    using G = Mf16Geom<F>;
    const int lane = (int)(threadIdx.x & 63u);
#pragma unroll
    for (int u = 0; u < G::NUW; u++) {
        const uint32_t unit = (uint32_t)(lane + 64 * u), ur = unit / (uint32_t)G::U, uu = unit % (uint32_t)G::U;
        if (ur < 16u) *reinterpret_cast<u32x4*>(slice + ur * G::ROW_STRIDE + uu * 16u) = pf[u];
    }
}

// acc += 16 rows of decoded weights (in `slice`, first row at byte `skew` of its pitch) x MB blocks of 16 columns; col[]: this lane's column at element 32 c
template <class F, int OUT, int MB>
GGQ_DEV void moe_span(const uint8_t* wspan, const GGQ_GLOBAL uint8_t* const (&col)[MB], uint32_t span, uint32_t k_len, f32x4 (&acc)[MB])
{
    constexpr int CPB = F::BS / 8;
    const int c = (int)(threadIdx.x & 63u) >> 4;
#pragma unroll
    for (int g = 0; g < 2; g++) {
        u32x4 xf[MB][4];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            const GGQ_GLOBAL uint8_t* src = col[mb] + (uint64_t)span * (MF_SPAN * 2) + (uint32_t)(g * 256);
            if constexpr (F::BS == 32) {                                                                   // past the end of k: zeros
                if (span * (uint32_t)MF_SPAN + (uint32_t)(128 * g + 32 * c) >= k_len) src = (GGQ_GLOBAL const uint8_t*)MF16_ZEROS;
            }
#pragma unroll
            for (int t = 0; t < 4; t++) xf[mb][t] = *(GGQ_GLOBAL const u32x4*)(src + t * 16);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int j = 16 * g + 4 * c + t;
            const Fields f = F::template fields<true>(wspan + (j / CPB) * F::TS, j % CPB);
            uint32_t w[4];
            weights8<F, OUT>(f, w);
            const u32x4 wa{w[0], w[1], w[2], w[3]};
#pragma unroll
            for (int mb = 0; mb < MB; mb++) acc[mb] = mfma16<OUT>(wa, xf[mb][t], acc[mb]);
        }
    }
}

struct MoeArgs {
    const uint8_t* x;
    const int32_t* ids;
    const float* weights;
    const uint8_t *gate, *up, *down;
    uint8_t* y;
    uint8_t* hidden;                 // [2][tokens * top_k][ff] of the activations' type: the rounded value, then the rest
    uint32_t tokens, top_k, experts, dim, ff;
    int act;
};

constexpr int MOE_UP_WAVES = 8, MOE_DOWN_WAVES = 8;

// hidden = act(Wg x) * (Wu x) for 16 hidden rows of one chosen expert.  Waves 0, 2, 4, ... contract gate rows, waves 1, 3, 5, ... up rows.
template <class F, int OUT, int MB>
__global__ __launch_bounds__(MOE_UP_WAVES * 64) void moe_up(const MoeArgs a)
{
    using G = Mf16Geom<F>;
    __shared__ uint32_t words[MOE_WORDS];
    __shared__ uint32_t slots[MOE_MAX_TOKENS];                                     // per column: where its hidden row goes (= token * top_k + place)
    constexpr int WORK = MOE_UP_WAVES * G::SLICE > MOE_UP_WAVES * MB * 1024 ? MOE_UP_WAVES * G::SLICE : MOE_UP_WAVES * MB * 1024;
    __shared__ __attribute__((aligned(16))) uint8_t work[WORK];
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, c = lane >> 4;
    const uint32_t pairs = a.tokens * a.top_k;

    moe_mark(words, a.ids, pairs, a.experts);
    const int expert = moe_nth(words, blockIdx.y);
    if (expert < 0) return;                                                        // fewer experts than the grid allows for
    uint32_t slot;
    float weight;
    const uint64_t mask = moe_tokens(a.ids, a.weights, a.tokens, a.top_k, expert, slot, weight);
    const uint32_t n_cols = (uint32_t)__builtin_popcountll(mask);
    if (wave == 0 && ((mask >> lane) & 1u)) slots[__builtin_popcountll(mask & ((1ull << lane) - 1ull))] = slot;
    __syncthreads();

    const uint32_t row0 = blockIdx.x * 16u;
    const uint64_t row_bytes = (uint64_t)(a.dim / F::BS) * F::TS;
    const uint32_t n_spans = (a.dim + MF_SPAN - 1) / MF_SPAN, tail_len = a.dim - (n_spans - 1) * (uint32_t)MF_SPAN;
    const gcptr rows = (gcptr)((wave & 1u) ? a.up : a.gate) + ((uint64_t)(uint32_t)expert * a.ff + row0) * row_bytes;
    uint8_t* slice = work + wave * G::SLICE;
    for (uint32_t c0 = 0; c0 < n_cols; c0 += MB * 16) {                            // more columns than fit: the rows are read again, from the caches
        const GGQ_GLOBAL uint8_t* col[MB];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            const uint32_t v = c0 + (uint32_t)(mb * 16) + r;
            col[mb] = (GGQ_GLOBAL const uint8_t*)a.x + (uint64_t)(slots[v < n_cols ? v : 0u] / a.top_k) * a.dim * 2 + c * 64u;
        }
        f32x4 acc[MB];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) acc[mb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        u32x4 pf[G::NUW];
        uint32_t span = wave >> 1;
        if (span < n_spans) moe_fetch<F>(rows, row_bytes, span, n_spans, tail_len, pf);
        for (; span < n_spans; span += MOE_UP_WAVES / 2) {
            moe_stash<F>(slice, pf);
            wave_sync();
            if (span + MOE_UP_WAVES / 2 < n_spans) moe_fetch<F>(rows, row_bytes, span + MOE_UP_WAVES / 2, n_spans, tail_len, pf);
            const uint32_t skew = G::SKEW ? (uint32_t)(uintptr_t)(rows + (uint64_t)r * row_bytes + (uint64_t)span * G::SPAN_BYTES) & 15u : 0u;
            moe_span<F, OUT, MB>(slice + r * G::ROW_STRIDE + skew, col, span, a.dim, acc);
            wave_sync();
        }
        __syncthreads();
        f32x4* red = reinterpret_cast<f32x4*>(work);
#pragma unroll
        for (int mb = 0; mb < MB; mb++) red[(wave * MB + (uint32_t)mb) * 64u + lane] = acc[mb];
        __syncthreads();
        if (wave < (uint32_t)MB) {
            f32x4 g = red[wave * 64u + lane], u = red[(MB + wave) * 64u + lane];
            for (uint32_t w = 2; w < MOE_UP_WAVES; w += 2) {
                g += red[(w * MB + wave) * 64u + lane];
                u += red[((w + 1) * MB + wave) * 64u + lane];
            }
            const uint32_t v = c0 + wave * 16u + r;                                // D[row = 4c + i][column = r]
            if (v < n_cols) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    float h0 = moe_act(g[2 * p], a.act) * u[2 * p], h1 = moe_act(g[2 * p + 1], a.act) * u[2 * p + 1];
                    asm volatile("" : "+v"(h0), "+v"(h1));                         // the product rounded to fp32 (no v_fma_mix with the conversion): both parts see it
                    if constexpr (OUT == OUT_F16) {
                        const h2 q{(_Float16)h0, (_Float16)h1};
                        hi[p] = as_u32(q);
                        lo[p] = as_u32(h2{(_Float16)__builtin_ldexpf(h0 - (float)q.x, 11), (_Float16)__builtin_ldexpf(h1 - (float)q.y, 11)});
                    } else {
                        hi[p] = pack_bf16(h0, h1);
                        lo[p] = pack_bf16(h0 - bits_f32(hi[p] << 16), h1 - bits_f32(hi[p] & 0xFFFF0000u));
                    }
                }
                uint8_t* dst = a.hidden + ((uint64_t)slots[v] * a.ff + row0 + 4u * c) * 2;
                *reinterpret_cast<u32x2*>(dst) = u32x2{hi[0], hi[1]};
                *reinterpret_cast<u32x2*>(dst + (uint64_t)pairs * a.ff * 2) = u32x2{lo[0], lo[1]};
            }
        }
        __syncthreads();                                                           // the partial sums become weight slices again
    }
}

// 16 rows of y for every token.  A wave's columns are (token, part of the hidden vector): column 2 i the value, 2 i + 1 the rest of token i of the expert.
template <class F, int OUT, int MB>
__global__ __launch_bounds__(MOE_DOWN_WAVES * 64) void moe_down(const MoeArgs a)
{
    using G = Mf16Geom<F>;
    extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];                  // y of each wave: [wave][token][16] floats
    __shared__ uint32_t words[MOE_WORDS];
    __shared__ uint32_t slots[MOE_DOWN_WAVES][MOE_MAX_TOKENS];
    __shared__ float shares[MOE_DOWN_WAVES][MOE_MAX_TOKENS];
    __shared__ __attribute__((aligned(16))) uint8_t work[MOE_DOWN_WAVES * G::SLICE];
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, c = lane >> 4;
    const uint32_t pairs = a.tokens * a.top_k;
    float* part = reinterpret_cast<float*>(dyn) + (uint64_t)wave * a.tokens * 16u;
    for (uint32_t i = lane; i < a.tokens * 16u; i += 64u) part[i] = 0.0f;

    moe_mark(words, a.ids, pairs, a.experts);
    uint32_t n_experts = 0;
    for (int w = 0; w < MOE_WORDS; w++) n_experts += (uint32_t)__builtin_popcount(words[w]);
    const uint32_t row0 = blockIdx.x * 16u;
    const uint64_t row_bytes = (uint64_t)(a.ff / F::BS) * F::TS;
    const uint32_t n_spans = (a.ff + MF_SPAN - 1) / MF_SPAN, tail_len = a.ff - (n_spans - 1) * (uint32_t)MF_SPAN;
    const uint32_t items = n_experts * n_spans, each = (items + MOE_DOWN_WAVES - 1) / MOE_DOWN_WAVES;
    const uint32_t last = (wave + 1) * each < items ? (wave + 1) * each : items;
    uint8_t* slice = work + wave * G::SLICE;

    for (uint32_t item = wave * each; item < last;) {                              // one expert at a time: items [item, stop)
        const uint32_t nth = item / n_spans, span0 = item - nth * n_spans;
        const uint32_t stop = (nth + 1) * n_spans < last ? (nth + 1) * n_spans : last, span1 = span0 + (stop - item);
        const int expert = moe_nth(words, nth);
        uint32_t slot;
        float weight;
        const uint64_t mask = moe_tokens(a.ids, a.weights, a.tokens, a.top_k, expert, slot, weight);
        const uint32_t n_cols = 2u * (uint32_t)__builtin_popcountll(mask);
        if ((mask >> lane) & 1u) {
            const uint32_t at = (uint32_t)__builtin_popcountll(mask & ((1ull << lane) - 1ull));
            slots[wave][at] = slot;
            shares[wave][at] = weight;
        }
        wave_sync();
        const gcptr rows = (gcptr)a.down + ((uint64_t)(uint32_t)expert * a.dim + row0) * row_bytes;
        for (uint32_t c0 = 0; c0 < n_cols; c0 += MB * 16) {
            const GGQ_GLOBAL uint8_t* col[MB];
#pragma unroll
            for (int mb = 0; mb < MB; mb++) {
                const uint32_t v0 = c0 + (uint32_t)(mb * 16) + r, v = v0 < n_cols ? v0 : 0u;
                col[mb] = (GGQ_GLOBAL const uint8_t*)a.hidden + ((uint64_t)(v & 1u) * pairs + slots[wave][v >> 1]) * a.ff * 2 + c * 64u;
            }
            f32x4 acc[MB];
#pragma unroll
            for (int mb = 0; mb < MB; mb++) acc[mb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            u32x4 pf[G::NUW];
            moe_fetch<F>(rows, row_bytes, span0, n_spans, tail_len, pf);
            for (uint32_t span = span0; span < span1; span++) {
                moe_stash<F>(slice, pf);
                wave_sync();
                if (span + 1 < span1) moe_fetch<F>(rows, row_bytes, span + 1, n_spans, tail_len, pf);
                const uint32_t skew = G::SKEW ? (uint32_t)(uintptr_t)(rows + (uint64_t)r * row_bytes + (uint64_t)span * G::SPAN_BYTES) & 15u : 0u;
                moe_span<F, OUT, MB>(slice + r * G::ROW_STRIDE + skew, col, span, a.ff, acc);
                wave_sync();
            }
            // D[row = 4c + i][column = r]: value and rest are neighbouring lanes; the even one adds the token's share to its wave's y
#pragma unroll
            for (int mb = 0; mb < MB; mb++) {
                const uint32_t v = c0 + (uint32_t)(mb * 16) + r;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float rest = dpp_f<0xB1, 0xF>(acc[mb][i]);                     // the neighbour's sum
                    if constexpr (OUT == OUT_F16) rest *= 1.0f / 2048.0f;
                    if (v < n_cols && (v & 1u) == 0) part[slots[wave][v >> 1] / a.top_k * 16u + 4u * c + (uint32_t)i] += shares[wave][v >> 1] * (acc[mb][i] + rest);
                }
            }
        }
        wave_sync();
        item = stop;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.tokens * 16u; i += MOE_DOWN_WAVES * 64) {
        const float* all = reinterpret_cast<const float*>(dyn);
        float v = all[i];
        for (uint32_t w = 1; w < MOE_DOWN_WAVES; w++) v += all[(uint64_t)w * a.tokens * 16u + i];
        const uint64_t at = (uint64_t)(i >> 4) * a.dim + row0 + (i & 15u);
        if constexpr (OUT == OUT_F16) reinterpret_cast<_Float16*>(a.y)[at] = (_Float16)v;
        else reinterpret_cast<uint16_t*>(a.y)[at] = (uint16_t)(pack_bf16(v, 0.0f) & 0xFFFFu);
    }
}

}  // namespace ggq
