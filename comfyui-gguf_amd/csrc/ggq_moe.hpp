// ggq_moe.hpp -- gfx950 device code: a mixture-of-experts layer for a few tokens, straight from packed GGUF expert weights.
//
// Mathematics, per token x:  l = Wr x;  p = softmax(l);  the top_k largest p (equal ones to the lower index), divided by their sum if asked;
//     y = sum_s p_s Wd[e_s] (act(Wg[e_s] x) * (Wu[e_s] x)).
//
// Kernels: the router (moe_route, or moe_scores and moe_pick), the gate and up projections with the activation (moe_up), the down projection with the weighted sum
// over experts (moe_down), and where the output has too few rows for the chip, a sum of its parts (moe_combine).  What bounds them is reading the
// packed bytes of the chosen experts, each ONCE for all tokens that chose it -- and, as closely, unpacking them (1100 cycles of vector instructions per 16
// rows x 256 columns of Q4_K for bf16: at the full rate that is 18 us where reading takes 19, for two experts of 2 x 10240 x 4096):
//   * moe_up: a workgroup owns some tiles of 16 rows of Wg and Wu of the chosen experts; half of its waves contract the gate rows, half the up rows, each a part
//     of k; the tokens of the expert are the columns of v_mfma_f32_16x16x32 (A = 16 rows of decoded weights).
//   * moe_down: a workgroup owns 16 rows of the output for ALL tokens and walks every chosen expert, so the sum over a token's experts needs no atomics; its
//     waves take equal, contiguous parts of the (expert, piece of k) list.
//   * the list of chosen experts and the tokens of each are found by every workgroup itself from the ids (at most 64 x 16 of them).
//   * a wave requests the columns (x, hidden) of this span, then the weights of a later one, then waits for all but those.  Loads return in order: columns
//     requested behind weights would wait for those weights.
// A weight is the reference's value bit for bit (ggq_device.hpp: same decode, same fp16 operations, then the rounding to the activations' type).
// The hidden vector act(g) * u is kept in two parts of the activations' type -- its rounded value and the rounded rest -- which ride as two columns of
// the down product: about 16 (bf16) or 22 (fp16) bits, for no more weight traffic.  The fp16 rest is kept times 2^11, out of the subnormals; a value that fp16
// does not hold is kept as a NaN that says what it is, and the columns that have one are added up again in fp32 (moe_big).
// Measured, bf16: one token, two of 8 x 10240 x 4096 (Q4_K, down Q6_K): moe_up 36 us (2.6 TB/s of packed bytes), moe_down 28 (2.5); 33 tokens, fp16, two of 4 x 6848 x
// 2432 (Q8_0, down Q5_0): 62 and 58 us.
// Sums: fp32 in the MFMA's order, k-parts in wave order, experts in ascending order within a wave: the result does not depend on timing.
#pragma once

#include "ggq_mfma16.hpp"
#include "ggq_rows.hpp"

namespace ggq {

constexpr int MOE_MAX_TOKENS = 64, MOE_MAX_TOPK = 16, MOE_MAX_EXPERTS = 512;
constexpr int MOE_WORDS = MOE_MAX_EXPERTS / 32;

// ---- the router

// The score of one expert, by one wave, in every lane: pieces of 4 x 512 elements on their way at once.  Products and sums in fp64: which of two close scores is
// larger decides which experts run.  A product of 24 x 11 bits is exact there, and that of two bf16 values may leave fp32's range.  RT: the router's type, fp32 in GGUF
// files.  What bounds it is the latency of the loads: one token, 8 experts x 4096 in bf16, the router of a layer in turn with its experts takes 4.5 us, and 10.6 where the
// compiler lets a piece's loads wait for the sums of the one before.
template <int OUT, int RT> GGQ_DEV double moe_score(const uint8_t* x, const uint8_t* w, uint32_t dim)
{
    constexpr uint32_t U = 4;
    double acc = 0.0;
    for (uint32_t i0 = (threadIdx.x & 63u) * 8u; i0 < dim; i0 += 512u * U) {
        RowRaw<OUT> xs[U];
        RowRaw<RT> ws[U];
#pragma unroll
        for (uint32_t p = 0; p < U; p++) {
            const uint64_t i = i0 + 512u * p < dim ? i0 + 512u * p : 0u;       // past the end: the row's start, not added
            xs[p] = row_raw<OUT, false>(x + i * 2u, 0, 8);
            ws[p] = row_raw<RT, false>(w + i * (RT == OUT_F32 ? 4u : 2u), 0, 8);
        }
        __builtin_amdgcn_sched_barrier(0);                                     // all of them before the first is used
#pragma unroll
        for (uint32_t p = 0; p < U; p++) {
            float u[8], v[8];
            double d[8];
            row_unpack<OUT>(xs[p], u);
            row_unpack<RT>(ws[p], v);
#pragma unroll
            for (int k = 0; k < 8; k++) d[k] = (double)u[k] * (double)v[k];
            const double sum = ((d[0] + d[1]) + (d[2] + d[3])) + ((d[4] + d[5]) + (d[6] + d[7]));
            acc += i0 + 512u * p < dim ? sum : 0.0;
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
    return acc;
}

// The top_k experts of one token and their weights, from the scores in LDS; by the whole workgroup, which has a thread for every expert.  rank_[e] = how many
// experts come before e.  A NaN comes last and makes all of the token's weights NaN, chosen or not: it is in the softmax's sum (rank_[experts]: whether there
// is one).  The comparisons of an expert are split over the threads there are.  Weights are fp32: exp of a difference of fp64 scores, v_exp_f32 and v_rcp_f32 within 2^-23.
GGQ_DEV void moe_choose(const double* score, uint32_t* rank_, double* chosen, uint32_t experts, uint32_t top_k, int renormalize, int32_t* ids, float* weights)
{
    const uint32_t padded = (experts + 63u) & ~63u, parts = blockDim.x / padded, t = threadIdx.x % padded, part = threadIdx.x / padded;
    for (uint32_t i = threadIdx.x; i <= experts; i += blockDim.x) rank_[i] = 0;
    __syncthreads();
    if (t < experts && part < parts) {
        const double own = score[t];
        uint32_t before = 0;
#pragma unroll 4
        for (uint32_t e = part; e < experts; e += parts) {
            const double o = score[e];
            before += (o > own || (o == own && e < t) || (own != own && (o == o || e < t))) ? 1u : 0u;
        }
        atomicAdd(&rank_[t], before);
        if (own != own) rank_[experts] = 1;                                 // whoever writes, the same value
    }
    __syncthreads();
    const uint32_t rank = threadIdx.x < experts ? rank_[threadIdx.x] : ~0u;
    if (rank < top_k) {
        chosen[rank] = score[threadIdx.x];
        ids[rank] = (int32_t)threadIdx.x;
    }
    __syncthreads();
    if (rank < top_k) {
        const double top = chosen[0];
        float sum = rank_[experts] ? __builtin_nanf("") : 0.0f;
        if (renormalize) {
#pragma unroll
            for (uint32_t s = 0; s < MOE_MAX_TOPK; s++) sum += s < top_k ? __expf((float)(chosen[s] - top)) : 0.0f;
        } else {
#pragma unroll 8
            for (uint32_t e = 0; e < experts; e++) sum += __expf((float)(score[e] - top));
        }
        weights[rank] = __expf((float)(score[threadIdx.x] - top)) * __builtin_amdgcn_rcpf(sum);
    }
}

// up to 16 experts: one workgroup per token, one wave per expert
constexpr int MOE_ROUTE_WAVES = 16;
template <int OUT, int RT>
__global__ __launch_bounds__(MOE_ROUTE_WAVES * 64) void moe_route(const uint8_t* __restrict__ x, const uint8_t* __restrict__ router, uint32_t dim, uint32_t experts,
                                                                 uint32_t top_k, int renormalize, int32_t* __restrict__ ids, float* __restrict__ weights)
{
    __shared__ double score[MOE_ROUTE_WAVES];
    __shared__ uint32_t rank[MOE_ROUTE_WAVES + 1];
    __shared__ double chosen[MOE_MAX_TOPK];
    const uint32_t wave = threadIdx.x >> 6;
    if (wave < experts) {
        const double v = moe_score<OUT, RT>(x + (uint64_t)blockIdx.x * dim * 2, router + (uint64_t)wave * dim * (RT == OUT_F32 ? 4 : 2), dim);
        if ((threadIdx.x & 63u) == 0) score[wave] = v;
    }
    __syncthreads();
    moe_choose(score, rank, chosen, experts, top_k, renormalize, ids + (uint64_t)blockIdx.x * top_k, weights + (uint64_t)blockIdx.x * top_k);
}

// more experts: a wave per (expert, token) for the scores, then a workgroup per token for the choice.  (64 experts x 2048, 7 tokens: 18 us with one workgroup per
// token for both, most of it one CU's latency.)
template <int OUT, int RT>
__global__ __launch_bounds__(256) void moe_scores(const uint8_t* __restrict__ x, const uint8_t* __restrict__ router, uint32_t dim, uint32_t experts, double* __restrict__ scores)
{
    const uint32_t e = blockIdx.x * 4u + (threadIdx.x >> 6), t = blockIdx.y;
    if (e >= experts) return;
    const double v = moe_score<OUT, RT>(x + (uint64_t)t * dim * 2, router + (uint64_t)e * dim * (RT == OUT_F32 ? 4 : 2), dim);
    if ((threadIdx.x & 63u) == 0) scores[(uint64_t)t * experts + e] = v;
}

__global__ __launch_bounds__(MOE_MAX_EXPERTS) void moe_pick(const double* __restrict__ scores, uint32_t experts, uint32_t top_k, int renormalize, int32_t* __restrict__ ids,
                                                           float* __restrict__ weights)
{
    __shared__ double score[MOE_MAX_EXPERTS];
    __shared__ uint32_t rank[MOE_MAX_EXPERTS + 1];
    __shared__ double chosen[MOE_MAX_TOPK];
    if (threadIdx.x < experts) score[threadIdx.x] = scores[(uint64_t)blockIdx.x * experts + threadIdx.x];
    __syncthreads();
    moe_choose(score, rank, chosen, experts, top_k, renormalize, ids + (uint64_t)blockIdx.x * top_k, weights + (uint64_t)blockIdx.x * top_k);
}

// ---- which experts were chosen, and by whom

struct MoeTable {
    uint32_t words[MOE_WORDS];                       // bit e: some token chose expert e
    int32_t ids[MOE_MAX_TOKENS * MOE_MAX_TOPK];
    uint16_t list[MOE_MAX_EXPERTS];                  // the chosen experts, ascending
    uint32_t n;                                      // how many
};

// Called by the whole workgroup; ends with a barrier.
GGQ_DEV void moe_table(MoeTable& s, const int32_t* __restrict__ ids, uint32_t pairs, uint32_t experts)
{
    if (threadIdx.x < MOE_WORDS) s.words[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < pairs; p += blockDim.x) {
        const uint32_t e = (uint32_t)ids[p];
        s.ids[p] = (int32_t)e;
        if (e < experts) atomicOr(&s.words[e >> 5], 1u << (e & 31u));
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        uint32_t b = threadIdx.x < MOE_WORDS ? s.words[threadIdx.x] : 0u;
        uint32_t upto = (uint32_t)__builtin_popcount(b);
        const uint32_t own = upto;
#pragma unroll
        for (int off = 1; off < MOE_WORDS; off <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)upto, off, 64);
            if (threadIdx.x >= (uint32_t)off) upto += o;
        }
        if (threadIdx.x == MOE_WORDS - 1) s.n = upto;
        for (uint32_t at = upto - own; b != 0; b &= b - 1u) s.list[at++] = (uint16_t)(32u * threadIdx.x + (uint32_t)__builtin_ctz(b));
    }
    __syncthreads();
}

// The tokens that chose `expert`: lane t looks at token t.  `slot`: its first place in ids, `weight`: the sum over its places (the same expert twice
// counts twice; weights_ may be null).  Returns the mask of tokens.
GGQ_DEV uint64_t moe_tokens(const MoeTable& s, const float* weights, uint32_t tokens, uint32_t top_k, int expert, uint32_t& slot, float& weight)
{
    const uint32_t t = threadIdx.x & 63u;
    bool has = false;
    slot = 0;
    weight = 0.0f;
    if (t < tokens)
        for (uint32_t k = top_k; k-- > 0;)
            if (s.ids[t * top_k + k] == expert) {
                has = true;
                slot = t * top_k + k;
                if (weights != nullptr) weight += weights[t * top_k + k];
            }
    return __ballot(has);
}

// a barrier for LDS only: weights that are on their way to registers stay on their way
GGQ_DEV void moe_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// v_exp_f32 and v_rcp_f32 are within 2^-23 of their value, the exponent's argument within |g| 2^-24: as much as the sums that g comes from.
GGQ_DEV float moe_act(float g, int act)
{
    if (act == 0) return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g));                                    // silu
    const float u = 0.7978845608028654f * (g + 0.044715f * g * g * g);                                     // gelu, tanh form: g / (1 + exp(-2u))
    return g * __builtin_amdgcn_rcpf(1.0f + __expf(-2.0f * u));
}

// A wave's packed bytes go from memory straight into its own LDS slots (LDS-DMA), one 256-element span of 16 rows per slot: row r at r * ROW_STRIDE, an
// odd number of 16-byte units, from the aligned address below the row's span on (Mf16Geom).  Two slots: the next span is on its way while one is decoded, at no cost
// in registers.  (A third slot does not put a second span on its way: loads return in order, and the wait for a span's columns, which are requested after the span
// behind it, is a wait for that span.  Measured: one token, two of 8 x 10240 x 4096 in Q4_K / Q6_K, bf16, 60.2 us with two slots, 60.7 with three; 7 tokens, eight of 64 x 1024 x 2048,
// 63.2 and 64.6; 33 tokens, two of 4 x 6848 x 2432 in Q8_0 / Q5_0, 128.3 and 127.3.)
constexpr uint32_t MOE_RING = 2;

template <class F> struct MoeGeom {
    using G = Mf16Geom<F>;
    static constexpr uint32_t PITCH_U = G::ROW_STRIDE / 16, UNITS = 16 * PITCH_U, LOADS = (UNITS + 63) / 64;       // units of a slot; DMA instructions
};

// byte offset of a row's span from the 16-byte boundary at or below the first row: 16 rows are within 32 bits of it
GGQ_DEV uint32_t moe_offset(gcptr rows, uint32_t row, uint32_t row_bytes, uint32_t span_at) { return ((uint32_t)(uintptr_t)rows & 15u) + row * row_bytes + span_at; }

// requests one span; at least one lane of every instruction loads where the span is whole (LOADS instructions), fewer for a short last one
template <class F> GGQ_DEV void moe_request(gcptr rows, uint32_t row_bytes, uint32_t span, uint32_t span_bytes, uint8_t* slot)
{
    using G = Mf16Geom<F>;
    using M = MoeGeom<F>;
    const uint32_t lane = threadIdx.x & 63u;
    const gcptr base = (gcptr)((uintptr_t)rows & ~(uintptr_t)15);
#pragma unroll
    for (uint32_t i = 0; i < M::LOADS; i++) {
        const uint32_t unit = lane + 64u * i, ur = unit / M::PITCH_U, uu = unit % M::PITCH_U;
        const uint32_t at = moe_offset(rows, ur, row_bytes, span * G::SPAN_BYTES), a = G::SKEW ? at & 15u : 0u;
        // loads start 16-byte aligned: what they read past the span lies in a unit that also holds bytes of the tensor
        if (ur < 16u && uu * 16u < a + span_bytes)
            __builtin_amdgcn_global_load_lds((const GGQ_GLOBAL void*)(base + (at - a + uu * 16u)), (__attribute__((address_space(3))) void*)(slot + 1024u * i), 16, 0, 0);
    }
}

// zeros behind a short last span: blocks that do not exist decode to weights of exactly 0
template <class F> GGQ_DEV void moe_cut(gcptr rows, uint32_t row_bytes, uint32_t span, uint32_t span_bytes, uint8_t* slot)
{
    using G = Mf16Geom<F>;
    using M = MoeGeom<F>;
    for (uint32_t unit = threadIdx.x & 63u; unit < M::UNITS; unit += 64u) {
        const uint32_t ur = unit / M::PITCH_U, uu = unit % M::PITCH_U;
        const uint32_t a = G::SKEW ? moe_offset(rows, ur, row_bytes, span * G::SPAN_BYTES) & 15u : 0u;
        const int32_t valid = (int32_t)(a + span_bytes) - (int32_t)(uu * 16u);
        if (valid >= 16) continue;
        u32x4* at = reinterpret_cast<u32x4*>(slot + unit * 16u);
        u32x4 d = *at;
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] &= valid >= 4 * i + 4 ? 0xFFFFFFFFu : (valid == 4 * i + 2 ? 0x0000FFFFu : 0u);
        *at = d;
    }
    wave_sync();
}

// at most `KEEP` of this wave's newest loads are still under way
template <int KEEP> GGQ_DEV void moe_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(KEEP) : "memory"); }

// half g of this lane's columns of one span: element 128 g + 32 c + 8 t ... + 7 of column (block mb, r) in x[mb][4 g + t].  Lanes without a column (null) load nothing and
// keep what they hold: a column of the product depends on that column alone.  (One token, 2 x 10240 x 4096: with every lane loading, the columns were 8 KiB
// per span against 2.3 of weights, and cost 8 of 38 us in the vector cache.)
template <class F, int MB>
GGQ_DEV void moe_half(const GGQ_GLOBAL uint8_t* const (&col)[MB], uint32_t span, uint32_t k_len, int g, u32x4 (&x)[MB][8])
{
    const int c = (int)(threadIdx.x & 63u) >> 4;
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        const GGQ_GLOBAL uint8_t* src = col[mb] + (uint64_t)span * (MF_SPAN * 2) + (uint32_t)(g * 256);
        if constexpr (F::BS == 32) {                                                                       // past the end of k: zeros
            if (span * (uint32_t)MF_SPAN + (uint32_t)(128 * g + 32 * c) >= k_len) src = (GGQ_GLOBAL const uint8_t*)MF16_ZEROS;
        }
        if (col[mb] != nullptr) {
#pragma unroll
            for (int t = 0; t < 4; t++) x[mb][4 * g + t] = *(GGQ_GLOBAL const u32x4*)(src + t * 16);
        }
    }
}

template <class F, int MB>
GGQ_DEV void moe_columns(const GGQ_GLOBAL uint8_t* const (&col)[MB], uint32_t span, uint32_t k_len, u32x4 (&x)[MB][8])
{
#pragma unroll
    for (int g = 0; g < 2; g++) moe_half<F, MB>(col, span, k_len, g, x);
}

// acc += 16 rows of weights, decoded from one span of packed bytes (`wspan`: this lane's row in LDS), times MB blocks of 16 columns.  after(g): half g of the columns
// has been multiplied
template <class F, int OUT, int MB, class After>
GGQ_DEV void moe_span(const uint8_t* wspan, const u32x4 (&x)[MB][8], f32x4 (&acc)[MB], After after)
{
    constexpr int CPB = F::BS / 8;
    const int c = (int)(threadIdx.x & 63u) >> 4;
#pragma unroll
    for (int g = 0; g < 2; g++) {
        if (g) __builtin_amdgcn_sched_barrier(0);                                                          // the second half's decode stays out of the first one's registers
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int j = 16 * g + 4 * c + t;
            const Fields f = F::template fields<true>(wspan + (j / CPB) * F::TS, j % CPB);
            uint32_t w[4];
            weights8<F, OUT>(f, w);
            const u32x4 wa{w[0], w[1], w[2], w[3]};
#pragma unroll
            for (int mb = 0; mb < MB; mb++) acc[mb] = mfma16<OUT>(wa, x[mb][4 * g + t], acc[mb]);
        }
        after(g);
    }
}

struct MoeArgs {
    const uint8_t* x;
    const int32_t* ids;
    const float* weights;
    const uint8_t *gate, *up, *down;
    uint8_t* y;
    uint8_t* hidden;                 // [2][tokens * top_k][ff] of the activations' type: the rounded value, then the rest
    float* part;                     // [parts][tokens][dim]: moe_down's parts of y (parts > 1)
    uint32_t tokens, top_k, experts, dim, ff;
    int act;
    uint32_t parts, spare;           // spare: blocks of 16 columns beyond the kernel's MB that the tokens could fill (their sums live in LDS)
};

constexpr int MOE_WAVES = 8;
// waves per SIMD that the registers are asked to leave room for: with one block of columns 4, two workgroups per CU
#define MOE_OCC(MB) __attribute__((amdgpu_waves_per_eu((MB) == 1 ? 4 : 2, 8)))

// Hidden values beyond fp16.  One of magnitude 65520 or more would round to infinity, and infinity and minus infinity as its two parts add up to NaN whatever the down
// projection makes of it.  Such a value h is kept as
//     first part   sign | 0x7E00 (a quiet NaN) | (exponent field of h - 142) << 2 | bits 21 and 22 of h        second part   bits 5 ... 20 of h
// of h in fp32, rounded to 18 bits behind its point (2^-19 of it).  The matrix product of its column is a NaN then, which moe_down finds when it adds the column
// up, at no cost to the others.  Infinities stay infinities, with a second part of 0; NaN is 0x7FFF.
constexpr uint32_t MOE_FP16_TOP = 0x477FF000u;                                 // 65520 in fp32
GGQ_DEV bool moe_is_big(float h) { return (__builtin_bit_cast(uint32_t, h) & 0x7FFFFFFFu) >= MOE_FP16_TOP; }
GGQ_DEV void moe_keep_big(float h, uint32_t& hi, uint32_t& lo)
{
    const uint32_t bits = __builtin_bit_cast(uint32_t, h), sign = (bits >> 16) & 0x8000u;
    uint32_t b = bits & 0x7FFFFFFFu;
    if (b >= 0x7F800000u) {
        hi = b > 0x7F800000u ? 0x7FFFu : sign | 0x7C00u;
        lo = 0;
        return;
    }
    b += 15u + ((b >> 5) & 1u);                                                // half to even
    hi = sign | 0x7E00u | ((b >> 23) - 142u) << 2 | ((b >> 21) & 3u);
    lo = (b >> 5) & 0xFFFFu;
}
GGQ_DEV float moe_hidden_f16(uint32_t hi, uint32_t lo)                         // the value of two parts
{
    if ((hi & 0x7E00u) != 0x7E00u) return (float)h_of(hi) + (float)h_of(lo) * (1.0f / 2048.0f);
    const uint32_t exponent = (hi >> 2) & 127u;
    return exponent == 127u ? __builtin_nanf("") : bits_f32((hi & 0x8000u) << 16 | (exponent + 142u) << 23 | (hi & 3u) << 21 | lo << 5);
}

// One hidden vector times 16 rows of packed weights, spans [s0, s1), in fp32: lane r, r + 16, r + 32, r + 48 share row r; the sum comes back in all of them.  For the few
// columns that need it: straight from memory, element by element.  (33 tokens, two of four experts of 2 x 6848 x 2432 in fp16: the layer 123 us, 261 with such values in every token.)
// `lane` is hidden from the compiler, so that nothing of this is computed ahead in registers of the loop that it stands in.
template <class F>
GGQ_DEV float moe_big(gcptr rows, uint64_t row_bytes, const GGQ_GLOBAL uint8_t* value, const GGQ_GLOBAL uint8_t* rest, uint32_t s0, uint32_t s1, uint32_t k_len, uint32_t lane)
{
    constexpr uint32_t CPB = F::BS / 8;
    const uint32_t r = lane & 15u, c = lane >> 4;
    const uint8_t* row = (const uint8_t*)(rows + r * row_bytes);
    float sum = 0.0f;
#pragma unroll 1
    for (uint32_t j = s0 * 32u + c; j < s1 * 32u && j * 8u < k_len; j += 4u) {                             // chunks of 8 elements
        const Fields f = F::template fields<false>(row + (uint64_t)(j / CPB) * F::TS, (int)(j % CPB));
        uint32_t w[4];
        weights8<F, OUT_F16>(f, w);
        const u32x4 hi = *(GGQ_GLOBAL const u32x4*)(value + (uint64_t)j * 16u), lo = *(GGQ_GLOBAL const u32x4*)(rest + (uint64_t)j * 16u);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const h2 v = as_h2(w[i]);
            sum += (float)v.x * moe_hidden_f16(hi[i] & 0xFFFFu, lo[i] & 0xFFFFu);
            sum += (float)v.y * moe_hidden_f16(hi[i] >> 16, lo[i] >> 16);
        }
    }
    sum += __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute((int)((lane ^ 16u) << 2), __builtin_bit_cast(int, sum)));
    return sum + __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute((int)((lane ^ 32u) << 2), __builtin_bit_cast(int, sum)));
}

// this wave's list of the columns' places: `per` columns for each token of the expert; returns how many columns
GGQ_DEV uint32_t moe_list(const MoeTable& s, const float* weights, const MoeArgs& a, int expert, uint32_t* slots, float* shares)
{
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t slot;
    float weight;
    const uint64_t mask = moe_tokens(s, weights, a.tokens, a.top_k, expert, slot, weight);
    if ((mask >> lane) & 1u) {
        const uint32_t at = (uint32_t)__builtin_popcountll(mask & ((1ull << lane) - 1ull));
        slots[at] = slot;
        if (shares != nullptr) shares[at] = weight;
    }
    wave_sync();
    return (uint32_t)__builtin_popcountll(mask);
}

// hidden = act(Wg x) * (Wu x), 16 hidden rows of a chosen expert at a time.  The (expert, tile of 16 rows) list is dealt out evenly: the first workgroups take
// one tile more.  With one block of columns, waves 0, 2, 4, 6 contract gate rows, waves 1, 3, 5, 7 up rows, every fourth span each.  With more, the columns are several
// times the weights' bytes, and a wave takes an equal, contiguous part of the list (span 0 of gate, span 0 of up, span 1 of gate, ...), with sums for both and the columns of
// a span loaded once for the two, ahead: as soon as the last span's have been used.  (33 tokens, two of four experts of 2 x 6848 x 2432 in Q8_0: 71 us as with one block, 76 with
// the columns shared but not ahead, 64 so; 64 tokens, two of eight of 2 x 10240 x 4096 in Q4_K: the layer 532 -> 415.)
template <class F, int OUT, int MB>
__global__ __launch_bounds__(MOE_WAVES * 64) MOE_OCC(MB) void moe_up(const MoeArgs a)
{
    using G = Mf16Geom<F>;
    // per wave: the sums of columns beyond MB blocks ([spare][64] f32x4), then, for all waves, their slots
    extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
    __shared__ MoeTable table;
    __shared__ uint32_t slots_[MOE_WAVES][MOE_MAX_TOKENS];                         // per column: where its hidden row goes (= token * top_k + place)
    constexpr int TURNS = MB == 1 ? 2 : 1;                                         // two tiles' partial sums: the next tile's are written while one is added up
    constexpr int MATS = MB == 1 ? 1 : 2;                                          // matrices that a wave has sums of
    __shared__ f32x4 red[TURNS][MOE_WAVES][MATS][MB][64];
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, c = lane >> 4;
    const uint32_t pairs = a.tokens * a.top_k;
    moe_table(table, a.ids, pairs, a.experts);

    const uint32_t tiles = a.ff / 16u, total = table.n * tiles, each = total / gridDim.x, more = total - each * gridDim.x;
    const uint32_t t0 = blockIdx.x * each + (blockIdx.x < more ? blockIdx.x : more), t1 = t0 + each + (blockIdx.x < more ? 1u : 0u);
    const uint64_t row_bytes = (uint64_t)(a.dim / F::BS) * F::TS;
    const uint32_t n_spans = (a.dim + MF_SPAN - 1) / MF_SPAN, tail_len = a.dim - (n_spans - 1) * (uint32_t)MF_SPAN;
    // this wave's units of a tile: [u0, u1) in steps of `by`, unit u = span u / MATS of matrix u % 2 (or of the wave's own)
    const uint32_t u0 = MATS == 1 ? wave >> 1 : 2u * n_spans * wave / MOE_WAVES, u1 = MATS == 1 ? n_spans : 2u * n_spans * (wave + 1u) / MOE_WAVES, by = MATS == 1 ? MOE_WAVES / 2 : 1;
    auto is_up = [&](uint32_t u) { return MATS == 1 ? wave & 1u : u & 1u; };
    uint8_t* ring = dyn + MOE_WAVES * MATS * a.spare * 1024u + wave * MOE_RING * (uint32_t)G::SLICE;
    uint32_t* slots = slots_[wave];
    f32x4* spare = reinterpret_cast<f32x4*>(dyn) + (uint64_t)wave * MATS * a.spare * 64u;
    uint32_t turn = 0;
    for (uint32_t t = t0; t < t1;) {                                               // one expert at a time: tiles [t, stop) of the list
        const uint32_t nth = t / tiles, stop = (nth + 1) * tiles < t1 ? (nth + 1) * tiles : t1;
        const uint32_t n_cols = moe_list(table, nullptr, a, table.list[nth], slots, nullptr);
        const uint64_t base = (uint64_t)table.list[nth] * a.ff * row_bytes;
        auto weights_at = [&](uint32_t i, uint32_t u) { return (gcptr)(is_up(u) ? a.up : a.gate) + base + (uint64_t)(i - nth * tiles) * 16u * row_bytes; };      // tile i of the list
        auto column = [&](uint32_t v) { return v < n_cols ? (GGQ_GLOBAL const uint8_t*)a.x + (uint64_t)(slots[v] / a.top_k) * a.dim * 2 + c * 64u : nullptr; };
        const GGQ_GLOBAL uint8_t* col[MB];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) col[mb] = column((uint32_t)(mb * 16) + r);
        const uint32_t blocks = (n_cols + 15u) / 16u;
        u32x4 both[MATS == 1 ? 1 : MB][8];                                         // the columns of a span, for its two units
        if constexpr (MATS == 2) {
            if (u0 < u1) moe_columns<F, MB>(col, u0 / MATS, a.dim, both);
        }

        uint32_t ft = t, fu = u0, in = 0, out = 0;                                 // the next unit to request; ring slots
        auto request = [&]() {                                                     // -> 2: a whole span, 1: a short one, 0: nothing left
            if (ft >= stop || fu >= u1) return 0;
            const uint32_t fs = fu / MATS;
            const bool tail = F::BS == 32 && fs + 1 == n_spans && tail_len != (uint32_t)MF_SPAN;
            moe_request<F>(weights_at(ft, fu), (uint32_t)row_bytes, fs, (tail ? tail_len : (uint32_t)MF_SPAN) / (uint32_t)F::BS * (uint32_t)F::TS, ring + in * G::SLICE);
            in ^= 1u;
            fu += by;
            if (fu >= u1) { fu = u0; ft++; }
            return tail ? 1 : 2;
        };
        request();
        f32x4 acc[MATS][MB];                                                       // acc[0]: of the matrix of this unit, acc[1] of the other
        auto clear = [&]() {
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int i = 0; i < MATS; i++) acc[i][mb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t q = 0; q < (blocks > (uint32_t)MB ? MATS * a.spare : 0u); q++) spare[q * 64u + lane] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        };
        uint32_t tile = t - nth * tiles, unit = u0;
        const uint32_t tile_end = stop - nth * tiles;
        auto one = [&]() {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                     // the slot that is filled next has been read
            const uint32_t span = unit / MATS, mat = is_up(unit);
            u32x4 own[MB][8];
            auto& x = [&]() -> u32x4 (&)[MB][8] { if constexpr (MATS == 1) return own; else return both; }();
            if constexpr (MATS == 1) moe_columns<F, MB>(col, span, a.dim, x);
            asm volatile("" ::: "memory");
            if (request() == 2) moe_wait<(int)MoeGeom<F>::LOADS>();                // all but the span just requested
            else moe_wait<0>();
            uint8_t* slot = ring + out * G::SLICE;
            out ^= 1u;
            const gcptr rows = weights_at(nth * tiles + tile, unit);
            if (F::BS == 32 && span + 1 == n_spans && tail_len != (uint32_t)MF_SPAN) moe_cut<F>(rows, (uint32_t)row_bytes, span, tail_len / (uint32_t)F::BS * (uint32_t)F::TS, slot);
            const uint32_t skew = G::SKEW ? moe_offset(rows, r, (uint32_t)row_bytes, span * G::SPAN_BYTES) & 15u : 0u;
            // MATS 2: the columns of the next span, if the next unit has another, are on their way as soon as this one's have been used
            const uint32_t next = unit + by < u1 ? unit + by : u0;
            const bool other = MATS == 2 && (next > unit ? (next & 1u) == 0 : tile + 1 < tile_end);
            moe_span<F, OUT, MB>(slot + r * G::ROW_STRIDE + skew, x, acc[0], [&](int g) {
                if constexpr (MATS == 2) {
                    if (other) moe_half<F, MB>(col, next / MATS, a.dim, g, both);
                }
            });
            for (uint32_t q = MB; q < blocks; q++) {                               // more tokens on one expert than the kernel was picked for
                const GGQ_GLOBAL uint8_t* const late[1] = {column(q * 16u + r)};
                u32x4 lx[1][8];
                f32x4& kept = spare[((MATS == 1 ? 0u : mat * a.spare) + q - MB) * 64u + lane];
                f32x4 sum[1] = {kept};
                moe_columns<F, 1>(late, span, a.dim, lx);
                moe_span<F, OUT, 1>(slot + r * G::ROW_STRIDE + skew, lx, sum, [](int) {});
                kept = sum[0];
            }
            wave_sync();
            if constexpr (MATS == 2) {                                             // units take turns between the matrices
#pragma unroll
                for (int mb = 0; mb < MB; mb++) {
                    const f32x4 o = acc[0][mb];
                    acc[0][mb] = acc[1][mb];
                    acc[1][mb] = o;
                }
            }
            unit += by;
        };
        // the sums of a tile over the waves, the activation, the two parts of the hidden value; the waves take turns at it
        auto finish = [&]() {
            if (TURNS == 1) moe_barrier();                                         // the last tile's sums have been added up: by waves that were a tile's time behind at most
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int i = 0; i < MATS; i++) red[turn][wave][MATS == 1 ? 0u : (unit + (uint32_t)i) & 1u][mb][lane] = acc[i][mb];
            moe_barrier();
            for (uint32_t q = (wave - tile * MB) % MOE_WAVES; q < blocks; q += MOE_WAVES) {
                auto sum = [&](uint32_t w, uint32_t i) {
                    return q < (uint32_t)MB ? red[turn][w][i][q][lane] : reinterpret_cast<const f32x4*>(dyn)[(uint64_t)((w * MATS + i) * a.spare + q - MB) * 64u + lane];
                };
                constexpr uint32_t EACH = 3 - MATS, UP = MATS == 1 ? 0 : 1;
                f32x4 g = sum(0, 0), u = sum(EACH - 1, UP);
                for (uint32_t w = EACH; w < MOE_WAVES; w += EACH) { g += sum(w, 0); u += sum(w + EACH - 1, UP); }
                const uint32_t v = q * 16u + r;                                    // D[row = 4c + i][column = r]
                if (v < n_cols) {
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        float h0 = moe_act(g[2 * p], a.act) * u[2 * p], h1 = moe_act(g[2 * p + 1], a.act) * u[2 * p + 1];
                        asm volatile("" : "+v"(h0), "+v"(h1));                     // the product rounded to fp32 (no v_fma_mix with the conversion): both parts see it
                        if constexpr (OUT == OUT_F16) {
                            const h2 n{(_Float16)h0, (_Float16)h1};
                            hi[p] = as_u32(n);
                            lo[p] = as_u32(h2{(_Float16)__builtin_ldexpf(h0 - (float)n.x, 11), (_Float16)__builtin_ldexpf(h1 - (float)n.y, 11)});
                            if (moe_is_big(h0) || moe_is_big(h1)) {
                                uint32_t top, rest;
                                if (moe_is_big(h0)) {
                                    moe_keep_big(h0, top, rest);
                                    hi[p] = (hi[p] & 0xFFFF0000u) | top;
                                    lo[p] = (lo[p] & 0xFFFF0000u) | rest;
                                }
                                if (moe_is_big(h1)) {
                                    moe_keep_big(h1, top, rest);
                                    hi[p] = (hi[p] & 0xFFFFu) | top << 16;
                                    lo[p] = (lo[p] & 0xFFFFu) | rest << 16;
                                }
                            }
                        } else {
                            hi[p] = pack_bf16(h0, h1);
                            lo[p] = pack_bf16(h0 - bits_f32(hi[p] << 16), h1 - bits_f32(hi[p] & 0xFFFF0000u));
                        }
                    }
                    uint8_t* dst = a.hidden + ((uint64_t)slots[v] * a.ff + tile * 16u + 4u * c) * 2;
                    *reinterpret_cast<u32x2*>(dst) = u32x2{hi[0], hi[1]};
                    *reinterpret_cast<u32x2*>(dst + (uint64_t)pairs * a.ff * 2) = u32x2{lo[0], lo[1]};
                }
            }
            if (blocks > (uint32_t)MB) moe_barrier();                              // the same sums' place is written next
            else if (TURNS == 2) turn ^= 1u;
            tile++;
            unit = u0;
            clear();
        };
        clear();
        while (tile < tile_end) {
            if (unit < u1) one();
            if (unit >= u1) finish();
        }
        t = stop;
    }
}

// 16 rows of y for every token, W waves; of gridDim.y = `parts` workgroups each takes a part of the (expert, span) list, and each of its waves an equal part of
// that, one wave after the other.  A wave's columns are (token, part of the hidden vector): column 2 i the value, 2 i + 1 the rest of token i of the expert.
template <class F, int OUT, int MB, int W>
__global__ __launch_bounds__(W * 64) MOE_OCC(MB) void moe_down(const MoeArgs a)
{
    using G = Mf16Geom<F>;
    // y of each wave ([wave][token][16] floats), sums of columns beyond MB blocks ([wave][spare][64] f32x4), the slots
    extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
    __shared__ MoeTable table;
    __shared__ float shares_all[MOE_MAX_TOKENS * MOE_MAX_TOPK];
    __shared__ uint32_t slots_[W][MOE_MAX_TOKENS];
    __shared__ float shares_[W][MOE_MAX_TOKENS];
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, c = lane >> 4;
    const uint32_t pairs = a.tokens * a.top_k;
    float* part = reinterpret_cast<float*>(dyn) + (uint64_t)wave * a.tokens * 16u;
    f32x4* spare = reinterpret_cast<f32x4*>(dyn + (uint64_t)W * a.tokens * 64u) + (uint64_t)wave * a.spare * 64u;
    for (uint32_t i = lane; i < a.tokens * 16u; i += 64u) part[i] = 0.0f;
    for (uint32_t p = threadIdx.x; p < pairs; p += W * 64) shares_all[p] = a.weights[p];
    moe_table(table, a.ids, pairs, a.experts);

    const uint32_t row0 = blockIdx.x * 16u;
    const uint64_t row_bytes = (uint64_t)(a.ff / F::BS) * F::TS, expert_bytes = (uint64_t)a.dim * row_bytes;
    const uint32_t n_spans = (a.ff + MF_SPAN - 1) / MF_SPAN, tail_len = a.ff - (n_spans - 1) * (uint32_t)MF_SPAN;
    const gcptr base = (gcptr)a.down + (uint64_t)row0 * row_bytes;
    const uint64_t items = (uint64_t)table.n * n_spans, share = blockIdx.y * W + wave, all = (uint64_t)a.parts * W;
    const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane((int)(items * share / all)), last = (uint32_t)__builtin_amdgcn_readfirstlane((int)(items * (share + 1) / all));
    uint8_t* ring = dyn + W * (a.tokens * 64u + a.spare * 1024u) + wave * MOE_RING * (uint32_t)G::SLICE;
    uint32_t* slots = slots_[wave];
    float* shares = shares_[wave];

    uint32_t fi = first, fn = first / n_spans, fs = first % n_spans, in = 0, out = 0;      // the next span to request, also of the next expert; ring slots
    auto request = [&]() {                                                         // -> 2: a whole span, 1: a short one, 0: nothing left
        if (fi >= last) return 0;
        const bool tail = F::BS == 32 && fs + 1 == n_spans && tail_len != (uint32_t)MF_SPAN;
        moe_request<F>(base + (uint64_t)table.list[fn] * expert_bytes, (uint32_t)row_bytes, fs, (tail ? tail_len : (uint32_t)MF_SPAN) / (uint32_t)F::BS * (uint32_t)F::TS, ring + in * G::SLICE);
        in ^= 1u;
        fi++;
        if (++fs == n_spans) { fs = 0; fn++; }
        return tail ? 1 : 2;
    };
    request();

    uint32_t item = first, nth = first / n_spans, span = first % n_spans, from = 0, n_cols = 0, blocks = 0;
    gcptr rows = base;
    const GGQ_GLOBAL uint8_t* col[MB];
    f32x4 acc[MB];
    auto column = [&](uint32_t v) {
        return v < n_cols ? (GGQ_GLOBAL const uint8_t*)a.hidden + ((uint64_t)(v & 1u) * pairs + slots[v >> 1]) * a.ff * 2 + c * 64u : nullptr;
    };
    auto start = [&]() {                                                           // the columns of the next expert
        n_cols = 2u * moe_list(table, shares_all, a, table.list[nth], slots, shares);
        blocks = (n_cols + 15u) / 16u;
        from = span;
        rows = base + (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)table.list[nth]) * expert_bytes;
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            col[mb] = column((uint32_t)(mb * 16) + r);
            acc[mb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (uint32_t q = MB; q < blocks; q++) spare[(q - MB) * 64u + lane] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    auto one = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                         // the slot that is filled next has been read
        u32x4 x[MB][8];
        moe_columns<F, MB>(col, span, a.ff, x);
        asm volatile("" ::: "memory");
        if (request() == 2) moe_wait<(int)MoeGeom<F>::LOADS>();                    // all but the span just requested
        else moe_wait<0>();
        uint8_t* slot = ring + out * G::SLICE;
        out ^= 1u;
        if (F::BS == 32 && span + 1 == n_spans && tail_len != (uint32_t)MF_SPAN) moe_cut<F>(rows, (uint32_t)row_bytes, span, tail_len / (uint32_t)F::BS * (uint32_t)F::TS, slot);
        const uint32_t skew = G::SKEW ? moe_offset(rows, r, (uint32_t)row_bytes, span * G::SPAN_BYTES) & 15u : 0u;
        moe_span<F, OUT, MB>(slot + r * G::ROW_STRIDE + skew, x, acc, [](int) {});
        for (uint32_t q = MB; q < blocks; q++) {                                   // more tokens on one expert than the kernel was picked for
            const GGQ_GLOBAL uint8_t* const late[1] = {column(q * 16u + r)};
            u32x4 lx[1][8];
            f32x4 sum[1] = {spare[(q - MB) * 64u + lane]};
            moe_columns<F, 1>(late, span, a.ff, lx);
            moe_span<F, OUT, 1>(slot + r * G::ROW_STRIDE + skew, lx, sum, [](int) {});
            spare[(q - MB) * 64u + lane] = sum[0];
        }
        wave_sync();
        item++;
        span++;
    };
    // D[row = 4c + i][column = r]: value and rest are neighbouring lanes; the even one adds the token's share to its wave's y
    // (anew: bit i: token i of the expert is to be added up anew, from its hidden values)
    auto add = [&](uint32_t q, f32x4 sum, uint64_t& anew) {
        const uint32_t v = q * 16u + r;
        bool fine = v < n_cols && (v & 1u) == 0;
        if constexpr (OUT == OUT_F16) {
            const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            const uint64_t lanes = __ballot(v < n_cols && all != all);
            if (lanes != 0) {
                uint32_t bad = (uint32_t)lanes | (uint32_t)(lanes >> 32);
                bad |= bad >> 16;
                bad = (bad | bad >> 1) & 0x5555u;                                  // column 2 i, its own or its rest's
                fine = fine && !((bad >> r) & 1u);
                for (; bad != 0; bad &= bad - 1u) anew |= 1ull << (q * 8u + (uint32_t)__builtin_ctz(bad) / 2u);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float rest = dpp_f<0xB1, 0xF>(sum[i]);                                 // the neighbour's sum
            if constexpr (OUT == OUT_F16) rest *= 1.0f / 2048.0f;
            if (fine) part[slots[v >> 1] / a.top_k * 16u + 4u * c + (uint32_t)i] += shares[v >> 1] * (sum[i] + rest);
        }
    };
    auto finish = [&]() {
        uint64_t anew = 0;
#pragma unroll
        for (int mb = 0; mb < MB; mb++) add((uint32_t)mb, acc[mb], anew);
        for (uint32_t q = MB; q < blocks; q++) add(q, spare[(q - MB) * 64u + lane], anew);
        if constexpr (OUT == OUT_F16) {
            for (; anew != 0; anew &= anew - 1u) {
                const uint32_t i = (uint32_t)__builtin_ctzll(anew), slot = slots[i];
                const GGQ_GLOBAL uint8_t* value = (GGQ_GLOBAL const uint8_t*)a.hidden + (uint64_t)slot * a.ff * 2;
                uint32_t at = lane;
                asm volatile("" : "+v"(at));
                const float y = moe_big<F>(rows, row_bytes, value, value + (uint64_t)pairs * a.ff * 2, from, span, a.ff, at);
                if (at < 16u) part[slot / a.top_k * 16u + at] += shares[i] * y;
            }
        }
        wave_sync();
        nth++;
        span = 0;
        if (item < last) start();
    };
    if (item < last) start();
    while (item < last) {
        one();
        if (span == n_spans || item == last) finish();
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.tokens * 16u; i += W * 64) {
        const float* sums = reinterpret_cast<const float*>(dyn);
        float v = sums[i];
        for (uint32_t w = 1; w < W; w++) v += sums[(uint64_t)w * a.tokens * 16u + i];
        const uint64_t at = (uint64_t)(i >> 4) * a.dim + row0 + (i & 15u);
        if (a.parts > 1) a.part[(uint64_t)blockIdx.y * a.tokens * a.dim + at] = v;
        else if constexpr (OUT == OUT_F16) reinterpret_cast<_Float16*>(a.y)[at] = (_Float16)v;
        else reinterpret_cast<uint16_t*>(a.y)[at] = (uint16_t)(pack_bf16(v, 0.0f) & 0xFFFFu);
    }
}

// y = the parts of moe_down in order, four values per lane
template <int OUT>
__global__ __launch_bounds__(256) void moe_combine(const float* __restrict__ part, uint8_t* __restrict__ y, uint32_t parts, uint32_t quads)
{
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= quads) return;
    f32x4 v = reinterpret_cast<const f32x4*>(part)[i];
    for (uint32_t p = 1; p < parts; p++) v += reinterpret_cast<const f32x4*>(part)[(uint64_t)p * quads + i];
    if constexpr (OUT == OUT_F16) reinterpret_cast<u32x2*>(y)[i] = u32x2{pack_f16(v.x, v.y), pack_f16(v.z, v.w)};
    else reinterpret_cast<u32x2*>(y)[i] = u32x2{pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)};
}

}  // namespace ggq
