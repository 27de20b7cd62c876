// ggq_rows.hpp -- gfx950 device code for what a transformer block does to whole ROWS between its linears: the residual sum with the block's gate, the
// norms before and after it, the modulation, and the 8-bit form of a row that the integer product (ggq_int8.hpp) reads.
//
// Mathematics, per row of `dim` elements (every optional part is skipped where its pointer is null):
//     h = branch                    | post_weight * N_post(branch)                       norm of the block's output
//     r = stream + gate * h                                                              new residual stream, stored in the stream's type
//     y = N(r) * weight + bias;  y = y * (1 + scale) + shift                             norm of the next block's input, modulated
//     N(v) = v / sqrt(mean(v^2) + eps)          or      (v - mean v) / sqrt(mean((v - mean v)^2) + eps)
// and, where 8-bit rows are asked for, with a = max |y|:   q = rint(127 y / a) (half to even),  q_scale = a / 127.
//
// Everything between the loads and the stores is fp32 in registers: r is NOT rounded to the stream's type before it is normed (one rounding less than
// separate kernels make), sums and squares are fp32, the variance is taken about the mean in a second pass over the registers.  The quotient 127 y / a is
// formed in fp64 and rounded to fp32 before rint: in 16-bit rows |y| = a/2 is common and 63.5 has to be seen as exactly half-way, which a reciprocal in
// fp32 misses; an fp32 product of two 24-bit values is not exact.  (A norm's rows are fp32 and share the code.)
//
// What bounds it: HBM.  One pass: stream and branch are read once, r and y written once.  A row lives in the registers of one wave (short rows: no
// barrier) or of the up to 16 waves of a workgroup, the longest in LDS.
#pragma once

#include "ggq_linear.hpp"

namespace ggq {

enum : int { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
// which parameter pointers hold fp32 (the others hold the stream's type)
enum : uint32_t { P32_POST = 1u, P32_GATE = 2u, P32_WEIGHT = 4u, P32_BIAS = 8u, P32_SCALE = 16u, P32_SHIFT = 32u };

struct RowArgs {
    const uint8_t *stream, *branch;
    uint8_t *stream_out, *y;
    float* y_scale;
    const uint8_t *post_weight, *gate, *weight, *bias, *scale, *shift;
    uint64_t rows, gate_stride, scale_stride, shift_stride;     // strides of the per-sample vectors, in elements
    uint64_t y_stride;                                          // 8-bit rows: bytes from one to the next; columns dim .. y_stride - 1 are written as zeros
    uint32_t dim, rows_per_mod, p32;
    int norm, post_norm;
    float eps;
};

// 16 bytes at any 2-byte boundary: rows of an odd number of 16-bit elements start there (global memory takes unaligned vector accesses)
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <int DT> GGQ_DEV float row_elem(const uint8_t* p, uint64_t i)
{
    if constexpr (DT == OUT_F32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (DT == OUT_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    else return bits_f32((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}

// elements i .. i + 7 of a vector of `dim`; zeros past its end
template <int DT> GGQ_DEV void row_load8(const uint8_t* p, uint32_t i, uint32_t dim, float (&v)[8])
{
    if (i + 8u <= dim) {
        if constexpr (DT == OUT_F32) {
            const u32x4_any a = *reinterpret_cast<const u32x4_any*>(p + (uint64_t)i * 4), b = *reinterpret_cast<const u32x4_any*>(p + (uint64_t)i * 4 + 16);
#pragma unroll
            for (int k = 0; k < 4; k++) { v[k] = bits_f32(a[k]); v[4 + k] = bits_f32(b[k]); }
        } else {
            const u32x4_any a = *reinterpret_cast<const u32x4_any*>(p + (uint64_t)i * 2);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (DT == OUT_F16) { const h2 h = as_h2(a[k]); v[2 * k] = (float)h.x; v[2 * k + 1] = (float)h.y; }
                else { v[2 * k] = bits_f32(a[k] << 16); v[2 * k + 1] = bits_f32(a[k] & 0xFFFF0000u); }
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = i + (uint32_t)k < dim ? row_elem<DT>(p, i + (uint32_t)k) : 0.0f;
    }
}

template <int DT> GGQ_DEV void row_store8(uint8_t* p, uint32_t i, uint32_t dim, const float (&v)[8])
{
    if (i + 8u <= dim) {
        if constexpr (DT == OUT_F32) {
            u32x4_any a, b;
#pragma unroll
            for (int k = 0; k < 4; k++) { a[k] = __builtin_bit_cast(uint32_t, v[k]); b[k] = __builtin_bit_cast(uint32_t, v[4 + k]); }
            *reinterpret_cast<u32x4_any*>(p + (uint64_t)i * 4) = a;
            *reinterpret_cast<u32x4_any*>(p + (uint64_t)i * 4 + 16) = b;
        } else {
            u32x4_any a;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (DT == OUT_F16) a[k] = as_u32(h2{(_Float16)v[2 * k], (_Float16)v[2 * k + 1]});
                else a[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
            }
            *reinterpret_cast<u32x4_any*>(p + (uint64_t)i * 2) = a;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (i + (uint32_t)k >= dim) break;
            if constexpr (DT == OUT_F32) reinterpret_cast<float*>(p)[i + (uint32_t)k] = v[k];
            else if constexpr (DT == OUT_F16) reinterpret_cast<_Float16*>(p)[i + (uint32_t)k] = (_Float16)v[k];
            else reinterpret_cast<uint16_t*>(p)[i + (uint32_t)k] = (uint16_t)(pack_bf16(v[k], 0.0f) & 0xFFFFu);
        }
    }
}

template <int CTRL, int ROWS> GGQ_DEV uint32_t dpp_u(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false); }
GGQ_DEV uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// over the 64 lanes of a wave, the same value in every lane
GGQ_DEV float wave_sum(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sum_lane63(v)), 63)); }
GGQ_DEV uint32_t wave_umax(uint32_t v)
{
    v = umax(v, dpp_u<0xB1, 0xF>(v));
    v = umax(v, dpp_u<0x4E, 0xF>(v));
    v = umax(v, dpp_u<0x141, 0xF>(v));
    v = umax(v, dpp_u<0x140, 0xF>(v));
    v = umax(v, dpp_u<0x142, 0xA>(v));
    v = umax(v, dpp_u<0x143, 0xC>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Sum / maximum over the waves of a team, the same value in every lane.  SOLO: the team is one wave.  Else through red[], one slot of 16 per reduction (the
// places of absent waves hold zeros), so that one barrier is enough: lane l reads place l % 16 and the 16 lanes of a DPP row fold them.
template <bool SOLO> GGQ_DEV float team_sum(float v, float* red)
{
    v = wave_sum(v);
    if constexpr (!SOLO) {
        if ((threadIdx.x & 63u) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[threadIdx.x & 15u];
        v += dpp_f<0xB1, 0xF>(v);
        v += dpp_f<0x4E, 0xF>(v);
        v += dpp_f<0x141, 0xF>(v);
        v += dpp_f<0x140, 0xF>(v);
    }
    return v;
}
template <bool SOLO> GGQ_DEV uint32_t team_umax(uint32_t v, float* red)
{
    v = wave_umax(v);
    if constexpr (!SOLO) {
        if ((threadIdx.x & 63u) == 0) red[threadIdx.x >> 6] = bits_f32(v);
        __syncthreads();
        v = __builtin_bit_cast(uint32_t, red[threadIdx.x & 15u]);
        v = umax(v, dpp_u<0xB1, 0xF>(v));
        v = umax(v, dpp_u<0x4E, 0xF>(v));
        v = umax(v, dpp_u<0x141, 0xF>(v));
        v = umax(v, dpp_u<0x140, 0xF>(v));
    }
    return v;
}

// The 8 fields of a row as integers of [-127, 127]; `to` = 127 / max|row| in fp64.
GGQ_DEV u32x2 row_quant8(const float (&v)[8], double to)
{
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; k++) w[k >> 2] |= ((uint32_t)(int)__builtin_rintf((float)((double)v[k] * to)) & 0xFFu) << (8 * (k & 3));
    return u32x2{w[0], w[1]};
}

// |v| of a row's largest element as bits (NaN counts as the largest), to 127 / a and a / 127.  A row of zeros: all quants 0, scale 0.  A row that
// holds an infinity or a NaN has no 8-bit form: its scale is NaN, its quants are 0, so that every product with it is NaN.
GGQ_DEV void row_scale(uint32_t amax_bits, double& to, float& scale)
{
    const float a = bits_f32(amax_bits);
    if (amax_bits >= 0x7F800000u) { to = 0.0; scale = __builtin_nanf(""); }
    else if (amax_bits == 0u) { to = 0.0; scale = 0.0f; }
    else { to = 127.0 / (double)a; scale = a / 127.0f; }
}

// A row as it was loaded: 8 elements per lane and vector
template <int DT> struct RowRaw { u32x4 a; };
template <> struct RowRaw<OUT_F32> { u32x4 a, b; };

template <int DT, bool TAIL> GGQ_DEV RowRaw<DT> row_raw(const uint8_t* p, uint32_t i, uint32_t dim)
{
    RowRaw<DT> r;
    constexpr int EB = DT == OUT_F32 ? 4 : 2;
    if constexpr (TAIL) {                                       // dim is no multiple of 8: the last vector element by element
        if (i + 8u > dim) {
            float v[8];
            row_load8<DT>(p, i, dim, v);
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; k++) w[k] = __builtin_bit_cast(uint32_t, v[k]);
            if constexpr (DT == OUT_F32) { r.a = u32x4{w[0], w[1], w[2], w[3]}; r.b = u32x4{w[4], w[5], w[6], w[7]}; }
            else {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if constexpr (DT == OUT_F16) r.a[k] = as_u32(h2{(_Float16)v[2 * k], (_Float16)v[2 * k + 1]});
                    else r.a[k] = (w[2 * k] >> 16) | (w[2 * k + 1] & 0xFFFF0000u);
                }
            }
            return r;
        }
        r.a = __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(p + (uint64_t)i * EB));
        if constexpr (DT == OUT_F32) r.b = __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(p + (uint64_t)i * EB + 16));
    } else {
        const bool in = i < dim;                                // lanes past the row read its start and keep zeros: no branch between the loads of a row
        const uint8_t* q = p + (uint64_t)(in ? i : 0u) * EB;
        r.a = __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(q));
        if constexpr (DT == OUT_F32) r.b = __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(q + 16));
#pragma unroll
        for (int k = 0; k < 4; k++) {
            r.a[k] = in ? r.a[k] : 0u;
            if constexpr (DT == OUT_F32) r.b[k] = in ? r.b[k] : 0u;
        }
    }
    return r;
}

template <int DT> GGQ_DEV void row_unpack(const RowRaw<DT>& r, float (&v)[8])
{
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (DT == OUT_F32) { v[k] = bits_f32(r.a[k]); v[4 + k] = bits_f32(r.b[k]); }
        else if constexpr (DT == OUT_F16) { const h2 h = as_h2(r.a[k]); v[2 * k] = (float)h.x; v[2 * k + 1] = (float)h.y; }
        else { v[2 * k] = bits_f32(r.a[k] << 16); v[2 * k + 1] = bits_f32(r.a[k] & 0xFFFF0000u); }
    }
}

// What a row is multiplied by, for 8 elements: G = post_weight * gate, A = weight * (1 + scale), B = bias * (1 + scale) + shift (1, 1, 0 where not given; 0
// past the row's end).  The same for all rows of a sample.
struct RowFactors { float g[8], a[8], b[8]; };

// `n` values of a parameter, widened: the loads only (their use comes after all parameters' loads)
struct RowParam { u32x4 a, b; };
template <int DT, bool TAIL> GGQ_DEV RowParam row_param_raw(const uint8_t* p, bool is32, uint64_t base, uint32_t i, uint32_t dim)
{
    RowParam r{};
    if (p == nullptr) return r;
    if (DT == OUT_F32 || is32) {
        const RowRaw<OUT_F32> w = row_raw<OUT_F32, TAIL>(p + base * 4, i, dim);
        r.a = w.a;
        r.b = w.b;
    } else {
        r.a = row_raw<DT, TAIL>(p + base * (DT == OUT_F32 ? 4 : 2), i, dim).a;
    }
    return r;
}
template <int DT> GGQ_DEV void row_param_unpack(const RowParam& r, bool is32, float (&v)[8])
{
    if (DT == OUT_F32 || is32) row_unpack<OUT_F32>(RowRaw<OUT_F32>{r.a, r.b}, v);
    else if constexpr (DT != OUT_F32) row_unpack<DT>(RowRaw<DT>{r.a}, v);
}

template <int DT, bool TAIL> GGQ_DEV void row_factors(const RowArgs& p, uint64_t sample, uint32_t i, uint32_t dim, RowFactors& f)
{
    const RowParam post = row_param_raw<DT, TAIL>(p.post_weight, p.p32 & P32_POST, 0, i, dim), gate = row_param_raw<DT, TAIL>(p.gate, p.p32 & P32_GATE, sample * p.gate_stride, i, dim);
    const RowParam weight = row_param_raw<DT, TAIL>(p.weight, p.p32 & P32_WEIGHT, 0, i, dim), bias = row_param_raw<DT, TAIL>(p.bias, p.p32 & P32_BIAS, 0, i, dim);
    const RowParam scale = row_param_raw<DT, TAIL>(p.scale, p.p32 & P32_SCALE, sample * p.scale_stride, i, dim);
    const RowParam shift = row_param_raw<DT, TAIL>(p.shift, p.p32 & P32_SHIFT, sample * p.shift_stride, i, dim);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) { f.g[k] = 1.0f; f.a[k] = 1.0f; f.b[k] = 0.0f; }
    if (p.post_weight != nullptr) row_param_unpack<DT>(post, p.p32 & P32_POST, f.g);
    if (p.gate != nullptr) {
        row_param_unpack<DT>(gate, p.p32 & P32_GATE, v);
#pragma unroll
        for (int k = 0; k < 8; k++) f.g[k] *= v[k];
    }
    if (p.weight != nullptr) row_param_unpack<DT>(weight, p.p32 & P32_WEIGHT, f.a);
    if (p.bias != nullptr) row_param_unpack<DT>(bias, p.p32 & P32_BIAS, f.b);
    if (p.scale != nullptr) {
        row_param_unpack<DT>(scale, p.p32 & P32_SCALE, v);
#pragma unroll
        for (int k = 0; k < 8; k++) { f.a[k] *= 1.0f + v[k]; f.b[k] *= 1.0f + v[k]; }
    }
    if (p.shift != nullptr) {
        row_param_unpack<DT>(shift, p.p32 & P32_SHIFT, v);
#pragma unroll
        for (int k = 0; k < 8; k++) f.b[k] += v[k];
    }
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (i + (TAIL ? (uint32_t)k : 0u) >= dim) { f.g[k] = 0.0f; f.a[k] = 0.0f; f.b[k] = 0.0f; }
}

// Zeros in red[]: what the places of waves that a team does not have hold.
GGQ_DEV void team_clear(float* red, uint32_t n)
{
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) red[i] = 0.0f;
    __syncthreads();
}

// Rows of up to 16 * 64 * 8 = 8192 elements (4096 where their number is no multiple of 8: the registers): 8 per lane, in registers from load to store.  A team of waves takes `rows_per_team` consecutive rows.  SOLO: a team
// is one wave, four teams to a workgroup, no barrier; else a team is a workgroup of up to 16 waves.  The next row's loads are under way while a row is
// computed, and a sample's factors stay in registers from row to row (read for every row, they would be up to 14 bytes per element from the caches
// beside the 8 from memory that the row itself moves).
// Measured: 9216 x 4096 bf16, rms, gate and modulation: 54 us from a kernel's start to its end, 66 us a call back to back in a replayed graph = 4.6 TB/s (a large copy: 6.3);
// 666 x 2432 fp16, layer norm: 9.1 us; one row of 4096: 3.3 us.  Rows of an odd number of elements go through the checks of every vector's end, in more registers: 36864 x 511
// fp16 71 us (512: 36), 9216 x 4095 114, and 9216 x 4097 bf16, through LDS, 163 us.  8-bit rows: 4608 x 4096 35 us, 3.7 TB/s, where 16-bit ones move 4.6.
template <int DT, bool SOLO, bool TAIL>
__global__ __launch_bounds__(SOLO ? 256 : TAIL ? 512 : 1024) void block_norm(const RowArgs a, uint32_t rows_per_team)
{
    constexpr int EB = DT == OUT_F32 ? 4 : 2;
    __shared__ __attribute__((aligned(16))) float red[2][5][16];            // two rows' reductions: a wave may be one row ahead of another
    const uint64_t team = SOLO ? (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6) : (uint64_t)blockIdx.x;
    const uint64_t first = team * rows_per_team, last = first + rows_per_team < a.rows ? first + rows_per_team : a.rows;
    if constexpr (!SOLO) team_clear(&red[0][0][0], 160);
    if (first >= last) return;                                              // a whole wave (SOLO: no barrier follows) or a whole workgroup
    const uint32_t lane = SOLO ? threadIdx.x & 63u : threadIdx.x;
    const uint32_t dim = a.dim, i = lane * 8u;
    const float inv_dim = 1.0f / (float)dim;

    // mean of squares of the row (about its mean: NORM_LAYER) -> mean, 1 / sqrt(mean square + eps); elements past the end are zeros, and stay out of the
    // centred sum
    auto moments = [&](const float (&v)[8], int kind, float* at, float& mean, float& rstd) {
        mean = 0.0f;
        float s = 0.0f;
        if (kind == NORM_LAYER) {
            mean = team_sum<SOLO>(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])), at) * inv_dim;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float d = i + (TAIL ? (uint32_t)k : 0u) < dim ? v[k] - mean : 0.0f;
                s = __builtin_fmaf(d, d, s);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) s = __builtin_fmaf(v[k], v[k], s);
        }
        rstd = 1.0f / __builtin_sqrtf(team_sum<SOLO>(s, at + 16) * inv_dim + a.eps);
    };

    RowRaw<DT> rs, rb;
    auto fetch = [&](uint64_t row) {
        rs = row_raw<DT, TAIL>(a.stream + row * dim * EB, i, dim);
        if (a.branch != nullptr) rb = row_raw<DT, TAIL>(a.branch + row * dim * EB, i, dim);
    };
    fetch(first);
    RowFactors f;
    uint64_t sample = first / a.rows_per_mod, sample_end = (sample + 1) * a.rows_per_mod;
    row_factors<DT, TAIL>(a, sample, i, dim, f);
    for (uint64_t row = first; row < last; row++) {
        float (*slot)[16] = red[(row - first) & 1u];
        if (row == sample_end) {
            sample++;
            sample_end += a.rows_per_mod;
            row_factors<DT, TAIL>(a, sample, i, dim, f);
        }
        float r[8], h[8];
        row_unpack<DT>(rs, r);
        if (a.branch != nullptr) row_unpack<DT>(rb, h);
        if (row + 1 < last) fetch(row + 1);
        const uint64_t at = row * dim * EB;
        if (a.branch != nullptr) {
            float mean = 0.0f, rstd = 1.0f;
            if (a.post_norm != NORM_NONE) moments(h, a.post_norm, slot[0], mean, rstd);
#pragma unroll
            for (int k = 0; k < 8; k++) r[k] = __builtin_fmaf((h[k] - mean) * rstd, f.g[k], r[k]);
            if (i < dim) row_store8<DT>(a.stream_out + at, i, TAIL ? dim : ~0u, r);
        }
        if (a.y == nullptr) continue;                                       // the last block: only the stream is wanted
        if (a.norm != NORM_NONE) {
            float mean, rstd;
            moments(r, a.norm, slot[2], mean, rstd);
#pragma unroll
            for (int k = 0; k < 8; k++) r[k] = __builtin_fmaf((r[k] - mean) * rstd, f.a[k], f.b[k]);
        }
        if (a.y_scale == nullptr) {
            if (i < dim) row_store8<DT>(a.y + at, i, TAIL ? dim : ~0u, r);
            continue;
        }
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) top = umax(top, __builtin_bit_cast(uint32_t, r[k]) & 0x7FFFFFFFu);
        double to;
        float scale;
        row_scale(team_umax<SOLO>(top, slot[4]), to, scale);
        if (lane == 0) a.y_scale[row] = scale;
        if (i < a.y_stride) {
#pragma unroll
            for (int k = 0; k < 8; k++) r[k] = to == 0.0 ? 0.0f : r[k];
            *reinterpret_cast<u32x2*>(a.y + row * a.y_stride + i) = row_quant8(r, to);
        }
    }
}

// 8-bit form of rows as they are: as block_norm without its norms, and without its registers -- a row per team, so many more rows are under way at once
// (4608 x 2432 bf16: 11 us, 22 with block_norm's kernel).
template <int DT, bool SOLO, bool TAIL>
__global__ __launch_bounds__(SOLO ? 256 : 1024) void quantize_rows(const uint8_t* __restrict__ x, uint64_t rows, uint32_t dim, uint8_t* __restrict__ q, uint64_t q_stride,
                                                                  float* __restrict__ q_scale)
{
    __shared__ float red[16];
    const uint64_t row = SOLO ? (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6) : (uint64_t)blockIdx.x;
    if (SOLO && row >= rows) return;
    const uint32_t lane = SOLO ? threadIdx.x & 63u : threadIdx.x, i = lane * 8u;
    const RowRaw<DT> raw = row_raw<DT, TAIL>(x + row * dim * (DT == OUT_F32 ? 4 : 2), i, dim);
    if constexpr (!SOLO) team_clear(red, 16);
    float v[8];
    row_unpack<DT>(raw, v);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) top = umax(top, __builtin_bit_cast(uint32_t, v[k]) & 0x7FFFFFFFu);
    double to;
    float scale;
    row_scale(team_umax<SOLO>(top, red), to, scale);
    if (lane == 0) q_scale[row] = scale;
    if (i < q_stride) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = to == 0.0 ? 0.0f : v[k];
        *reinterpret_cast<u32x2*>(q + row * q_stride + i) = row_quant8(v, to);
    }
}

// Longer rows, up to 32768 elements: a workgroup per row, the row in LDS as fp32 (each lane reads back what it wrote itself: no barrier for that).
constexpr uint32_t ROW_LONG_THREADS = 1024;
template <int DT>
__global__ __launch_bounds__(1024) void block_norm_long(const RowArgs a)
{
    constexpr int EB = DT == OUT_F32 ? 4 : 2;
    __shared__ __attribute__((aligned(16))) float red[5][16];
    extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
    const uint32_t dim = a.dim, span = a.y_scale != nullptr ? (uint32_t)a.y_stride : dim;
    const uint64_t row = blockIdx.x, at = row * dim * EB, sample = row / a.rows_per_mod;
    const float inv_dim = 1.0f / (float)dim;
    team_clear(&red[0][0], 80);
    f32x4* mine = reinterpret_cast<f32x4*>(dyn) + threadIdx.x * 2u;         // vector j of this lane: mine[2048 j], mine[2048 j + 1]
    auto get = [&](uint32_t i, float (&v)[8]) {
        const f32x4 p = mine[i / (ROW_LONG_THREADS * 8u) * (ROW_LONG_THREADS * 2u)], q = mine[i / (ROW_LONG_THREADS * 8u) * (ROW_LONG_THREADS * 2u) + 1u];
#pragma unroll
        for (int k = 0; k < 4; k++) { v[k] = p[k]; v[4 + k] = q[k]; }
    };
    auto put = [&](uint32_t i, const float (&v)[8]) {
        mine[i / (ROW_LONG_THREADS * 8u) * (ROW_LONG_THREADS * 2u)] = f32x4{v[0], v[1], v[2], v[3]};
        mine[i / (ROW_LONG_THREADS * 8u) * (ROW_LONG_THREADS * 2u) + 1u] = f32x4{v[4], v[5], v[6], v[7]};
    };
    auto each = [&](auto&& f) {
#pragma unroll 1
        for (uint32_t i = threadIdx.x * 8u; i < span; i += ROW_LONG_THREADS * 8u) f(i);
    };
    auto moments = [&](auto&& load, int kind, float* slot, float& mean, float& rstd) {
        mean = 0.0f;
        float s = 0.0f;
        if (kind == NORM_LAYER) {
            each([&](uint32_t i) {
                float v[8];
                load(i, v);
                s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            });
            mean = team_sum<false>(s, slot) * inv_dim;
            s = 0.0f;
        }
        each([&](uint32_t i) {
            float v[8];
            load(i, v);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float d = i + (uint32_t)k < dim ? v[k] - mean : 0.0f;
                s = __builtin_fmaf(d, d, s);
            }
        });
        rstd = 1.0f / __builtin_sqrtf(team_sum<false>(s, slot + 16) * inv_dim + a.eps);
    };
    float mean = 0.0f, rstd = 1.0f;
    auto branch = [&](uint32_t i, float (&v)[8]) { row_load8<DT>(a.branch + at, i, dim, v); };
    if (a.branch != nullptr && a.post_norm != NORM_NONE) moments(branch, a.post_norm, red[0], mean, rstd);
    each([&](uint32_t i) {
        float r[8];
        row_load8<DT>(a.stream + at, i, dim, r);
        if (a.branch != nullptr) {
            float h[8];
            branch(i, h);
            RowFactors f;
            row_factors<DT, true>(a, sample, i, dim, f);
#pragma unroll
            for (int k = 0; k < 8; k++) r[k] = __builtin_fmaf((h[k] - mean) * rstd, f.g[k], r[k]);
            if (i < dim) row_store8<DT>(a.stream_out + at, i, dim, r);
        }
        put(i, r);
    });
    if (a.y == nullptr) return;
    mean = 0.0f;
    rstd = 1.0f;
    if (a.norm != NORM_NONE) moments(get, a.norm, red[2], mean, rstd);
    uint32_t top = 0;
    each([&](uint32_t i) {
        float r[8];
        get(i, r);
        if (a.norm != NORM_NONE) {
            RowFactors f;
            row_factors<DT, true>(a, sample, i, dim, f);
#pragma unroll
            for (int k = 0; k < 8; k++) r[k] = __builtin_fmaf((r[k] - mean) * rstd, f.a[k], f.b[k]);
        }
        if (a.y_scale == nullptr) {
            row_store8<DT>(a.y + at, i, dim, r);
        } else {
            put(i, r);
#pragma unroll
            for (int k = 0; k < 8; k++) top = umax(top, __builtin_bit_cast(uint32_t, r[k]) & 0x7FFFFFFFu);
        }
    });
    if (a.y_scale == nullptr) return;
    double to;
    float scale;
    row_scale(team_umax<false>(top, red[4]), to, scale);
    if (threadIdx.x == 0) a.y_scale[row] = scale;
    each([&](uint32_t i) {
        float r[8];
        get(i, r);
#pragma unroll
        for (int k = 0; k < 8; k++) r[k] = to == 0.0 ? 0.0f : r[k];
        *reinterpret_cast<u32x2*>(a.y + row * a.y_stride + i) = row_quant8(r, to);
    });
}

}  // namespace ggq
