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
// fp32 misses; an fp32 product of two 24-bit values is not exact.
//
// What bounds it: HBM.  One pass: stream and branch are read once, r and y written once.  A row lives in the registers of one wave (long launches: no
// barrier, no LDS) or of 4 / 8 waves (few rows: the row's latency is what counts).
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

template <int DT> GGQ_DEV void row_param8(const uint8_t* p, bool is32, uint64_t base, uint32_t i, uint32_t dim, float (&v)[8])
{
    if (is32) row_load8<OUT_F32>(p + base * 4, i, dim, v);
    else row_load8<DT>(p + base * (DT == OUT_F32 ? 4 : 2), i, dim, v);
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

// Sum / maximum over the WAVES waves of a row.  `slot` numbers the reductions of a kernel: each has LDS of its own, so one barrier is enough.
template <int WAVES> GGQ_DEV float row_sum(float v, float (*red)[8], int slot)
{
    v = wave_sum(v);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63u) == 0) red[slot][threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) v += red[slot][w];
    }
    return v;
}
template <int WAVES> GGQ_DEV uint32_t row_umax(uint32_t v, float (*red)[8], int slot)
{
    v = wave_umax(v);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63u) == 0) red[slot][threadIdx.x >> 6] = bits_f32(v);
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) v = umax(v, __builtin_bit_cast(uint32_t, red[slot][w]));
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

// One row per WAVES waves; NV vectors of 8 elements per lane.  WAVES = 1: the four waves of a workgroup hold four rows.
template <int DT, int WAVES, int NV>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void block_norm(const RowArgs a)
{
    __shared__ float red[6][8];
    const uint64_t row = WAVES == 1 ? (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6) : (uint64_t)blockIdx.x;
    if (row >= a.rows) return;                                              // a whole wave (WAVES = 1: no barrier follows) or a whole workgroup
    const uint32_t lane = WAVES == 1 ? threadIdx.x & 63u : threadIdx.x;
    constexpr uint32_t STEP = WAVES * 64 * 8;
    constexpr int EB = DT == OUT_F32 ? 4 : 2;
    const uint32_t dim = a.dim;
    const float inv_dim = 1.0f / (float)dim;
    const uint64_t at = row * dim * EB;
    const uint64_t sample = row / a.rows_per_mod;

    float r[NV][8];
#pragma unroll
    for (int j = 0; j < NV; j++) row_load8<DT>(a.stream + at, lane * 8u + (uint32_t)j * STEP, dim, r[j]);

    // mean and 1 / sqrt(var + eps) of the row in v; padded elements are 0 and stay out of the centred sum
    auto moments = [&](const float (&v)[NV][8], int kind, int slot, float& mean, float& rstd) {
        mean = 0.0f;
        if (kind == NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int k = 0; k < 8; k++) s += v[j][k];
            mean = row_sum<WAVES>(s, red, slot) * inv_dim;
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float d = lane * 8u + (uint32_t)j * STEP + (uint32_t)k < dim ? v[j][k] - mean : 0.0f;
                s += d * d;
            }
        rstd = 1.0f / __builtin_sqrtf(row_sum<WAVES>(s, red, slot + 1) * inv_dim + a.eps);
    };

    if (a.branch != nullptr) {
        float h[NV][8];
#pragma unroll
        for (int j = 0; j < NV; j++) row_load8<DT>(a.branch + at, lane * 8u + (uint32_t)j * STEP, dim, h[j]);
        if (a.post_norm != NORM_NONE) {
            float mean, rstd;
            moments(h, a.post_norm, 0, mean, rstd);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                float w[8];
                if (a.post_weight != nullptr) row_param8<DT>(a.post_weight, a.p32 & P32_POST, 0, lane * 8u + (uint32_t)j * STEP, dim, w);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    h[j][k] = (h[j][k] - mean) * rstd;
                    if (a.post_weight != nullptr) h[j][k] *= w[k];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t i = lane * 8u + (uint32_t)j * STEP;
            if (a.gate != nullptr) {
                float g[8];
                row_param8<DT>(a.gate, a.p32 & P32_GATE, sample * a.gate_stride, i, dim, g);
#pragma unroll
                for (int k = 0; k < 8; k++) h[j][k] *= g[k];
            }
#pragma unroll
            for (int k = 0; k < 8; k++) r[j][k] = i + (uint32_t)k < dim ? r[j][k] + h[j][k] : 0.0f;
            if (i < dim) row_store8<DT>(a.stream_out + at, i, dim, r[j]);
        }
    }
    if (a.y == nullptr) return;                                             // the last block: only the stream is wanted

    if (a.norm != NORM_NONE) {
        float mean, rstd;
        moments(r, a.norm, 2, mean, rstd);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t i = lane * 8u + (uint32_t)j * STEP;
            float w[8], b[8], sc[8], sh[8];
            if (a.weight != nullptr) row_param8<DT>(a.weight, a.p32 & P32_WEIGHT, 0, i, dim, w);
            if (a.bias != nullptr) row_param8<DT>(a.bias, a.p32 & P32_BIAS, 0, i, dim, b);
            if (a.scale != nullptr) row_param8<DT>(a.scale, a.p32 & P32_SCALE, sample * a.scale_stride, i, dim, sc);
            if (a.shift != nullptr) row_param8<DT>(a.shift, a.p32 & P32_SHIFT, sample * a.shift_stride, i, dim, sh);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                float v = (r[j][k] - mean) * rstd;
                if (a.weight != nullptr) v *= w[k];
                if (a.bias != nullptr) v += b[k];
                if (a.scale != nullptr) v *= 1.0f + sc[k];
                if (a.shift != nullptr) v += sh[k];
                r[j][k] = i + (uint32_t)k < dim ? v : 0.0f;
            }
        }
    }
    if (a.y_scale == nullptr) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t i = lane * 8u + (uint32_t)j * STEP;
            if (i < dim) row_store8<DT>(a.y + at, i, dim, r[j]);
        }
        return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < 8; k++) top = umax(top, __builtin_bit_cast(uint32_t, r[j][k]) & 0x7FFFFFFFu);
    double to;
    float scale;
    row_scale(row_umax<WAVES>(top, red, 4), to, scale);
    if (lane == 0) a.y_scale[row] = scale;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const uint32_t i = lane * 8u + (uint32_t)j * STEP;
        if (i < a.y_stride) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = to == 0.0 ? 0.0f : r[j][k];
            *reinterpret_cast<u32x2*>(a.y + row * a.y_stride + i) = row_quant8(v, to);
        }
    }
}

}  // namespace ggq
