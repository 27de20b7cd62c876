// ggq_int8.hpp -- gfx950 device code: y = (xq . wq^T) * x_scale[row] * w_scale[column] + bias on v_mfma_i32_*_i8.
//
// Mathematics: 8-bit integers times 8-bit integers, summed exactly in int32 (|sum| <= 2^14 k < 2^31 for k <= 131071); the two scales factor out of the
// sum, so they, the bias and the one rounding to the output type are an epilogue in fp32.
//
// Two kernels:
//   linear_i8_tile   many rows of x: a workgroup owns TM rows of x  x  TN rows of w, both staged through LDS 128 bytes of k at a time (LDS-DMA, two
//                    buffers), every fragment one ds_read_b128.  Bound by the matrix cores' rate.
//   linear_i8_rows   up to 16 rows of x: a workgroup owns 16 rows of w, its waves split k, operands go straight from memory to registers.  Bound by
//                    reading w once.
// The contraction index may be permuted as long as both operands agree; out-of-range rows are clamped and their results not stored; columns of k past
// the end are read as zeros on the x side.
#pragma once

#include "ggq_rows.hpp"

namespace ggq {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int I8_BK = 128;                         // bytes (= elements) of k per staged step

__device__ const u32x4 I8_ZEROS[1] = {};

// the 16-byte column of row `row` sits at column ^ swz: the 16-lane groups of a ds_read_b128 ({0-3, 12-15, 20-27}, {4-11, 16-19, 28-31}, and + 32) then
// read 16 different bank quads at a row pitch of 128 bytes
GGQ_DEV uint32_t i8_swz(uint32_t row) { return (row >> 1) & 7u; }

GGQ_DEV void i8_dma16(const GGQ_GLOBAL uint8_t* src, uint8_t* lds_wave_base)
{
    __builtin_amdgcn_global_load_lds((const GGQ_GLOBAL void*)src, (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

template <int DT> GGQ_DEV float i8_bias(const uint8_t* bias, uint32_t n)
{
    return bias == nullptr ? 0.0f : row_elem<DT>(bias, n);
}

template <int DT> GGQ_DEV void i8_store(uint8_t* y, uint64_t at, float v)
{
    if constexpr (DT == OUT_F32) reinterpret_cast<float*>(y)[at] = v;
    else if constexpr (DT == OUT_F16) reinterpret_cast<_Float16*>(y)[at] = (_Float16)v;
    else reinterpret_cast<uint16_t*>(y)[at] = (uint16_t)(pack_bf16(v, 0.0f) & 0xFFFFu);
}

struct I8Args {
    const uint8_t *xq, *wq;
    const float *x_scale, *w_scale;
    const uint8_t* bias;
    uint8_t* y;
    uint64_t x_stride, w_stride;
    uint32_t m, n, k, tiles_m, tiles_n;
};

// TM x TN outputs per workgroup, WM x WN waves of (TM / WM) x (TN / WN) outputs each.  w is the A operand (rows of D = columns of y), x the B operand:
// a lane holds 4 consecutive columns of one row of y.
template <int DT, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void linear_i8_tile(const I8Args a)
{
    constexpr int THREADS = WM * WN * 64;
    constexpr int MT = TM / WM / 32, NT = TN / WN / 32;
    constexpr int UNITS = (TM + TN) * 8, UN = UNITS / THREADS;
    static_assert(UNITS % THREADS == 0 && MT >= 1 && NT >= 1 && TM % 16 == 0, "tile shape");
    constexpr uint32_t STAGE = (TM + TN) * I8_BK;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];

    const uint32_t t = threadIdx.x, lane = t & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 6));
    // XCD x takes a contiguous eighth of the tile list (rows of x fastest): its L2 holds a few rows of w tiles and all of x
    const uint32_t n_tiles = a.tiles_m * a.tiles_n;
    uint32_t tile = blockIdx.x;
    {
        const uint32_t q = n_tiles >> 3, r = n_tiles & 7u, xcd = tile & 7u, idx = tile >> 3;
        tile = (xcd < r ? xcd * (q + 1u) : r * (q + 1u) + (xcd - r) * q) + idx;
    }
    const uint32_t tn = tile / a.tiles_m, tm = tile - tn * a.tiles_m;
    const uint32_t m0 = tm * TM, n0 = tn * TN;

    // unit u = t + THREADS i of a stage: row u / 8 (x rows, then w rows), LDS slot u % 8, which holds 16-byte column (u % 8) ^ swz(row)
    const GGQ_GLOBAL uint8_t* src[UN];
    uint32_t col[UN];
#pragma unroll
    for (int i = 0; i < UN; i++) {
        const uint32_t u = t + (uint32_t)(THREADS * i), row = u >> 3;
        const bool is_x = row < (uint32_t)TM;
        const uint32_t rl = is_x ? row : row - (uint32_t)TM;
        col[i] = ((u & 7u) ^ i8_swz(rl)) * 16u;
        const uint32_t gr = (is_x ? m0 : n0) + rl, top = is_x ? a.m : a.n;
        src[i] = (GGQ_GLOBAL const uint8_t*)(is_x ? a.xq : a.wq) + (uint64_t)(gr < top ? gr : top - 1u) * (is_x ? a.x_stride : a.w_stride);
    }
    const uint32_t steps = (a.k + I8_BK - 1u) / I8_BK;
    auto stage = [&](uint32_t step) {
        uint8_t* dst = smem + (step & 1u) * STAGE;
        const uint32_t k0 = step * I8_BK;
        if (k0 + I8_BK <= a.k) {
#pragma unroll
            for (int i = 0; i < UN; i++) i8_dma16(src[i] + k0 + col[i], dst + (wave * 64u + (uint32_t)(THREADS * i)) * 16u);
        } else {                                       // the last step: columns past k are zeros of x against whatever starts the row of w
#pragma unroll
            for (int i = 0; i < UN; i++) {
                const bool in = k0 + col[i] < a.k, is_x = t + (uint32_t)(THREADS * i) < (uint32_t)TM * 8u;
                const GGQ_GLOBAL uint8_t* p = in ? src[i] + k0 + col[i] : (is_x ? (const GGQ_GLOBAL uint8_t*)I8_ZEROS : src[i]);
                i8_dma16(p, dst + (wave * 64u + (uint32_t)(THREADS * i)) * 16u);
            }
        }
    };

    const uint32_t wm = wave / WN, wn = wave % WN, r32 = lane & 31u, h = lane >> 5, fswz = i8_swz(r32);
    const uint32_t xrow = wm * (TM / WM) + r32, wrow = (uint32_t)TM + wn * (TN / WN) + r32;
    i32x16 acc[NT][MT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[nt][mt][i] = 0;

    stage(0);
    for (uint32_t s = 0; s < steps; s++) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // this wave's part of step s has landed; the barrier publishes it, and says that every
        __syncthreads();                                       // wave is done reading step s - 1, whose buffer step s + 1 goes to
        if (s + 1 < steps) stage(s + 1);
        const uint8_t* buf = smem + (s & 1u) * STAGE;
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
            const uint32_t c = (((uint32_t)(2 * kk) + h) ^ fswz) * 16u;
            i32x4 wa[NT], xb[MT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) wa[nt] = *reinterpret_cast<const i32x4*>(buf + (wrow + 32u * (uint32_t)nt) * I8_BK + c);
#pragma unroll
            for (int mt = 0; mt < MT; mt++) xb[mt] = *reinterpret_cast<const i32x4*>(buf + (xrow + 32u * (uint32_t)mt) * I8_BK + c);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++) acc[nt][mt] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wa[nt], xb[mt], acc[nt][mt], 0, 0, 0);
        }
    }

    // D[row = 8 (i / 4) + 4 h + i % 4][column = r32] = sum of (row of w, row of x): four consecutive columns of y per lane and register group.  Each wave turns
    // 32 rows x (TN / WN) columns of sums through its own part of LDS, so that a lane then holds 8 consecutive columns of a row (whose scales and bias it keeps)
    // and a row is stored in full lines.  (Stored straight from the accumulators, 2 bytes at a time, the epilogue took longer than the product.)
    constexpr uint32_t COLS = TN / WN, LPR = COLS / 8, RPI = 64 / LPR;      // columns of a wave, lanes per row, rows per store instruction
    constexpr uint32_t SLOTS = COLS / 4;                                    // 16-byte places of a row in LDS, XOR-swizzled by the row
    static_assert(WM * WN * 32 * COLS * 4 <= 2 * STAGE, "the turned sums fit the staging buffers");
    __syncthreads();                                                        // every wave is done with the staging buffers
    int* turn = reinterpret_cast<int*>(smem) + wave * (32u * COLS);
    const uint32_t nc = n0 + wn * COLS + (lane % LPR) * 8u;
    float sw[8], bias[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const uint32_t c = nc + (uint32_t)k < a.n ? nc + (uint32_t)k : a.n - 1u;
        sw[k] = a.w_scale[c];
        bias[k] = i8_bias<DT>(a.bias, c);
    }
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<i32x4*>(turn + r32 * COLS + (((uint32_t)(8 * nt + 2 * g) + h) ^ (r32 & (SLOTS - 1u))) * 4u) =
                    i32x4{acc[nt][mt][4 * g], acc[nt][mt][4 * g + 1], acc[nt][mt][4 * g + 2], acc[nt][mt][4 * g + 3]};
        wave_sync();
#pragma unroll
        for (uint32_t i = 0; i < 32u / RPI; i++) {
            const uint32_t row = i * RPI + lane / LPR, mr = m0 + wm * (TM / WM) + 32u * (uint32_t)mt + row;
            const i32x4 p = *reinterpret_cast<const i32x4*>(turn + row * COLS + (((lane % LPR) * 2u) ^ (row & (SLOTS - 1u))) * 4u);
            const i32x4 q = *reinterpret_cast<const i32x4*>(turn + row * COLS + (((lane % LPR) * 2u + 1u) ^ (row & (SLOTS - 1u))) * 4u);
            if (mr < a.m && nc < a.n) {
                const float sx = a.x_scale[mr];
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = (float)(k < 4 ? p[k] : q[k - 4]) * (sx * sw[k]) + bias[k];
                row_store8<DT>(a.y + (uint64_t)mr * a.n * (DT == OUT_F32 ? 4 : 2), nc, a.n, v);
            }
        }
        wave_sync();
    }
}

// Up to 16 rows of x: 16 rows of w per workgroup, k split over its waves in pieces of 64, partial sums added through LDS (integers: any order is exact).
constexpr int I8_ROW_WAVES = 8;
template <int DT>
__global__ __launch_bounds__(I8_ROW_WAVES * 64) void linear_i8_rows(const I8Args a)
{
    __shared__ i32x4 red[I8_ROW_WAVES][64];
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, c = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t n0 = blockIdx.x * 16u, m0 = blockIdx.y * 16u;
    const uint32_t wr = n0 + r < a.n ? n0 + r : a.n - 1u, xr = m0 + r < a.m ? m0 + r : a.m - 1u;
    const GGQ_GLOBAL uint8_t* w = (GGQ_GLOBAL const uint8_t*)a.wq + (uint64_t)wr * a.w_stride;
    const GGQ_GLOBAL uint8_t* x = (GGQ_GLOBAL const uint8_t*)a.xq + (uint64_t)xr * a.x_stride;
    const uint32_t steps = (a.k + 63u) / 64u;
    i32x4 acc{0, 0, 0, 0};
    for (uint32_t s = wave; s < steps; s += I8_ROW_WAVES) {
        const uint32_t k = s * 64u + c * 16u;
        const bool in = k < a.k;                       // past the end: zeros of x against the start of the row of w
        const i32x4 wa = *(const GGQ_GLOBAL i32x4*)(in ? w + k : w);
        const i32x4 xb = *(const GGQ_GLOBAL i32x4*)(in ? x + k : (const GGQ_GLOBAL uint8_t*)I8_ZEROS);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa, xb, acc, 0, 0, 0);
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave != 0) return;
    for (int v = 1; v < I8_ROW_WAVES; v++) acc += red[v][lane];
    const uint32_t mr = m0 + r;
    if (mr >= a.m) return;
    const float sx = a.x_scale[mr];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t nc = n0 + 4u * c + (uint32_t)i;
        if (nc < a.n) i8_store<DT>(a.y, (uint64_t)mr * a.n + nc, (float)acc[i] * (sx * a.w_scale[nc]) + i8_bias<DT>(a.bias, nc));
    }
}

}  // namespace ggq
