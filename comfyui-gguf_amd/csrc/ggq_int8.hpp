// ggq_int8.hpp -- gfx950 device code: y = (xq . wq^T) * x_scale[row] * w_scale[column] + bias on v_mfma_i32_*_i8.
//
// Mathematics: 8-bit integers times 8-bit integers, summed exactly in int32 (|sum| <= 2^14 k < 2^31 for k <= 131071); the two scales factor out of the
// sum, so they, the bias and the one rounding to the output type are an epilogue in fp32.
//
// Two kernels:
//   linear_i8_tile   many rows of x: a workgroup owns TM rows of x  x  TN rows of w, both staged through LDS 128 bytes of k at a time (LDS-DMA, two
//                    to four buffers), every fragment one ds_read_b128.  Bound by the matrix cores' rate.
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

// TM x TN outputs per workgroup of WM x WN x KS waves: (TM / WM) x (TN / WN) outputs per wave, KS waves sharing them and splitting each step's k.  w is the A
// operand (rows of D = columns of y), x the B operand.
//
// A step's fragments are read one k-piece ahead of the matrix instructions that use them, across the barrier too: the barrier that publishes step s + 1
// stands BEFORE the last k-piece of step s is multiplied, so that the first fragments of s + 1 arrive under it.  At that barrier every wave has read
// step s completely, so its buffer takes the loads of step s + 2 (NB = 2), or step s + 3's went to the buffer of step s - 1 when step s began (NB = 4).
// With 256 x 256 the reads (24 x 64 x 16 bytes per wave and step) and the LDS-DMA writes take as long as the matrix instructions (32 per wave, 32 cycles each):
// they have to overlap completely, hence the interleaved issue order that sched_group_barrier asks for.
//
// Measured (4608 x 9728 x 2432 / 4608 x 10240 x 4096, us): fragments read where they are used 151 / 206; tiles in groups of 4 rows of tiles (L2) 126 / 203; read one
// piece ahead 130 / 193, interleaved 122 / 188; the branches for a partial last step out of the loop, so that the compiler counts the reads in flight
// instead of waiting for all, 118 / 178 = 1840 / 2172 TOP/s (in turn with the library's int8 product, which stores int32: 118 and
// 118, 179 and 182; 512 x 10240 x 4096: 32 and 39).  4 waves of 128 x 128: 137 / 203; 64 bytes of k and 4 buffers: 131 / 204.
template <int DT, int TM, int TN, int WM, int WN, int KS, int NB>
__global__ __launch_bounds__(WM * WN * KS * 64) void linear_i8_tile(const I8Args a)
{
    constexpr int THREADS = WM * WN * KS * 64;
    constexpr int MT = TM / WM / 32, NT = TN / WN / 32;
    constexpr int UNITS = (TM + TN) * 8, UN = UNITS / THREADS;
    constexpr int KK = 4 / KS;                                              // k-pieces of 32 per wave and step
    static_assert(UNITS % THREADS == 0 && MT >= 1 && NT >= 1 && TM % 16 == 0 && KK % 2 == 0 && NB >= 2, "tile shape");
    constexpr uint32_t STAGE = (TM + TN) * I8_BK;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];

    const uint32_t t = threadIdx.x, lane = t & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 6));
    // XCD x takes a contiguous eighth of the tile list; in the list, 4 rows of tiles at a time run through all columns: an L2 holds their x while w streams by
    const uint32_t n_tiles = a.tiles_m * a.tiles_n;
    uint32_t tile = blockIdx.x;
    {
        const uint32_t q = n_tiles >> 3, r = n_tiles & 7u, xcd = tile & 7u, idx = tile >> 3;
        tile = (xcd < r ? xcd * (q + 1u) : r * (q + 1u) + (xcd - r) * q) + idx;
    }
    const uint32_t group = tile / (4u * a.tiles_n), in = tile - group * 4u * a.tiles_n;
    const uint32_t high = a.tiles_m - group * 4u < 4u ? a.tiles_m - group * 4u : 4u;
    const uint32_t tm = group * 4u + in % high, tn = in / high;
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
        src[i] = (GGQ_GLOBAL const uint8_t*)(is_x ? a.xq : a.wq) + (uint64_t)(gr < top ? gr : top - 1u) * (is_x ? a.x_stride : a.w_stride) + col[i];
    }
    const uint32_t steps = (a.k + I8_BK - 1u) / I8_BK;
    auto stage_whole = [&](uint32_t step, uint32_t buf) {
#pragma unroll
        for (int i = 0; i < UN; i++) i8_dma16(src[i] + step * I8_BK, smem + buf * STAGE + (wave * 64u + (uint32_t)(THREADS * i)) * 16u);
    };
    auto stage = [&](uint32_t step, uint32_t buf) {
        uint8_t* dst = smem + buf * STAGE;
        const uint32_t k0 = step * I8_BK;
        if (k0 + I8_BK <= a.k) {
            stage_whole(step, buf);
        } else {                                       // the last step: columns past k are zeros of x against whatever starts the row of w
#pragma unroll
            for (int i = 0; i < UN; i++) {
                const bool in_k = k0 + col[i] < a.k, is_x = t + (uint32_t)(THREADS * i) < (uint32_t)TM * 8u;
                const GGQ_GLOBAL uint8_t* p = in_k ? src[i] + k0 : (is_x ? (const GGQ_GLOBAL uint8_t*)I8_ZEROS : src[i] - col[i]);
                i8_dma16(p, dst + (wave * 64u + (uint32_t)(THREADS * i)) * 16u);
            }
        }
    };

    const uint32_t ks = wave / (WM * WN), place = wave % (WM * WN), wm = place / WN, wn = place % WN, r32 = lane & 31u, h = lane >> 5, fswz = i8_swz(r32);
    const uint32_t xrow = wm * (TM / WM) + r32, wrow = (uint32_t)TM + wn * (TN / WN) + r32;
    i32x16 acc[NT][MT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[nt][mt][i] = 0;
    i32x4 wa[2][NT], xb[2][MT];
    auto fragments = [&](const uint8_t* buf, int kk, int set) {
        const uint32_t c = ((2u * (uint32_t)(KK * (int)ks + kk) + h) ^ fswz) * 16u;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) wa[set][nt] = *reinterpret_cast<const i32x4*>(buf + (wrow + 32u * (uint32_t)nt) * I8_BK + c);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) xb[set][mt] = *reinterpret_cast<const i32x4*>(buf + (xrow + 32u * (uint32_t)mt) * I8_BK + c);
    };
    // every load but the newest IN_FLIGHT of this wave has landed and its LDS reads have returned; the barrier says so to the others.  (Raw s_barrier: with
    // __syncthreads() the compiler would wait for all loads.)
    auto publish_keep = [&]() {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(UN * (NB == 2 ? 1 : NB - 2)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto publish_all = [&]() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    constexpr uint32_t AHEAD = NB == 2 ? 2 : NB - 1;                        // steps requested before the first is used
#pragma unroll
    for (uint32_t s = 0; s < AHEAD; s++)
        if (s < steps) stage(s, s);
    if (steps >= AHEAD) publish_keep();
    else publish_all();
    fragments(smem, 0, 0);
    uint32_t cur = 0, free_buf = NB - 1;
    auto multiply = [&](int set) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) acc[nt][mt] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wa[set][nt], xb[set][mt], acc[nt][mt], 0, 0, 0);
        if constexpr (NT * MT >= NT + MT) {                                 // one LDS read behind each of the first matrix instructions
#pragma unroll
            for (int q = 0; q < NT + MT; q++) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, NT * MT - NT - MT, 0);
        }
    };
    auto turn_buffers = [&]() {
        free_buf = cur;
        cur = cur + 1 == NB ? 0 : cur + 1;
    };
    uint32_t s = 0;
    // steps whose requests are whole: no branch but the loop's
    const uint32_t whole = a.k / I8_BK > AHEAD ? a.k / I8_BK - AHEAD : 0u;
    for (; s < whole; s++) {
        const uint32_t next = cur + 1 == NB ? 0 : cur + 1;
        if constexpr (NB > 2) stage_whole(s + NB - 1, free_buf);
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (kk + 1 < KK) {
                fragments(smem + cur * STAGE, kk + 1, (kk + 1) & 1);
            } else {
                if constexpr (NB > 2) publish_keep();
                else publish_all();
                if constexpr (NB == 2) stage_whole(s + 2, cur);
                fragments(smem + next * STAGE, 0, 0);
            }
            multiply(kk & 1);
        }
        turn_buffers();
    }
    for (; s < steps; s++) {
        const uint32_t next = cur + 1 == NB ? 0 : cur + 1;
        if constexpr (NB > 2) {
            if (s + NB - 1 < steps) stage(s + NB - 1, free_buf);
        }
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (kk + 1 < KK) {
                fragments(smem + cur * STAGE, kk + 1, (kk + 1) & 1);
            } else if (s + 1 < steps) {
                if (NB > 2 && s + NB - 1 < steps) publish_keep();
                else publish_all();
                if constexpr (NB == 2) {
                    if (s + 2 < steps) stage(s + 2, cur);
                }
                fragments(smem + next * STAGE, 0, 0);
            }
            multiply(kk & 1);
        }
        turn_buffers();
    }
    if constexpr (KS > 1) {                                                 // integers: the k-parts add up to the same in any order
        __syncthreads();
        i32x16* part = reinterpret_cast<i32x16*>(smem);
        static_assert((KS - 1) * WM * WN * 64 * 64 <= NB * STAGE, "partial sums fit the staging buffers");
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if (ks) part[((ks - 1u) * (WM * WN) + place) * 64u + lane] = acc[nt][mt];
                __syncthreads();
                if (!ks)
                    for (uint32_t q = 0; q < KS - 1; q++) acc[nt][mt] += part[(q * (WM * WN) + place) * 64u + lane];
                __syncthreads();
            }
        if (ks) return;
    } else {
        __syncthreads();                                                    // every wave is done with the staging buffers
    }

    // D[row = 8 (i / 4) + 4 h + i % 4][column = r32] = sum of (row of w, row of x): four consecutive columns of y per lane and register group.  Each wave turns
    // 32 rows x (TN / WN) columns of sums through its own part of LDS, so that a lane then holds 8 consecutive columns of a row (whose scales and bias it keeps)
    // and a row is stored in full lines.  (Stored straight from the accumulators, 2 bytes at a time, the epilogue took longer than the product.)
    constexpr uint32_t COLS = TN / WN, LPR = COLS / 8, RPI = 64 / LPR;      // columns of a wave, lanes per row, rows per store instruction
    constexpr uint32_t SLOTS = COLS / 4;                                    // 16-byte places of a row in LDS, XOR-swizzled by the row
    static_assert(WM * WN * 32 * COLS * 4 <= NB * STAGE, "the turned sums fit the staging buffers");
    int* turn = reinterpret_cast<int*>(smem) + place * (32u * COLS);
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

// Up to 16 rows of x: 16 rows of w per workgroup, k split over its waves in pieces of 64, partial sums added through LDS (integers: any order is exact).  A
// wave has CHUNK pieces of w on their way at once, the first ones before anything else happens.
// FEW: x comes as it is, at most 16384 elements; every workgroup puts it into 8 bits for itself, in LDS, while its first weights arrive: the 2 x m x k
// bytes come from the caches, and one launch and a round trip of x through memory are saved.  x is requested BEFORE the weights: loads return in order, and
// behind the weights' 8 pieces the whole preparation came after them (one row, 10240 x 4096: 12.7 us so, 3.3 TB/s; 16.6 with x behind the weights; 13.7 in two launches).
constexpr int I8_ROW_WAVES = 8, I8_CHUNK = 8, I8_FEW = 16384;

// a barrier for LDS only: loads that are on their way to registers stay on their way
GGQ_DEV void i8_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int DT, bool FEW>
__global__ __launch_bounds__(I8_ROW_WAVES * 64) void linear_i8_rows(const I8Args a)
{
    constexpr uint32_t VECS = I8_FEW / 8 / (I8_ROW_WAVES * 64);             // vectors of 8 elements of x per lane
    __shared__ i32x4 partial[I8_ROW_WAVES][64];
    __shared__ uint32_t top_[16];                                           // per row: the largest magnitude's bits,
    __shared__ double to_[16];                                              // 127 / it,
    __shared__ float scale_[16];                                            // it / 127
    extern __shared__ __attribute__((aligned(16))) uint8_t xs[];            // FEW: rows of 8-bit x, `pitch` bytes apart (an odd number of 16-byte units)
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, c = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t n0 = blockIdx.x * 16u;
    const uint32_t wr = n0 + r < a.n ? n0 + r : a.n - 1u, xr = r < a.m ? r : a.m - 1u;
    const GGQ_GLOBAL uint8_t* w = (GGQ_GLOBAL const uint8_t*)a.wq + (uint64_t)wr * a.w_stride;
    const uint32_t steps = (a.k + 63u) / 64u, pitch = steps * 64u + 16u;
    RowRaw<DT> raw[VECS];
    const uint32_t per_row = a.k / 8u, vecs = FEW ? a.m * per_row : 0u;     // FEW: rows of whole vectors, one behind the other
    if constexpr (FEW) {
#pragma unroll
        for (uint32_t j = 0; j < VECS; j++) raw[j] = row_raw<DT, false>(a.xq, (threadIdx.x + j * (I8_ROW_WAVES * 64)) * 8u, vecs * 8u);
        asm volatile("" ::: "memory");
    }
    i32x4 wa[I8_CHUNK];
    auto load = [&](uint32_t s0) {                                          // pieces s0, s0 + 8, ...; past the end: the start of the row, against zeros of x
#pragma unroll
        for (int i = 0; i < I8_CHUNK; i++) {
            const uint32_t k = (s0 + (uint32_t)(i * I8_ROW_WAVES)) * 64u + c * 16u;
            wa[i] = *(const GGQ_GLOBAL i32x4*)(k < a.k ? w + k : w);
        }
    };
    load(wave);
    if constexpr (FEW) {
        if (threadIdx.x < 16) top_[threadIdx.x] = 0;
        for (uint32_t i = threadIdx.x; i < a.m * 8u; i += I8_ROW_WAVES * 64) {               // zeros behind a row's end: at most 56 bytes
            const uint32_t at = a.k + (i & 7u) * 8u;
            if (at < steps * 64u) *reinterpret_cast<u32x2*>(xs + (i >> 3) * pitch + at) = u32x2{0, 0};
        }
        i8_barrier();
        float v[8];
#pragma unroll
        for (uint32_t j = 0; j < VECS; j++) {
            const uint32_t at = threadIdx.x + j * (I8_ROW_WAVES * 64);
            row_unpack<DT>(raw[j], v);
            uint32_t top = 0;
#pragma unroll
            for (int q = 0; q < 8; q++) top = umax(top, __builtin_bit_cast(uint32_t, v[q]) & 0x7FFFFFFFu);
            if (at < vecs) atomicMax(&top_[at / per_row], top);
        }
        i8_barrier();
        if (threadIdx.x < a.m) {
            double to;
            float scale;
            row_scale(top_[threadIdx.x], to, scale);
            to_[threadIdx.x] = to;
            scale_[threadIdx.x] = scale;
        }
        i8_barrier();
#pragma unroll
        for (uint32_t j = 0; j < VECS; j++) {
            const uint32_t at = threadIdx.x + j * (I8_ROW_WAVES * 64);
            if (at < vecs) {
                const uint32_t row = at / per_row;
                const double to = to_[row];
                row_unpack<DT>(raw[j], v);
#pragma unroll
                for (int q = 0; q < 8; q++) v[q] = to == 0.0 ? 0.0f : v[q];
                *reinterpret_cast<u32x2*>(xs + row * pitch + (at - row * per_row) * 8u) = row_quant8(v, to);
            }
        }
        i8_barrier();
    }
    i32x4 acc{0, 0, 0, 0};
    for (uint32_t s0 = wave; s0 < steps; s0 += I8_ROW_WAVES * I8_CHUNK) {
        if (s0 != wave) load(s0);
        i32x4 xb[I8_CHUNK];
#pragma unroll
        for (int i = 0; i < I8_CHUNK; i++) {
            const uint32_t k = (s0 + (uint32_t)(i * I8_ROW_WAVES)) * 64u + c * 16u;
            if constexpr (FEW) xb[i] = k < steps * 64u ? *reinterpret_cast<const i32x4*>(xs + xr * pitch + k) : i32x4{0, 0, 0, 0};
            else xb[i] = *(const GGQ_GLOBAL i32x4*)(k < a.k ? (GGQ_GLOBAL const uint8_t*)a.xq + (uint64_t)xr * a.x_stride + k : (const GGQ_GLOBAL uint8_t*)I8_ZEROS);
        }
#pragma unroll
        for (int i = 0; i < I8_CHUNK; i++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa[i], xb[i], acc, 0, 0, 0);
    }
    partial[wave][lane] = acc;
    __syncthreads();
    if (wave != 0) return;
    for (int v = 1; v < I8_ROW_WAVES; v++) acc += partial[v][lane];
    if (r >= a.m) return;
    const float sx = FEW ? scale_[r] : a.x_scale[r];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t nc = n0 + 4u * c + (uint32_t)i;
        if (nc < a.n) i8_store<DT>(a.y, (uint64_t)r * a.n + nc, (float)acc[i] * (sx * a.w_scale[nc]) + i8_bias<DT>(a.bias, nc));
    }
}

}  // namespace ggq
