// ggq_rows.hip -- C ABI over ggq_rows.hpp: residual + gate + norms + modulation of a block's rows, and the 8-bit form of rows.
#include "ggq_rows.hpp"
#include "ggq_host.hpp"
#include "../../include/ggq.h"

namespace {

using namespace ggq;

typedef void (*rows_fn)(const RowArgs);

// rows of up to WAVES * 64 * NV * 8 elements: 24576 at most (8 vectors per lane on 8 waves would not fit the registers)
#define GGQ_ROW_NV(DT, W) {block_norm<DT, W, 1>, block_norm<DT, W, 2>, block_norm<DT, W, 3>, block_norm<DT, W, 4>, block_norm<DT, W, 6>, block_norm<DT, W, (W == 8 ? 6 : 8)>}
#define GGQ_ROW_DT(DT) {GGQ_ROW_NV(DT, 1), GGQ_ROW_NV(DT, 4), GGQ_ROW_NV(DT, 8)}
const rows_fn ROWS[3][3][6] = {GGQ_ROW_DT(OUT_F16), GGQ_ROW_DT(OUT_BF16), GGQ_ROW_DT(OUT_F32)};
constexpr uint32_t NVS[6] = {1, 2, 3, 4, 6, 8}, WAVES[3] = {1, 4, 8};

int launch_rows(const RowArgs& a, int dtype, hipStream_t s)
{
    const uint64_t span = a.y_scale != nullptr ? a.y_stride : a.dim;       // elements a row's lanes have to cover (8-bit rows: their zero padding too)
    const uint32_t vecs = (uint32_t)((span + 7) / 8);
    int w = 0;
    if (a.rows < 2048u || vecs > 64u * 8u) w = vecs > 4u * 64u * 8u || (a.rows < 256u && vecs > 64u) ? 2 : 1;
    int nv = 0;
    while (nv < 6 && (uint64_t)NVS[nv] * WAVES[w] * 64u < vecs) nv++;
    if (nv == 6 || (w == 2 && nv == 5)) return GGQ_ERR_ARG;
    const uint64_t grid = w == 0 ? (a.rows + 3) / 4 : a.rows;
    if (grid > 0x7FFFFFFFull) return GGQ_ERR_ARG;
    hipLaunchKernelGGL(ROWS[dtype][w][nv], dim3((uint32_t)grid), dim3(w == 0 ? 256u : WAVES[w] * 64u), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}

bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" int ggq_block_norm(const ggq_norm_desc* d, void* hip_stream)
{
    if (!d) return GGQ_ERR_ARG;
    if (d->dtype < 0 || d->dtype > 2 || d->norm < NORM_NONE || d->norm > NORM_LAYER || d->post_norm < NORM_NONE || d->post_norm > NORM_LAYER) return GGQ_ERR_ARG;
    if (d->rows == 0) return GGQ_OK;
    if (d->dim == 0 || d->rows_per_mod == 0 || !d->stream || (d->branch && !d->stream_out) || (!d->branch && !d->y)) return GGQ_ERR_ARG;
    if (d->y_scale && (!d->y || d->y_stride < d->dim || d->y_stride % 16 != 0)) return GGQ_ERR_ARG;
    const uintptr_t eb = d->dtype == GGQ_F32 ? 4 : 2;
    if (!aligned_to(d->stream, eb) || !aligned_to(d->branch, eb) || !aligned_to(d->stream_out, eb) || !aligned_to(d->y, d->y_scale ? 16 : eb)) return GGQ_ERR_ALIGN;
    const void* params[6] = {d->post_weight, d->gate, d->weight, d->bias, d->scale, d->shift};
    for (int i = 0; i < 6; i++)
        if (!aligned_to(params[i], (d->params_f32 >> i) & 1u ? 4 : eb)) return GGQ_ERR_ALIGN;
    auto b = [](const void* p) { return static_cast<const uint8_t*>(p); };
    RowArgs a{b(d->stream), b(d->branch), static_cast<uint8_t*>(d->stream_out), static_cast<uint8_t*>(d->y), d->y_scale, b(d->post_weight), b(d->gate), b(d->weight),
              b(d->bias), b(d->scale), b(d->shift), d->rows, d->gate_stride, d->scale_stride, d->shift_stride, d->y_stride, d->dim, d->rows_per_mod, d->params_f32,
              d->norm, d->post_norm, d->eps};
    return launch_rows(a, d->dtype, static_cast<hipStream_t>(hip_stream));
}

extern "C" int ggq_quantize_rows(const void* x, uint64_t rows, uint32_t cols, void* q, uint64_t q_stride, float* scale, int dtype, void* hip_stream)
{
    if (dtype < 0 || dtype > 2) return GGQ_ERR_ARG;
    if (rows == 0) return GGQ_OK;
    if (!x || !q || !scale || cols == 0 || q_stride < cols || q_stride % 16 != 0) return GGQ_ERR_ARG;
    if (!aligned_to(x, dtype == GGQ_F32 ? 4 : 2) || !aligned_to(q, 16)) return GGQ_ERR_ALIGN;
    RowArgs a{};
    a.stream = static_cast<const uint8_t*>(x);
    a.y = static_cast<uint8_t*>(q);
    a.y_scale = scale;
    a.rows = rows;
    a.y_stride = q_stride;
    a.dim = cols;
    a.rows_per_mod = 1;
    return launch_rows(a, dtype, static_cast<hipStream_t>(hip_stream));
}
