// ggq_rows.hip -- C ABI over ggq_rows.hpp: residual + gate + norms + modulation of a block's rows, and the 8-bit form of rows.
#include "ggq_rows.hpp"
#include "ggq_launch.hpp"
#include "../../include/ggq.h"

namespace {

using namespace ggq;

typedef void (*rows_fn)(const RowArgs, uint32_t);
typedef void (*long_fn)(const RowArgs);

// [dtype][dim % 8 != 0][a wave per row, a workgroup per row]
#define GGQ_ROW_SET(DT) {{block_norm<DT, true, false>, block_norm<DT, false, false>}, {block_norm<DT, true, true>, block_norm<DT, false, true>}}
const rows_fn ROWS[3][2][2] = {GGQ_ROW_SET(OUT_F16), GGQ_ROW_SET(OUT_BF16), GGQ_ROW_SET(OUT_F32)};
const long_fn LONG_ROWS[3] = {block_norm_long<OUT_F16>, block_norm_long<OUT_BF16>, block_norm_long<OUT_F32>};
constexpr uint32_t MAX_DIM = 32768;                                        // 128 KiB of LDS

int launch_rows(const RowArgs& a, int dtype, hipStream_t s)
{
    const uint64_t span = a.y_scale != nullptr ? a.y_stride : a.dim;       // elements a row's lanes have to cover (8-bit rows: their zero padding too)
    if (span > MAX_DIM) return GGQ_ERR_ARG;
    const uint32_t vecs = (uint32_t)((span + 7) / 8);
    if (vecs > (a.dim % 8 != 0 ? 512u : 1024u)) {
        if (!launchable(a.rows, ROW_LONG_THREADS)) return GGQ_ERR_ARG;
        static std::atomic<uint64_t> raised[3];
        hipError_t e = allow_lds(reinterpret_cast<const void*>(LONG_ROWS[dtype]), MAX_DIM * 4, raised[dtype]);
        if (e == hipSuccess) {
            hipLaunchKernelGGL(LONG_ROWS[dtype], dim3((uint32_t)a.rows), dim3(ROW_LONG_THREADS), (vecs + 1023u) / 1024u * (ROW_LONG_THREADS * 32u), s, a);
            e = hipGetLastError();
        }
        return e == hipSuccess ? GGQ_OK : hip_fail(e);
    }
    const bool solo = vecs <= 64u;
    const uint32_t waves = solo ? 1u : (vecs + 63u) / 64u;
    // as many teams as the chip holds at 16 waves per CU, each with as few rows as that leaves.  (Where dim is no multiple of 8 the registers of fp16 rows, 170 and 161, and of
    // short bf16 rows, 134, leave 8 ... 12 waves per CU: there the last teams run as a second round.)
    const uint64_t teams = 256u * 16u / waves, per = (a.rows + teams - 1) / teams;
    if (per > 0xFFFFFFFFull) return GGQ_ERR_ARG;
    const uint64_t need = (a.rows + per - 1) / per, grid = solo ? (need + 3) / 4 : need;
    hipLaunchKernelGGL(ROWS[dtype][a.dim % 8 != 0][solo ? 0 : 1], dim3((uint32_t)grid), dim3(solo ? 256u : waves * 64u), 0, s, a, (uint32_t)per);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GGQ_OK : hip_fail(e);
}

bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Whether the rows of two arrays lie on one another, in part (`same`: or wholly).  A row is read before its own place is written, other rows may not be.
bool on_one_another(const void* a, uint64_t a_row, const void* b, uint64_t b_row, uint64_t rows, bool same)
{
    if (!a || !b || (a == b && a_row == b_row && !same)) return false;
    const unsigned __int128 p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p < q + (unsigned __int128)rows * b_row && q < p + (unsigned __int128)rows * a_row;
}

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
    const uint64_t in_row = d->dim * eb, y_row = d->y_scale ? d->y_stride : in_row;
    if (on_one_another(d->y, y_row, d->stream, in_row, d->rows, d->y_scale) || on_one_another(d->y, y_row, d->branch, in_row, d->rows, d->y_scale)) return GGQ_ERR_ARG;
    if (d->branch && (on_one_another(d->stream_out, in_row, d->stream, in_row, d->rows, false) || on_one_another(d->stream_out, in_row, d->branch, in_row, d->rows, false) ||
                      on_one_another(d->y, y_row, d->stream_out, in_row, d->rows, true))) return GGQ_ERR_ARG;
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
    if (on_one_another(q, q_stride, x, (uint64_t)cols * (dtype == GGQ_F32 ? 4 : 2), rows, true)) return GGQ_ERR_ARG;
    const bool solo = q_stride <= 512u;
    const uint64_t blocks = solo ? rows / 4 + (rows % 4 != 0) : rows;
    const uint32_t threads = solo ? 256u : (uint32_t)((q_stride <= 8192u ? q_stride : 8192u) + 511u) / 512u * 64u;
    if (q_stride <= 8192u && launchable(blocks, threads)) {                // more rows than that: dealt out to the teams that fit the chip
        typedef void (*quantize_fn)(const uint8_t*, uint64_t, uint32_t, uint8_t*, uint64_t, float*);
#define GGQ_QUANTIZE(DT) {{quantize_rows<DT, true, false>, quantize_rows<DT, false, false>}, {quantize_rows<DT, true, true>, quantize_rows<DT, false, true>}}
        static const quantize_fn QUANTIZE[3][2][2] = {GGQ_QUANTIZE(OUT_F16), GGQ_QUANTIZE(OUT_BF16), GGQ_QUANTIZE(OUT_F32)};
        hipLaunchKernelGGL(QUANTIZE[dtype][cols % 8 != 0][solo ? 0 : 1], dim3((uint32_t)blocks), dim3(threads), 0, static_cast<hipStream_t>(hip_stream), static_cast<const uint8_t*>(x),
                           rows, cols, static_cast<uint8_t*>(q), q_stride, scale);
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? GGQ_OK : hip_fail(e);
    }
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
