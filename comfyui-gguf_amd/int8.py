"""Rows in 8 bits, and the product of 8-bit integers with a scale per token and per output channel (include/ggq.h ``ggq_quantize_rows`` /
``ggq_linear_int8``, csrc/ggq_rows.hpp, csrc/ggq_int8.hpp):

    scale_i = max|x_i| / 127,   q_i = rint(127 x_i / max|x_i|)                       (half to even; the same for the rows of a weight)
    y_ij = (sum_k q_ik w_jk) * x_scale_i * w_scale_j + bias_j                        (the sum exact in int32, the rest in fp32)

Where ``GGMLOps.Linear`` (ops.py:242-244) sees many tokens, the fused linears hand over to unpack + a library product in 16 bits (fused.linear_mfma); this
is the path at twice the matrix rate for a user who keeps a weight in 8 bits.  It is never chosen by itself: 8-bit activations are another
result.  ``ops.GGMLInt8Linear`` is the layer.
"""
import torch

from . import _native
from .dequant import GGQUnsupported, _DEVICE_OK, _OUT_CODE, _cur_device, _device_served, _is_compiling, _raw_stream
from .norms import MAX_DIM, _on_gpu, _plain, _refuse_grad

MAX_K = 131071                     # |sum| <= 128 * 128 * k stays below 2^31
FEW = 16384                        # elements of x up to which (and 16 rows) one launch does both: the kernels' I8_FEW
FEW_ROWS = 16 * ((1 << 23) - 1)    # ... and fewer rows of the weight than this: a workgroup of 512 threads for 16 of them, 2^32 threads a launch
_quantize_call = _linear_call = _few_call = None


def _bind():
    global _quantize_call, _linear_call, _few_call
    L = _native.lib()
    _quantize_call, _linear_call, _few_call = L.ggq_quantize_rows, L.ggq_linear_int8, L.ggq_linear_int8_few


def _launch(call, name, device, *args):
    index = device.index
    if _cur_device() != index:
        with torch.cuda.device(index):
            rc = call(*args, _raw_stream(index))
    else:
        rc = call(*args, _raw_stream(index))
    if rc == _native.GGQ_ERR_ARG:
        raise GGQUnsupported(f"shape outside what {name} takes")
    if rc:
        _native.check(rc, name)


def _pad16(k):
    return (k + 15) // 16 * 16


def _quantize(x):
    """(rows x padded columns int8, zeros behind the last column; scales) of a 2-D x."""
    if _quantize_call is None:
        _bind()
    m, k = x.shape
    x = x if x.is_contiguous() else x.contiguous()
    q = torch.empty((m, _pad16(k)), dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    if m:
        _launch(_quantize_call, "ggq_quantize_rows", x.device, x.data_ptr(), m, k, q.data_ptr(), q.shape[1], scale.data_ptr(), _OUT_CODE[x.dtype])
    return q, scale


def quantize_rows(x):
    """-> (q, scale): q int8 of x's shape with rows a multiple of 16 bytes apart, scale fp32 of x's leading dimensions; x ~ q * scale[..., None].
    x: (..., k) fp16 / bf16 / fp32 on the GPU, 1 <= k <= 32768.  A row of zeros has scale 0; a row with an infinity or a NaN has q = 0 and scale NaN."""
    if _is_compiling():
        return _eager_quantize(x)
    return _quantize_rows(x)


def _quantize_rows(x):
    _refuse_grad("quantize_rows", x)
    x = _on_gpu(x, "quantize_rows")
    if x.dim() == 0 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise GGQUnsupported(f"quantize_rows: rows of 1 ... {MAX_DIM} elements")
    lead, k = x.shape[:-1], x.shape[-1]
    q, scale = _quantize(x.reshape(-1, k))
    q = q.view(*lead, q.shape[1])
    return (q if q.shape[-1] == k else q[..., :k]), scale.view(lead)


def _rows8(q, what, zero_padded):
    """A 2-D int8 matrix as the kernels read it: rows a multiple of 16 bytes apart, 16-byte aligned, every row readable up to a multiple of 16 columns
    (zeros there if `zero_padded`, which only a copy can promise).  A tensor laid out by quantize_rows is taken as it is, another one is copied."""
    q = _plain(q)
    n, k = q.shape
    k16 = _pad16(k)
    ok = (q.stride(1) == 1 or k == 1) and q.stride(0) % 16 == 0 and q.stride(0) >= k16 and q.data_ptr() % 16 == 0 and not (zero_padded and k != k16)
    if ok and k != k16:                             # the last row's padding has to be there too
        ok = q.untyped_storage().nbytes() - q.storage_offset() >= (n - 1) * q.stride(0) + k16
    if not ok:
        p = torch.zeros((n, k16), dtype=torch.int8, device=q.device)
        p[:, :k] = q
        q = p
    return q


def _linear_int8(x, weight, weight_scale, bias, x_scale, out_dtype):
    if not isinstance(weight, torch.Tensor) or weight.dtype is not torch.int8 or weight.dim() != 2 or not weight.is_cuda:
        raise GGQUnsupported("linear_int8: weight is an int8 matrix (rows x columns) on the GPU")
    n, k = weight.shape
    device = weight.device
    if not 1 <= k <= MAX_K:
        raise GGQUnsupported(f"linear_int8: 1 ... {MAX_K} columns")
    if not (_DEVICE_OK.get(device.index) or _device_served(device.index)):
        raise GGQUnsupported(f"{device} is not a gfx950 device")
    if not isinstance(weight_scale, torch.Tensor) or weight_scale.dtype is not torch.float32 or weight_scale.numel() != n or weight_scale.device != device:
        raise GGQUnsupported(f"linear_int8: weight_scale is {n} fp32 values on {device}")
    if x.dtype is torch.int8:
        if x_scale is None or out_dtype not in _OUT_CODE:
            raise GGQUnsupported("linear_int8: 8-bit rows come with x_scale and out_dtype (fp16 / bf16 / fp32)")
        if x.device != device or x_scale.device != device or x_scale.dtype is not torch.float32 or x_scale.shape != x.shape[:-1]:
            raise GGQUnsupported("linear_int8: x_scale is one fp32 value per row of x, on the weight's device")
    else:
        if x_scale is not None:
            raise GGQUnsupported("linear_int8: x_scale belongs to 8-bit rows; x holds " + str(x.dtype))
        x = _on_gpu(x, "linear_int8")
        out_dtype = x.dtype if out_dtype is None else out_dtype
        if out_dtype not in _OUT_CODE:
            raise GGQUnsupported("linear_int8: results in fp16 / bf16 / fp32")
        if x.device != device or k > MAX_DIM:
            raise GGQUnsupported(f"linear_int8: x on {x.device}, the weight on {device}; rows of at most {MAX_DIM} elements are quantized")
    _refuse_grad("linear_int8", x, x_scale, weight_scale, bias, packed=(weight,))
    if x.dim() == 0 or x.shape[-1] != k:
        raise GGQUnsupported(f"linear_int8: rows of {k} elements for this weight")
    lead = x.shape[:-1]
    if bias is not None:
        bias = _plain(bias)
        if bias.numel() != n:
            raise GGQUnsupported("linear_int8: bias does not match the weight's rows")
        if bias.dtype is not out_dtype or bias.device != device or not bias.is_contiguous():
            bias = bias.to(device=device, dtype=out_dtype).contiguous()
    m = x.numel() // k
    if m >= 1 << 31 or n >= 1 << 31:
        raise GGQUnsupported("linear_int8: fewer than 2^31 rows of x and of the weight")
    y = torch.empty((*lead, n), dtype=out_dtype, device=device)
    if not m or not n:
        return y
    if _linear_call is None:
        _bind()
    weight = _rows8(weight, "weight", False)
    weight_scale = weight_scale if weight_scale.is_contiguous() else weight_scale.contiguous()
    x = _plain(x)
    if x.dtype is torch.int8:
        xq, x_scale = _rows8(x.reshape(m, k) if x.dim() != 2 else x, "x", True), x_scale.reshape(m).contiguous()
    elif m <= 16 and m * k <= FEW and k % 8 == 0 and out_dtype is x.dtype and n < FEW_ROWS:
        if not x.is_contiguous() or x.data_ptr() & 15:
            x = x.clone(memory_format=torch.contiguous_format)
        _launch(_few_call, "ggq_linear_int8_few", device, x.data_ptr(), m, weight.data_ptr(), weight.stride(0), weight_scale.data_ptr(), n, k,
                None if bias is None else bias.data_ptr(), y.data_ptr(), _OUT_CODE[out_dtype])
        return y
    else:
        xq, x_scale = _quantize(x.reshape(m, k))
    _launch(_linear_call, "ggq_linear_int8", device, xq.data_ptr(), xq.stride(0), x_scale.data_ptr(), m, weight.data_ptr(), weight.stride(0), weight_scale.data_ptr(), n, k,
            None if bias is None else bias.data_ptr(), y.data_ptr(), _OUT_CODE[out_dtype])
    return y


def linear_int8(x, weight, weight_scale, bias=None, *, x_scale=None, out_dtype=None):
    """``F.linear`` on 8-bit integers, see the module's formulas.

    x: (..., k) fp16 / bf16 / fp32 (put into 8 bits row by row), or int8 with ``x_scale`` (the leading dimensions of x, fp32) and ``out_dtype``.
    weight: int8 (n, k), weight_scale: fp32 (n,) -- what ``quantize_rows`` makes of a weight.  Rows of either that are not a multiple of 16 bytes apart, or
    x rows in 8 bits whose k is no multiple of 16, are copied on every call.  The result has ``out_dtype`` (x's type unless given); a bias of
    another type is rounded to it."""
    if _is_compiling():
        return _eager_linear(x, weight, weight_scale, bias, x_scale, out_dtype)
    return _linear_int8(x, weight, weight_scale, bias, x_scale, out_dtype)


# while torch.compile traces, the launches are a graph break: nothing in them can be traced
_eager_quantize, _eager_linear = torch.compiler.disable(_quantize_rows), torch.compiler.disable(_linear_int8)
