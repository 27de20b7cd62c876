"""What a transformer block does to its rows between two linears, in one pass over memory (include/ggq.h ``ggq_block_norm``, csrc/ggq_rows.hpp):

    r = stream + gate * [post_weight * N_post(branch)]            the residual sum, with the gate and the norm behind the block
    y = (N(r) * weight + bias) * (1 + scale) + shift              the norm in front of the next block, modulated

The models that the reference loads run these as separate torch operations around ``GGMLOps.Linear`` (ops.py:242-244; the layer norm itself through
``GGMLOps.LayerNorm``, ops.py:262-266).  Here r stays in fp32 registers between the sum and the norm.  ``quantize=True`` returns y as 8-bit rows with a
scale each, ready for ``int8.linear_int8``.

As the fused linears do, the call raises GGQUnsupported for what the kernel does not take (CPU tensors, other types, a recording autograd, torch.func's transforms); the caller
keeps its torch operations then.
"""
import ctypes
import struct

import torch

from . import _native
from .dequant import GGQUnsupported, _DEVICE_OK, _OUT_CODE, _cur_device, _device_served, _is_compiling, _forward_ad, _raw_stream, _transform_stack, _transformed, dequantize_tensor, is_quantized

NORMS = {None: 0, "none": 0, "rms": 1, "layer": 2}
MAX_DIM = 32768                    # elements of a row: they live in the registers or the LDS of one workgroup
_PACK = struct.Struct("@16Q3I3if4x").pack         # ggq_norm_desc in one step: a ctypes structure costs 3 us more per call to fill
_call = None


def _bind():
    global _call
    fn = _native.lib()["ggq_block_norm"]            # a function object of its own: the argument is the descriptor's bytes
    fn.argtypes, fn.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_int
    _call = fn
    return _call


def _plain(t):
    """t without its subclass -- GGMLTensor's attributes go with it, so a patched one is refused."""
    if type(t) is torch.Tensor:
        return t
    if getattr(t, "patches", None):
        raise GGQUnsupported("LoRA-patched parameter: needs the reference's get_weight")
    return t.as_subclass(torch.Tensor)


def _on_gpu(x, what):
    """x as a plain tensor on a served GPU, of a type that the row kernels take."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _OUT_CODE:
        raise GGQUnsupported(f"{what}: fp16 / bf16 / fp32 tensors on the GPU")
    index = x.device.index
    if not (_DEVICE_OK.get(index) or _device_served(index)):
        raise GGQUnsupported(f"cuda:{index} is not a gfx950 device")
    return _plain(x)


def _refuse_grad(what, *tensors, packed=()):
    """Before anything asks a tensor for its memory: inside vmap it has none.  (packed: integers, which require no grad.)"""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise GGQUnsupported(f"{what}: autograd is recording -- torch's operations build the graph")
    if (_transform_stack() is not None or _forward_ad._current_level >= 0) and _transformed(*tensors, *packed):
        raise GGQUnsupported(f"{what}: inside a torch.func transform or forward-mode autograd -- torch's operations carry it on")


def _vector(v, dim, dtype, device, what):
    """A parameter of `dim` values as (tensor, is fp32)."""
    if is_quantized(v) and not getattr(v, "patches", None):
        v = dequantize_tensor(v, torch.float32)
    v = _plain(v)
    if v.device != device or v.numel() != dim:
        raise GGQUnsupported(f"block_norm: {what} holds {v.numel()} values on {v.device}, rows have {dim} on {device}")
    if v.dtype is not dtype and v.dtype is not torch.float32:
        v = v.float()
    return v.contiguous(), v.dtype is torch.float32


def _per_sample(v, lead, dim, dtype, device, what, vectors):
    """A modulation vector per sample as (tensor, stride between vectors, vectors so far or its own, is fp32).  v's leading dimensions are the stream's, or the
    first of them followed by ones."""
    v = _plain(v)
    shape = v.shape
    if v.device != device or not shape or shape[-1] != dim:
        raise GGQUnsupported(f"block_norm: {what} of shape {tuple(shape)} on {v.device} for rows of {dim} on {device}")
    if v.dtype is not dtype and v.dtype is not torch.float32:
        v = v.float()
    if not (len(lead) == 2 and len(shape) == 3 and shape[1] == 1 and shape[0] == lead[0] and v.stride(2) == 1):      # the usual (batch, 1, dim): no view to make
        own = list(shape[:-1])
        while own and own[-1] == 1:
            own.pop()
        if own != list(lead[:len(own)]):
            raise GGQUnsupported(f"block_norm: {what} of shape {tuple(shape)} does not follow the stream's leading dimensions {tuple(lead)}")
        v = v.reshape(-1, dim)                      # a view where the vectors are one stride apart (a chunk of a modulation linear's output)
        if v.stride(1) != 1:
            v = v.contiguous()
    n = v.shape[0]
    if n <= 1:
        return v, 0, vectors, v.dtype is torch.float32
    if vectors not in (1, n):
        raise GGQUnsupported(f"block_norm: gate, scale and shift of {vectors} and {n} vectors: give them for the same rows")
    return v, v.stride(0), n, v.dtype is torch.float32


def _rows_per_vector(rows, vectors):
    """Rows that share a modulation vector, in the descriptor's 32 bits.  With one vector for all (stride 0) any number does: vector after vector is the same."""
    per = max(rows // vectors, 1)
    if per >> 32:
        if vectors > 1:
            raise GGQUnsupported(f"block_norm: {per} rows for each modulation vector, fewer than 2^32")
        per = (1 << 32) - 1
    return per


def _block_norm(stream, branch, gate, post_norm, post_weight, norm, weight, bias, scale, shift, eps, quantize):
    _refuse_grad("block_norm", stream, branch, gate, post_weight, weight, bias, scale, shift)
    stream = _on_gpu(stream, "block_norm")
    if stream.dim() == 0 or norm not in NORMS or post_norm not in NORMS:
        raise GGQUnsupported(f"block_norm: rows of a tensor, and norms of {sorted(k for k in NORMS if k)} or None")
    kind, post_kind = NORMS[norm], NORMS[post_norm]
    if branch is None and (gate is not None or post_kind or post_weight is not None):
        raise GGQUnsupported("block_norm: gate and post_norm act on branch, which is not given")
    if post_weight is not None and not post_kind:
        raise GGQUnsupported("block_norm: post_weight belongs to post_norm, which is not given")
    if not kind and (weight is not None or bias is not None or scale is not None or shift is not None):
        raise GGQUnsupported("block_norm: weight, bias, scale and shift belong to norm, which is not given")
    if not kind and branch is None and not quantize:
        raise GGQUnsupported("block_norm: nothing to compute")
    device, dtype, lead, dim = stream.device, stream.dtype, stream.shape[:-1], stream.shape[-1]
    if not 1 <= dim <= MAX_DIM:
        raise GGQUnsupported(f"block_norm: rows of 1 ... {MAX_DIM} elements")
    rows = stream.numel() // dim
    out = stream
    stream = stream if stream.is_contiguous() else stream.contiguous()
    flags = at_branch = at_out = at_post = at_weight = at_bias = at_gate = at_scale = at_shift = at_y = at_y_scale = gate_stride = scale_stride = shift_stride = y_stride = 0
    if branch is not None:
        branch = _plain(branch)
        if branch.shape != stream.shape or branch.dtype is not dtype or branch.device != device:
            raise GGQUnsupported(f"block_norm: branch {tuple(branch.shape)} {branch.dtype} is not like the stream {tuple(stream.shape)} {dtype}")
        branch = branch if branch.is_contiguous() else branch.contiguous()
        at_branch = branch.data_ptr()
    if post_weight is not None:
        post_weight, is32 = _vector(post_weight, dim, dtype, device, "post_weight")
        at_post, flags = post_weight.data_ptr(), 1 if is32 else 0
    if weight is not None:
        weight, is32 = _vector(weight, dim, dtype, device, "weight")
        at_weight, flags = weight.data_ptr(), flags | (4 if is32 else 0)
    if bias is not None:
        bias, is32 = _vector(bias, dim, dtype, device, "bias")
        at_bias, flags = bias.data_ptr(), flags | (8 if is32 else 0)
    vectors = 1                                     # vectors per parameter, where one of them has more than one
    if gate is not None:
        gate, gate_stride, vectors, is32 = _per_sample(gate, lead, dim, dtype, device, "gate", vectors)
        at_gate, flags = gate.data_ptr(), flags | (2 if is32 else 0)
    if scale is not None:
        scale, scale_stride, vectors, is32 = _per_sample(scale, lead, dim, dtype, device, "scale", vectors)
        at_scale, flags = scale.data_ptr(), flags | (16 if is32 else 0)
    if shift is not None:
        shift, shift_stride, vectors, is32 = _per_sample(shift, lead, dim, dtype, device, "shift", vectors)
        at_shift, flags = shift.data_ptr(), flags | (32 if is32 else 0)
    if branch is not None:
        out = torch.empty_like(stream)
        at_out = out.data_ptr()
    y = y_scale = None
    if quantize:
        y_stride = (dim + 15) // 16 * 16
        y = torch.empty((*lead, y_stride), dtype=torch.int8, device=device)
        y_scale = torch.empty(lead, dtype=torch.float32, device=device)
        at_y, at_y_scale = y.data_ptr(), y_scale.data_ptr()
        y = y[..., :dim] if y_stride != dim else y
    elif kind:
        y = torch.empty_like(stream)
        at_y = y.data_ptr()
    if rows:
        index = device.index
        call = _call or _bind()
        desc = _PACK(stream.data_ptr(), at_branch, at_out, at_y, at_y_scale, at_post, at_gate, at_weight, at_bias, at_scale, at_shift,
                     rows, gate_stride, scale_stride, shift_stride, y_stride, dim, (rows // vectors or 1) if rows < 1 << 32 else _rows_per_vector(rows, vectors), flags, _OUT_CODE[dtype], kind, post_kind, eps)
        if _cur_device() != index:
            with torch.cuda.device(index):
                rc = call(desc, _raw_stream(index))
        else:
            rc = call(desc, _raw_stream(index))
        if rc == _native.GGQ_ERR_ARG:
            raise GGQUnsupported("shape outside what ggq_block_norm takes")
        if rc:
            _native.check(rc, "ggq_block_norm")
    return out, ((y, y_scale) if quantize else y)


def block_norm(stream, branch=None, *, gate=None, post_norm=None, post_weight=None, norm="rms", weight=None, bias=None, scale=None, shift=None, eps=1e-6, quantize=False):
    """-> (r, y), see the module's formulas.

    stream, branch: (..., dim), fp16 / bf16 / fp32, on the GPU.  Without ``branch`` r is ``stream`` itself.  ``norm`` / ``post_norm``: "rms", "layer" or None;
    with ``norm=None`` y is None (the last block), or with ``quantize`` the 8-bit form of r.  ``weight``, ``bias``, ``post_weight``: dim values, fp32 or the
    stream's type (GGUF norm weights are fp32).  ``gate``, ``scale``, ``shift``: one vector for all rows, or one per sample -- shape (batch, dim),
    (batch, 1, dim), or the stream's own -- and may be chunks of one modulation linear's output.
    ``quantize=True``: y is (q, q_scale), q int8 like the stream with rows 16 bytes apart, y ~ q * q_scale[..., None]; a row with an infinity or a NaN gets
    q = 0 and scale NaN.  r and y are rounded once, from fp32."""
    if _is_compiling():
        return _eager(stream, branch, gate, post_norm, post_weight, norm, weight, bias, scale, shift, eps, quantize)
    return _block_norm(stream, branch, gate, post_norm, post_weight, norm, weight, bias, scale, shift, eps, quantize)


# while torch.compile traces, the launch is a graph break: nothing in it can be traced
_eager = torch.compiler.disable(_block_norm)
