"""A mixture-of-experts layer for a few tokens, straight from packed expert weights (include/ggq.h ``ggq_moe_route`` / ``ggq_moe_experts``,
csrc/ggq_moe.hpp):

    p = softmax(x Wr^T);  e_1 ... e_k = the k largest, equal ones to the lower index;  p_s /= sum_s p_s if ``renormalize``
    y = sum_s p_s Wd[e_s] (act(Wg[e_s] x) * (Wu[e_s] x))

The reference's ``GGMLOps.Linear`` (ops.py:242-244) would unpack a dense weight per expert and projection.  Here the packed bytes of the chosen experts
are read once, for all tokens that chose them; no dense weight exists.  Expert weights are GGUF stacks: a byte tensor with ``tensor_type`` and a
``tensor_shape`` of three dimensions (experts, rows, columns), as GGMLTensor has.  ``ops.GGMLMoE`` is the layer; it takes over with unpacked
experts where this module raises GGQUnsupported (more tokens, CPU tensors, a recording autograd).
"""
import ctypes

import torch

from . import _native
from .dequant import GGQUnsupported, _HIP_TABLE, _OUT_CODE, _cur_device, _is_compiling, _qtype_key, _raw_stream
from .norms import _on_gpu, _plain, _refuse_grad

MAX_TOKENS, MAX_TOP_K, MAX_EXPERTS, MAX_WIDTH = 64, 16, 512, 1 << 24
ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}
_route_call = _experts_call = _workspace = None


def _bind():
    global _route_call, _experts_call, _workspace
    L = _native.lib()
    _route_call, _experts_call, _workspace = L.ggq_moe_route, L.ggq_moe_experts, L.ggq_moe_workspace


def _rows16(x, what, f32=False):
    """A 2-D fp16 / bf16 matrix (``f32``: fp32 too) of contiguous rows, 16-byte aligned."""
    x = _on_gpu(x, what)
    if x.dim() != 2 or (x.dtype is torch.float32 and not f32):
        raise GGQUnsupported(f"{what}: fp16 / bf16 matrices")
    if not x.is_contiguous() or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _with_device(device, call, name, *args):
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


def _route(x, router, top_k, renormalize):
    _refuse_grad("moe.route", x, router)
    return _run_route(_rows16(x, "moe.route"), router, top_k, renormalize)


def _run_route(x, router, top_k, renormalize):
    router = _rows16(router, "moe.route", True)
    tokens, dim = x.shape
    experts = router.shape[0]
    if router.shape[1] != dim or router.dtype not in (x.dtype, torch.float32) or router.device != x.device:
        raise GGQUnsupported(f"moe.route: a router (experts x {dim}) of {x.dtype} or fp32 on {x.device}")
    if dim % 8 or dim == 0 or not 1 <= experts <= MAX_EXPERTS or not 1 <= top_k <= min(MAX_TOP_K, experts) or tokens > 65535:
        raise GGQUnsupported(f"moe.route: at most 65535 rows of a multiple of 8 elements, 1 ... {MAX_EXPERTS} experts, 1 ... {MAX_TOP_K} of them per token")
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=x.device)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=x.device)
    if tokens:
        if _route_call is None:
            _bind()
        size = tokens * experts * 8 if experts > 16 else 0           # ggq_moe_route_workspace()
        scratch = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        _with_device(x.device, _route_call, "ggq_moe_route", x.data_ptr(), router.data_ptr(), tokens, dim, experts, top_k, int(bool(renormalize)), ids.data_ptr(),
                     weights.data_ptr(), _OUT_CODE[x.dtype], _OUT_CODE[router.dtype], scratch.data_ptr() if size else None, size)
    return ids, weights


def _stack(w, what, device):
    """(type id, shape, packed bytes) of a stack of expert weights."""
    ent = _HIP_TABLE.get(_qtype_key(getattr(w, "tensor_type", None)))
    if ent is None:
        raise GGQUnsupported(f"moe_experts: no kernel for {what} of type {getattr(getattr(w, 'tensor_type', None), 'name', getattr(w, 'tensor_type', None))!r}")
    if getattr(w, "patches", None):
        raise GGQUnsupported(f"moe_experts: {what} is LoRA-patched: needs the reference's get_weight")
    shape = tuple(int(d) for d in getattr(w, "tensor_shape", ()))
    if len(shape) != 3:
        raise GGQUnsupported(f"moe_experts: {what} of shape (experts, rows, columns)")
    qid, block, size = ent
    w = _plain(w)
    if w.device != device or w.dtype is not torch.uint8 or not w.is_contiguous() or w.data_ptr() & 15:
        raise GGQUnsupported(f"moe_experts: packed {what} must be a contiguous, 16-byte aligned byte tensor on {device}")
    if shape[2] % (256 if block == 256 else 64) or w.numel() != shape[0] * shape[1] * shape[2] // block * size:
        raise GGQUnsupported(f"moe_experts: {what} rows of a multiple of {256 if block == 256 else 64} elements, and {w.numel()} bytes for the shape {shape}")
    return qid, shape, w


def _stacks(x, gate, up, down, activation):
    """What is refused of x (rows as _rows16 gives them) and of the stacks, whatever the routes -> (experts, ff, their type ids, their bytes)."""
    if activation not in ACTIVATIONS:
        raise GGQUnsupported(f"moe_experts: activations {sorted(ACTIVATIONS)}")
    tokens, dim = x.shape
    if tokens > MAX_TOKENS:
        raise GGQUnsupported(f"moe_experts: at most {MAX_TOKENS} tokens, got {tokens}")
    (gate_id, gate_shape, gate), (up_id, up_shape, up), (down_id, down_shape, down) = (_stack(w, name, x.device) for w, name in ((gate, "gate"), (up, "up"), (down, "down")))
    experts, ff = up_shape[0], up_shape[1]
    if gate_id != up_id or gate_shape != up_shape or up_shape[2] != dim or down_shape != (experts, dim, ff):
        raise GGQUnsupported(f"moe_experts: gate and up of one type and shape (experts, ff, {dim}), down (experts, {dim}, ff); got {gate_shape}, {up_shape}, {down_shape}")
    if not 1 <= experts <= MAX_EXPERTS or not 1 <= ff <= MAX_WIDTH or not 1 <= dim <= MAX_WIDTH:
        raise GGQUnsupported(f"moe_experts: 1 ... {MAX_EXPERTS} experts, widths of 1 ... {MAX_WIDTH}")
    return experts, ff, up_id, down_id, gate, up, down


def _experts(x, ids, weights, gate, up, down, activation):
    _refuse_grad("moe_experts", x, weights, packed=(ids, gate, up, down))
    x = _rows16(x, "moe_experts")
    return _run(x, ids, weights, _stacks(x, gate, up, down, activation), activation)


def _run(x, ids, weights, stacks, activation):
    experts, ff, up_id, down_id, gate, up, down = stacks
    (tokens, dim), device = x.shape, x.device
    if ids.dim() != 2 or ids.shape != weights.shape or ids.shape[0] != tokens or ids.device != device or weights.device != device or ids.dtype not in (torch.int32, torch.int64):
        raise GGQUnsupported("moe_experts: ids (int32 / int64) and weights of shape (tokens, top_k) on x's device")
    top_k = ids.shape[1]
    if not 1 <= top_k <= MAX_TOP_K:
        raise GGQUnsupported(f"moe_experts: 1 ... {MAX_TOP_K} experts per token")
    y = torch.empty_like(x)
    if not tokens:
        return y
    if ids.dtype is torch.int64:
        ids = ids.clamp(-1, experts).int()          # what is no expert stays none in 32 bits
    ids, weights = ids.contiguous(), weights.to(torch.float32).contiguous()
    if _experts_call is None:
        _bind()
    size = int(_workspace(tokens, top_k, dim, ff))
    scratch = torch.empty(size, dtype=torch.uint8, device=device)
    d = _native.ggq_moe_desc(x.data_ptr(), ids.data_ptr(), weights.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), y.data_ptr(), scratch.data_ptr(), size,
                             tokens, top_k, experts, dim, ff, up_id, down_id, ACTIVATIONS[activation], _OUT_CODE[x.dtype])
    _with_device(device, _experts_call, "ggq_moe_experts", ctypes.byref(d))
    return y


def _layer(x, router, gate, up, down, top_k, renormalize, activation):
    _refuse_grad("moe_layer", x, router, packed=(gate, up, down))
    lead = x.shape
    if not lead or not lead[-1]:
        raise GGQUnsupported(f"moe_layer: rows of a tensor, got shape {tuple(lead)}")
    if x.numel() // lead[-1] > MAX_TOKENS:
        raise GGQUnsupported(f"moe_layer: at most {MAX_TOKENS} tokens, got {x.numel() // lead[-1]}")
    x = _rows16(x.reshape(-1, lead[-1]) if x.dim() != 2 else x, "moe_layer")
    stacks = _stacks(x, gate, up, down, activation)              # refusals come before the router is launched
    if router.shape[0] != stacks[0]:
        raise GGQUnsupported(f"moe_layer: a router of {router.shape[0]} experts, stacks of {stacks[0]}")
    ids, weights = _run_route(x, router, top_k, renormalize)
    return _run(x, ids, weights, stacks, activation).reshape(lead)


# while torch.compile traces, the launches are a graph break: nothing in them can be traced
_eager_route, _eager_experts, _eager_layer = (torch.compiler.disable(f) for f in (_route, _experts, _layer))


def route(x, router, top_k, *, renormalize=True):
    """-> (ids int32, weights fp32), both (tokens, top_k), the largest probability first.  x: (tokens, dim) fp16 / bf16 on the GPU, router: (experts, dim) of x's type or
    fp32 (as GGUF files keep it), dim % 8 == 0.  Scores are fp64; a NaN score comes last, and all of its token's weights are NaN."""
    return (_eager_route if _is_compiling() else _route)(x, router, top_k, renormalize)


def moe_experts(x, ids, weights, gate, up, down, *, activation="silu"):
    """y (tokens, dim) for routes that the caller has: x (tokens, dim) fp16 / bf16 on the GPU, at most 64 tokens; ids (tokens, top_k) int32 / int64, weights
    like ids.  An id that is no expert adds nothing (a padded place, a masked token: y is 0 where all are); the same expert twice counts twice.
    gate, up: packed stacks (experts, ff, dim) of one type; down: (experts, dim, ff); columns a multiple of 256, or of 64 for the 32-element blocks."""
    return (_eager_experts if _is_compiling() else _experts)(x, ids, weights, gate, up, down, activation)


def moe_layer(x, router, gate, up, down, *, top_k, renormalize=True, activation="silu"):
    """``route`` and ``moe_experts`` for x of shape (..., dim), at most 64 tokens in all."""
    return (_eager_layer if _is_compiling() else _layer)(x, router, gate, up, down, top_k, renormalize, activation)
