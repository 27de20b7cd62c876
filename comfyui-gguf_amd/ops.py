"""The boundary types the hot path is called through, in the smallest form that needs no
ComfyUI import: ``GGMLTensor`` (reference ops.py:44-91), the ``get_weight`` / ``cast_bias_weight``
call chain of ``GGMLLayer`` (reference ops.py:166-211) and the five layer types that call it
(``GGMLOps.Linear / Conv2d / Embedding / LayerNorm / GroupNorm``, reference ops.py:227-271).

In a real ComfyUI install the reference's own classes stay in place (they are "reused as-is",
SURVEY.md section 2 rows 7-8) and only the dequant functions underneath them are replaced by
install.py.  These stand-ins exist so the path can be driven end to end -- tests, smoke, bench --
on a machine that has neither ComfyUI nor the reference checked out (the GPU box).  LoRA patches,
state-dict hooks and VRAM accounting belong to the reference's control plane and are not
re-implemented here.
"""
import torch

from .dequant import _is_compiling, _transform_stack, _transforms, dequantize_tensor, is_quantized


class GGMLTensor(torch.Tensor):
    """Packed GGUF bytes + the logical view: ``tensor_type`` (ggml type id), ``tensor_shape``."""

    def __new__(cls, data, *, tensor_type, tensor_shape, patches=None):
        t = torch.Tensor._make_subclass(cls, data, False)
        t.tensor_type = tensor_type
        t.tensor_shape = torch.Size(tensor_shape)
        t.patches = list(patches or [])
        return t

    def _carry(self, new):
        new.tensor_type = getattr(self, "tensor_type", None)
        new.tensor_shape = getattr(self, "tensor_shape", new.size())
        new.patches = list(getattr(self, "patches", []))
        return new

    def to(self, *args, **kwargs):                 # ops.py:57-62: the attrs survive a device move
        return self._carry(super().to(*args, **kwargs))

    def clone(self, *args, **kwargs):              # ops.py:64-68
        return self

    def detach(self, *args, **kwargs):
        return self

    def copy_(self, *args, **kwargs):              # ops.py:70-75: a failing in-place copy is logged, not raised
        try:
            return super().copy_(*args, **kwargs)
        except Exception as e:                     # noqa: BLE001 -- the reference swallows everything here
            import logging
            logging.warning(f"ignoring 'copy_' on tensor: {e}")

    def new_empty(self, size, *args, **kwargs):    # ops.py:77-85: same type and attrs, logical shape = the new size
        return GGMLTensor(super().new_empty(size, *args, **kwargs), tensor_type=getattr(self, "tensor_type", None),
                          tensor_shape=size, patches=getattr(self, "patches", []))

    @property
    def shape(self):                               # ops.py:87-91: the LOGICAL shape
        return getattr(self, "tensor_shape", self.size())


class GGMLLayer(torch.nn.Module):
    """What the reference's ``GGMLLayer`` does on the hot path (ops.py:93-211): keep the packed weight / bias, and on
    every forward re-dequantize them (no caching, ops.py:166-191) on the device the input lives on.  LoRA patches,
    state-dict hooks and VRAM accounting are the reference's control plane and are not restated."""

    dequant_dtype = None                           # ops.py:98; set by the loader nodes (nodes.py:152-157)
    _dequantize = staticmethod(dequantize_tensor)  # what get_weight calls; resident.DenseCache may be put here

    def __init__(self, weight, bias=None):
        super().__init__()
        self.weight = weight
        self.bias = bias

    def is_ggml_quantized(self):                   # ops.py:103-108
        return is_quantized(self.weight) or is_quantized(self.bias)

    def get_weight(self, tensor, dtype):           # ops.py:166-181 without the LoRA branch
        if tensor is None:
            return None
        weight = self._dequantize(tensor, dtype, self.dequant_dtype)
        if isinstance(weight, GGMLTensor):         # ops.py:180-181: never hand the subclass on
            weight = weight.as_subclass(torch.Tensor)
        return weight

    def cast_bias_weight(self, input=None, dtype=None, device=None, bias_dtype=None):   # ops.py:194-211
        if input is not None:
            if dtype is None:
                dtype = getattr(input, "dtype", torch.float32)
            if bias_dtype is None:
                bias_dtype = dtype
            if device is None:
                device = input.device
        bias = None
        if self.bias is not None:
            bias = self.get_weight(self.bias.to(device), dtype)
            bias = bias.to(device=device, dtype=bias_dtype)
        weight = self.get_weight(self.weight.to(device), dtype)
        weight = weight.to(device=device, dtype=dtype)
        return weight, bias


class GGMLLinear(GGMLLayer):
    """``GGMLOps.Linear`` (ops.py:227-244).  ``fuse_small_m`` / ``fuse_mfma_max_m`` (off in this stand-in; install()'s default over the reference's class, fused.py): inputs of at most four rows /
    of at most that many rows go through a fused dequantize + linear kernel instead of dequantize-then-F.linear."""

    fuse_small_m = False
    fuse_mfma_max_m = 0                            # opt-in: inputs of up to this many rows go through fused.linear_mfma

    def forward(self, input):
        if (self.fuse_small_m or self.fuse_mfma_max_m) and is_quantized(self.weight):
            from .fused import linear_auto                 # the policy of install()'s default (fused.py): GEMV / 16-row / 32-row MFMA kernel by rows of x
            from .dequant import GGQUnsupported
            try:
                return linear_auto(input, self.weight, self.bias, self.dequant_dtype, input.device, self.fuse_small_m, self.fuse_mfma_max_m)
            except GGQUnsupported:
                pass
        if not self.is_ggml_quantized():
            return torch.nn.functional.linear(input, self.weight.to(input.dtype), None if self.bias is None else self.bias.to(input.dtype))
        weight, bias = self.cast_bias_weight(input)
        return torch.nn.functional.linear(input, weight, bias)


class GGMLEmbedding(GGMLLayer):
    """``GGMLOps.Embedding`` (ops.py:251-260): the (possibly quantized) table is dequantized whole, then indexed.  As in the
    reference, a table stored in fp16 / bf16 is used in its own dtype and the result cast to ``out_dtype``."""

    def __init__(self, weight, padding_idx=None):
        super().__init__(weight, None)
        self.padding_idx = padding_idx

    gather_rows = True                             # quantized table on the GPU: unpack only the rows asked for (bit-identical)

    def forward(self, input, out_dtype=None):
        output_dtype = out_dtype
        if self.weight.dtype == torch.float16 or self.weight.dtype == torch.bfloat16:
            out_dtype = None
        if self.gather_rows and is_quantized(self.weight) and input.is_cuda and not getattr(self.weight, "patches", None):
            from .dequant import GGQUnsupported, dequantize_rows
            try:
                # cast_bias_weight(self, dtype=None) falls back to getattr(self, "dtype", float32) (ops.py:196-197): same here
                table_dtype = out_dtype if out_dtype is not None else getattr(self, "dtype", torch.float32)
                rows = dequantize_rows(self.weight.to(input.device), input, table_dtype, self.dequant_dtype)
                return rows.to(dtype=output_dtype)
            except GGQUnsupported:
                pass
        weight, _ = self.cast_bias_weight(self, device=input.device, dtype=out_dtype)
        return torch.nn.functional.embedding(input, weight, self.padding_idx).to(dtype=output_dtype)


class GGMLConv2d(GGMLLayer):
    """``GGMLOps.Conv2d`` (ops.py:246-249); the packed weight's logical shape is (out, in, kh, kw)."""

    def __init__(self, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
        super().__init__(weight, bias)
        self.stride, self.padding, self.dilation, self.groups = stride, padding, dilation, groups

    def forward(self, input):
        weight, bias = self.cast_bias_weight(input)
        return torch.nn.functional.conv2d(input, weight, bias, self.stride, self.padding, self.dilation, self.groups)


class GGMLLayerNorm(GGMLLayer):
    """``GGMLOps.LayerNorm`` (ops.py:262-266)."""

    def __init__(self, normalized_shape, weight, bias=None, eps=1e-5):
        super().__init__(weight, bias)
        self.normalized_shape, self.eps = tuple(normalized_shape), eps

    def forward(self, input):
        if self.weight is None:
            return torch.nn.functional.layer_norm(input, self.normalized_shape, None, None, self.eps)
        weight, bias = self.cast_bias_weight(input)
        return torch.nn.functional.layer_norm(input, self.normalized_shape, weight, bias, self.eps)


class GGMLGroupNorm(GGMLLayer):
    """``GGMLOps.GroupNorm`` (ops.py:268-271)."""

    def __init__(self, num_groups, weight, bias=None, eps=1e-5):
        super().__init__(weight, bias)
        self.num_groups, self.eps = num_groups, eps

    def forward(self, input):
        weight, bias = self.cast_bias_weight(input)
        return torch.nn.functional.group_norm(input, self.num_groups, weight, bias, self.eps)


class GGMLInt8Linear(torch.nn.Module):
    """A linear layer whose weight is kept in 8 bits with a scale per output channel (int8.linear_int8): made once from a quantized (or plain) weight, a
    byte per element from then on, the packed weight is not needed any more.  Activations are put into 8 bits token by token, so the result is another one
    than GGMLLinear's: nothing chooses this layer by itself.  What the kernels do not take -- CPU tensors, a recording autograd -- is computed as F.linear
    with the 8-bit weight's values."""

    def __init__(self, weight, bias=None):
        super().__init__()
        from .int8 import quantize_rows
        if getattr(weight, "patches", None) or getattr(bias, "patches", None):
            raise ValueError("GGMLInt8Linear: the weight or bias is LoRA-patched; apply the patches first")
        dense = dequantize_tensor(weight, torch.float16) if is_quantized(weight) else weight
        dense = dense if type(dense) is torch.Tensor else dense.as_subclass(torch.Tensor)
        q, scale = quantize_rows(dense.detach())
        if bias is not None:
            bias = dequantize_tensor(bias, torch.float32) if is_quantized(bias) else bias
            bias = (bias if type(bias) is torch.Tensor else bias.as_subclass(torch.Tensor)).detach()
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", bias)

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype is not torch.float32:         # .half() and the like cast the bias only: 16-bit scales are other weights
            self.weight_scale = scale.to(self.weight_scale.device)
        if not self.weight.is_meta:
            from .int8 import _rows8
            laid_out = _rows8(self.weight, "weight", False)      # a move packs rows of odd widths: apart again, so that no call has to copy them
            if laid_out is not self.weight:
                self.weight = laid_out[:, :self.weight.shape[1]]
        return self

    def forward(self, input):
        from .dequant import GGQUnsupported
        from .int8 import linear_int8
        weight, scale, bias = (t if t is None or t.device == input.device else t.to(input.device) for t in (self.weight, self.weight_scale, self.bias))
        try:
            return linear_int8(input, weight, scale, bias)
        except GGQUnsupported:
            weight = (weight.float() * scale[:, None]).to(input.dtype)
            return torch.nn.functional.linear(input, weight, None if bias is None else bias.to(input.dtype))


class GGMLMoE(torch.nn.Module):
    """A mixture-of-experts layer over packed expert stacks (moe.moe_layer): ``router`` (experts, dim); ``gate``, ``up`` (experts, ff, dim) and ``down``
    (experts, dim, ff) are GGMLTensors of three dimensions, on any device: they come to the input's for the call, as a GGMLLayer's weight does.  What the fused
    kernels do not take -- more than 64 tokens, CPU tensors, a recording autograd, torch.func's transforms -- runs one expert after the other: get_weight + F.linear,
    the reference's way (ops.py:242-244), rounded to the input's type after each.  (Packed weights are unpacked on the GPU alone.)"""

    def __init__(self, router, gate, up, down, top_k, renormalize=True, activation="silu"):
        super().__init__()
        from .moe import ACTIVATIONS
        if activation not in ACTIVATIONS:
            raise ValueError(f"GGMLMoE: activations {sorted(ACTIVATIONS)}, got {activation!r}")
        if getattr(router, "patches", None):
            raise ValueError("GGMLMoE: the router is LoRA-patched; apply the patches first")
        router = dequantize_tensor(router, torch.float32) if is_quantized(router) else router
        if not 1 <= top_k <= router.shape[0]:
            raise ValueError(f"GGMLMoE: {top_k} of {router.shape[0]} experts")
        if not router.shape[0] == gate.shape[0] == up.shape[0] == down.shape[0]:
            raise ValueError(f"GGMLMoE: a router of {router.shape[0]} experts, stacks of {gate.shape[0]}, {up.shape[0]} and {down.shape[0]}")
        self.router = (router if type(router) is torch.Tensor else router.as_subclass(torch.Tensor)).float()      # one type for activations of any
        self.gate, self.up, self.down = gate, up, down
        self.top_k, self.renormalize, self.activation = top_k, renormalize, activation

    def forward(self, input):
        from .dequant import GGQUnsupported
        from .moe import MAX_TOKENS, moe_layer
        stacks = self.router, self.gate, self.up, self.down
        with torch._C.DisableTorchFunctionSubclass():            # (a GGMLTensor's device asked for the long way is 4 us)
            away = input.is_cuda and input.numel() <= MAX_TOKENS * input.shape[-1] and any(w.device != input.device for w in stacks)
        if away:
            stacks = [w.to(input.device) for w in stacks]        # weights that are kept elsewhere come over for the call, as GGMLLayer's do (ops.py:209)
        try:
            return moe_layer(input, *stacks, top_k=self.top_k, renormalize=self.renormalize, activation=self.activation)
        except GGQUnsupported:
            return self._one_by_one(input)

    def _one_by_one(self, input):
        x = input.reshape(-1, input.shape[-1])
        ids, share = self._route(x)
        inside = not _is_compiling() and any(_transforms())      # of torch.func's transforms: no value can be looked at
        y = self._sum_of_experts(x, ids, share, inside, inside and x.dtype is torch.float16)
        if x.dtype is torch.float16 and not inside and not bool(y.isfinite().all()):
            y = self._sum_of_experts(x, ids, share, inside, True)
        return y.to(input.dtype).reshape(input.shape)

    def _route(self, x):
        """moe.route, in torch where it refuses: scores in 64 bits, as which of two close ones is larger decides which experts run."""
        from .dequant import GGQUnsupported
        from .moe import route
        router = self.router if self.router.device == x.device else self.router.to(x.device)
        try:
            return route(x, router, self.top_k, renormalize=self.renormalize)
        except GGQUnsupported:
            scores = x.double() @ router.double().t()
            ids = torch.sort(scores, dim=-1, descending=True, stable=True)[1][:, :self.top_k]
            share = torch.softmax(scores, -1).gather(-1, ids)
            return ids, (share / share.sum(-1, keepdim=True) if self.renormalize else share).float()

    def _sum_of_experts(self, x, ids, share, every, in_range):
        """The experts' results, weighted and added in 32 bits: each for its own tokens, or for all of them (every).  in_range: fp16 hidden values beyond 65504 are divided by a
        power of two per row -- |act(left)| <= |left| -- which is 1 for the other rows: those have the same bits with and without."""
        act = torch.nn.functional.silu if self.activation == "silu" else (lambda v: torch.nn.functional.gelu(v, approximate="tanh"))

        def one(expert, rows, part):
            gate, up, down = (self._expert(w, expert, x.dtype, x.device) for w in (self.gate, self.up, self.down))
            left, right = torch.nn.functional.linear(rows, gate), torch.nn.functional.linear(rows, up)
            if in_range:
                reach = left.detach().abs().amax(-1, keepdim=True).float() * right.detach().abs().amax(-1, keepdim=True).float()
                down_by = torch.exp2(torch.ceil(torch.log2(reach / 32768)).clamp_min(0))
                right, part = (right.float() / down_by).to(x.dtype), part * down_by
            return torch.nn.functional.linear(act(left) * right, down).float() * part

        y = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
        if every:
            for expert in range(self.gate.shape[0]):
                mine = ids == expert
                y = y + torch.where(mine.any(-1, keepdim=True), one(expert, x, torch.where(mine, share, 0.0).sum(-1, keepdim=True)), 0.0)
            return y
        for expert in torch.unique(ids).tolist():
            token, place = torch.nonzero(ids == expert, as_tuple=True)
            y = y.index_add(0, token, one(expert, x[token], share[token, place][:, None]))
        return y

    @staticmethod
    def _expert(stack, expert, dtype, device):
        if getattr(stack, "patches", None):
            raise ValueError("GGMLMoE: the experts are LoRA-patched; patches are not applied to a stack")
        plain = stack if type(stack) is torch.Tensor else stack.as_subclass(torch.Tensor)
        if not is_quantized(stack):
            return plain.reshape(stack.shape)[expert].to(device, dtype)
        experts, rows, cols = stack.tensor_shape
        per = plain.numel() // experts

        def unpack():
            one = plain.reshape(-1)[expert * per:(expert + 1) * per].clone()
            one = GGMLTensor(one if one.is_cuda else one.to(device), tensor_type=stack.tensor_type, tensor_shape=(rows, cols))
            dense = dequantize_tensor(one, dtype)
            return dense if dense.device == device else dense.to(device)
        if _transform_stack() is None:
            return unpack()
        with torch._C._DisableFuncTorch():               # a weight is the same inside torch.func's transforms, and has to have memory there
            return unpack()
