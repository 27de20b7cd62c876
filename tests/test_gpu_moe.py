"""moe.route / moe.moe_experts / moe.moe_layer (include/ggq.h) on an MI355X, against the formulas in 64 bits on the ORACLE's weights.

Tolerance, with u = 2^-24, e half a step of the activations' type: a projection of K terms is within K u sum|w x| of its exact value (the bound of
test_gpu_linear.py).  With dg, du the gate's and up's errors, the hidden value h = act(g) u is off by |u| |act'| dg + |act(g)| du (|act'| <= 1.13) plus 16 u |h| (1 + |g|)
for exp, reciprocal and products; kept in two parts it loses a step of the second part: e^2 |h| (and 2^-35 absolute in fp16).  y collects share * (ff u sum|wd h| + sum|wd| dh),
32 u more of sum|share wd h| for the sums over waves and experts, and its own half step."""
import numpy as np
import pytest
import torch

import oracle
from test_gpu_linear import ALL, _dense_weight

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


class Stack:
    """A packed stack of expert weights and its oracle values [experts, rows, cols] in 64 bits."""

    def __init__(self, pkg, name, shape, kind, seed, mode="signed", shrink=1.0):
        q = pkg.qtypes.Q[name]
        blocks = pkg.synth.make_tensor_bytes(q, shape, seed=seed, mode=mode)
        if shrink != 1.0:                                       # smaller scales: sums of a size that the hidden type holds
            ts = pkg.qtypes.block_geometry(q)[1]
            b = blocks.reshape(-1, ts)
            for off in pkg.qtypes.SCALE_FIELDS[q]:
                d = b[:, off:off + 2].copy().view(np.float16) * np.float16(shrink)
                b[:, off:off + 2] = d.view(np.uint8).reshape(-1, 2)
            blocks = b.reshape(-1)
        self.tensor = pkg.ops.GGMLTensor(torch.from_numpy(blocks).to(DEV), tensor_type=q, tensor_shape=shape)
        self.dense = torch.from_numpy(_dense_weight(q, blocks, kind, shape[0] * shape[1], shape[2]).reshape(shape)).to(DEV)


def _act(g, name):
    return g * torch.sigmoid(g) if name == "silu" else 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3)))


def _want(x, ids, weights, gate, up, down, act, dtype):
    e = torch.finfo(dtype).eps / 2
    x = x.double()
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    dim, ff = gate.shape[2], gate.shape[1]
    for t in range(x.shape[0]):
        for s in range(ids.shape[1]):
            i = int(ids[t, s])
            if not 0 <= i < gate.shape[0]:
                continue
            g, u = gate[i] @ x[t], up[i] @ x[t]
            dg, du = dim * U * (gate[i].abs() @ x[t].abs()), dim * U * (up[i].abs() @ x[t].abs())
            a = _act(g, act)
            h = a * u
            dh = 1.13 * u.abs() * dg + a.abs() * du + 1.13 * dg * du + 16 * U * h.abs() * (1 + g.abs()) + e * e * h.abs() + 2.0 ** -35
            w = float(weights[t, s])
            y[t] += w * (down[i] @ h)
            mag = down[i].abs() @ h.abs()
            bound[t] += abs(w) * ((ff + 32) * U * mag + down[i].abs() @ dh)
    return y, bound


def _close(got, want, bound, dtype):
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    got, want, bound = got[fine], want[fine], bound[fine]
    tol = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    # and as a whole: half a step of every result, plus what independent roundings leave of the worst case (its 1 / 16th: they grow with the root of their number)
    e = torch.finfo(dtype).eps / 2
    assert float(err.norm()) <= e * float(want.norm()) + float(bound.norm()) / 16 + err.numel() ** 0.5 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _routes(tokens, top_k, experts, g):
    ids = torch.stack([torch.randperm(experts, device=DEV, generator=g)[:top_k] for _ in range(tokens)]).int()
    return ids, torch.rand(tokens, top_k, device=DEV, generator=g)


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_experts_in_every_format(pkg, name, kind):
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(41)
    legacy = pkg.qtypes.block_geometry(pkg.qtypes.Q[name])[0] == 32
    # tokens, experts, top_k, dim, ff: one token; a column block not filled; several blocks of columns (17, 33, 64 tokens); short last spans in the 32-element formats
    for tokens, experts, top_k, dim, ff, act in ((1, 4, 2, 256, 512, "silu"), (5, 6, 3, 512, 256, "gelu_tanh"), (17, 2, 1, 256, 256, "silu"), (64, 3, 2, 256, 256, "silu")) + (
            ((3, 3, 2, 192, 320, "silu"), (33, 2, 2, 64, 64, "silu")) if legacy else ()):
        gate, up = (Stack(pkg, name, (experts, ff, dim), kind, 50 + i, shrink=0.25) for i in range(2))
        down = Stack(pkg, name, (experts, dim, ff), kind, 52, shrink=0.25)
        x = (torch.randn(tokens, dim, device=DEV, generator=g) * 0.5).to(dtype)
        ids, weights = _routes(tokens, top_k, experts, g)
        y = pkg.moe.moe_experts(x, ids, weights, gate.tensor, up.tensor, down.tensor, activation=act)
        assert y.shape == x.shape and y.dtype == dtype
        want, bound = _want(x, ids, weights, gate.dense, up.dense, down.dense, act, dtype)
        _close(y, want, bound, dtype)
        assert torch.equal(y, pkg.moe.moe_experts(x, ids.long(), weights, gate.tensor, up.tensor, down.tensor, activation=act))       # deterministic; 64-bit ids


def _model(pkg, kind, experts=6, dim=512, ff=768, up="Q4_K", down="Q6_K", seed=60):
    return (Stack(pkg, up, (experts, ff, dim), kind, seed, shrink=0.25), Stack(pkg, up, (experts, ff, dim), kind, seed + 1, shrink=0.25),
            Stack(pkg, down, (experts, dim, ff), kind, seed + 2, shrink=0.25))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_ids_that_are_no_experts_and_experts_twice(pkg, kind):
    """Masked places add nothing, a token of masked places only is 0, whatever their weights hold; an expert twice counts twice; one expert for all tokens."""
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(43)
    gate, up, down = _model(pkg, kind)
    x = torch.randn(20, 512, device=DEV, generator=g).to(dtype)
    ids, weights = _routes(20, 4, 6, g)
    ids[0], ids[1, 2], ids[2] = -1, 6, torch.tensor([3, 3, 3, 1], device=DEV)
    ids[3], ids[4, 0], ids[5] = 2 ** 31 - 1, -2 ** 31, 5
    weights[0], weights[1, 2] = float("nan"), float("inf")
    y = pkg.moe.moe_experts(x, ids, weights, gate.tensor, up.tensor, down.tensor)
    want, bound = _want(x, ids, weights, gate.dense, up.dense, down.dense, "silu", dtype)
    _close(y, want, bound, dtype)
    assert not bool(y[0].any()) and not bool(y[3].any())
    big = ids.long()
    big[3] = 2 ** 32 + 1                                        # no expert in 64 bits either, whatever its low half says
    assert torch.equal(pkg.moe.moe_experts(x, big, weights, gate.tensor, up.tensor, down.tensor), y)
    none = torch.full_like(ids, -1)
    assert not bool(pkg.moe.moe_experts(x, none, weights, gate.tensor, up.tensor, down.tensor).any())
    one = torch.full((20, 1), 4, device=DEV)
    y = pkg.moe.moe_experts(x, one, weights[:, 1:2], gate.tensor, up.tensor, down.tensor)
    want, bound = _want(x, one, weights[:, 1:2], gate.dense, up.dense, down.dense, "silu", dtype)
    _close(y, want, bound, dtype)
    # tokens do not see each other: an infinity in one leaves the others as they were
    x2 = x.clone()
    x2[7] = float("inf")
    y2 = pkg.moe.moe_experts(x2, one, weights[:, 1:2], gate.tensor, up.tensor, down.tensor)
    others = torch.arange(20, device=DEV) != 7
    assert torch.equal(y2[others].nan_to_num(12345), y[others].nan_to_num(12345)) and not bool(y2[7].isfinite().any())
    assert pkg.moe.moe_experts(x[:0], ids[:0], weights[:0], gate.tensor, up.tensor, down.tensor).shape == (0, 512)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,experts", [(64, 64), (40, 33), (64, 5), (17, 64), (9, 3)])
def test_all_tokens_on_one_expert(pkg, kind, tokens, experts):
    """Far more tokens on one expert than evenly spread choices give (the kernels are picked for those): every block of 16 columns, in the registers or not; beside it
    an expert with one token, and many tiles per workgroup."""
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(51)
    gate, up, down = _model(pkg, kind, experts=experts, dim=256, ff=512, up="Q5_0", down="Q3_K")
    x = (torch.randn(tokens, 256, device=DEV, generator=g) * 0.5).to(dtype)
    ids = torch.full((tokens, 2), experts - 1, device=DEV, dtype=torch.int32)
    ids[:, 1] = -1
    ids[3, 1] = 1
    weights = torch.rand(tokens, 2, device=DEV, generator=g)
    y = pkg.moe.moe_experts(x, ids, weights, gate.tensor, up.tensor, down.tensor)
    want, bound = _want(x, ids, weights, gate.dense, up.dense, down.dense, "silu", dtype)
    _close(y, want, bound, dtype)


def test_hidden_values_of_all_sizes(pkg):
    """bf16: hidden values from 1e-30 to 1e8 keep their 16 bits (the two parts share no range).  fp16: small hidden values do not fall into the subnormals."""
    g = torch.Generator(device=DEV)
    g.manual_seed(45)
    for kind, sizes in (("bf16", (1e-15, 1e-4, 1.0, 3e3)), ("f16", (1e-2, 1.0))):
        gate, up, down = _model(pkg, kind)
        ids, weights = _routes(2, 2, 6, g)
        for size in sizes:
            x = (torch.randn(2, 512, device=DEV, generator=g) * size).to(DT[kind])
            y = pkg.moe.moe_experts(x, ids, weights, gate.tensor, up.tensor, down.tensor)
            want, bound = _want(x, ids, weights, gate.dense, up.dense, down.dense, "silu", DT[kind])
            _close(y, want, bound, DT[kind])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("wide", [False, True])
def test_router_against_64_bits(pkg, kind, wide):
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(47)
    for tokens, experts, top_k, dim, renormalize in ((1, 8, 2, 4096, True), (64, 64, 8, 2048, False), (3, 1, 1, 8, True), (200, 512, 16, 264, True), (5, 70, 7, 2432, False)):
        x = torch.randn(tokens, dim, device=DEV, generator=g).to(dtype)
        w = (torch.randn(experts, dim, device=DEV, generator=g) * (2 / dim ** 0.5)).to(torch.float32 if wide else dtype)
        ids, weights = pkg.moe.route(x, w, top_k, renormalize=renormalize)
        assert ids.dtype == torch.int32 and weights.dtype == torch.float32 and ids.shape == weights.shape == (tokens, top_k)
        scores = x.double() @ w.double().T
        p, order = torch.sort(torch.softmax(scores, -1), dim=-1, descending=True, stable=True)
        # scores closer than fp64's error (dim 2^-53 sum|x w|) may come in either order; none are in these inputs
        gap = (torch.sort(scores, dim=-1, descending=True)[0].diff(dim=-1).abs()[:, :top_k] if experts > 1 else torch.ones(1, 1, device=DEV))
        assert float(gap.min()) > dim * 2.0 ** -53 * float((x.double().abs() @ w.double().abs().T).max())
        assert torch.equal(ids.long(), order[:, :top_k])
        want = p[:, :top_k] / (p[:, :top_k].sum(-1, keepdim=True) if renormalize else 1)
        # exp of a difference of scores rounded to fp32 (|difference| u), exp, reciprocal and the sum of up to 512 terms
        assert bool(((weights.double() - want).abs() <= want * (600 + 40) * U).all())


def test_router_ties_and_nans(pkg):
    x = torch.ones(2, 16, device=DEV, dtype=torch.bfloat16)
    w = torch.zeros(9, 16, device=DEV, dtype=torch.bfloat16)
    w[3], w[7], w[5] = 1, 1, 2
    ids, weights = pkg.moe.route(x, w, 6)
    assert ids.tolist() == [[5, 3, 7, 0, 1, 2]] * 2            # equal scores: the lower expert first
    w[5, 0] = float("nan")
    ids, weights = pkg.moe.route(x, w, 9, renormalize=False)
    assert ids.tolist() == [[3, 7, 0, 1, 2, 4, 6, 8, 5]] * 2 and bool(weights.isnan().all())
    x[1] = float("nan")
    ids, weights = pkg.moe.route(x, w[:4], 2)
    assert ids.tolist() == [[3, 0], [0, 1]] and bool(weights[1].isnan().all()) and abs(float(weights[0].sum()) - 1) < 1e-6
    x[0] = 0
    ids, weights = pkg.moe.route(x[:1], w[:4], 4)
    assert ids.tolist() == [[0, 1, 2, 3]] and weights.tolist() == [[0.25] * 4]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_the_whole_layer_and_its_module(pkg, kind):
    """moe_layer is route + moe_experts; the module is moe_layer, and beyond 64 tokens or under autograd the experts one by one, with gradients."""
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(49)
    gate, up, down = _model(pkg, kind, up="Q5_K", down="Q8_0")
    router = torch.randn(6, 512, device=DEV, generator=g) * 0.1
    x = (torch.randn(2, 9, 512, device=DEV, generator=g) * 0.5).to(dtype)
    ids, weights = pkg.moe.route(x.view(18, 512), router, 2)
    y = pkg.moe.moe_layer(x, router, gate.tensor, up.tensor, down.tensor, top_k=2)
    assert torch.equal(y.view(18, 512), pkg.moe.moe_experts(x.view(18, 512), ids, weights, gate.tensor, up.tensor, down.tensor))
    layer = pkg.ops.GGMLMoE(router, gate.tensor, up.tensor, down.tensor, top_k=2)
    assert torch.equal(layer(x), y)
    many = (torch.randn(70, 512, device=DEV, generator=g) * 0.5).to(dtype)
    with pytest.raises(pkg.dequant.GGQUnsupported):
        pkg.moe.moe_layer(many, router, gate.tensor, up.tensor, down.tensor, top_k=2)
    slow, fast = layer(many), layer(many[:64])
    # the one-by-one path rounds gate, up, act, hidden and output of each expert to the activations' type: a few steps of the largest magnitudes
    assert float((slow[:64].double() - fast.double()).norm() / fast.double().norm()) < 8 * torch.finfo(dtype).eps
    # gradients of the one-by-one path: against the formula's in 64 bits, and that against a difference.  (A plain sum: the square of these outputs has
    # gradients beyond fp16's 65504.)
    x = x.clone().requires_grad_()
    layer(x).float().sum().backward()

    def formula(v):
        top, chosen = torch.sort(torch.softmax(v @ router.double().T, -1), dim=-1, descending=True, stable=True)
        top, chosen = top[:, :2] / top[:, :2].sum(-1, keepdim=True), chosen[:, :2]
        h = _act(torch.einsum("td,tsfd->tsf", v, gate.dense[chosen]), "silu") * torch.einsum("td,tsfd->tsf", v, up.dense[chosen])
        return (torch.einsum("tsf,tsdf->tsd", h, down.dense[chosen]) * top[:, :, None]).sum()

    v = x.detach().double().view(18, 512).requires_grad_()
    want, = torch.autograd.grad(formula(v), v)
    step = torch.randn(18, 512, device=DEV, generator=g).double() * 1e-5
    diff = float(formula(v.detach() + step) - formula(v.detach() - step)) / 2
    assert abs(diff - float((want * step).sum())) <= 1e-6 * float((want * step).abs().sum())        # third derivatives times 1e-15, far below
    assert float((x.grad.double().view(18, 512) - want).norm() / want.norm()) < 16 * torch.finfo(dtype).eps


def test_refusals_on_the_gpu(pkg):
    M, no = pkg.moe, pkg.dequant.GGQUnsupported
    gate, up, down = (s.tensor for s in _model(pkg, "f16"))
    x = torch.zeros(3, 512, device=DEV, dtype=torch.float16)
    ids, weights = torch.zeros(3, 2, device=DEV, dtype=torch.int32), torch.zeros(3, 2, device=DEV)
    G = pkg.ops.GGMLTensor
    plain = gate.as_subclass(torch.Tensor)
    for args in ((x.float(), ids, weights, gate, up, down), (x.cpu(), ids, weights, gate, up, down), (x[:, :256], ids, weights, gate, up, down), (x, ids[:2], weights, gate, up, down),
                 (x, ids.float(), weights, gate, up, down), (x, ids, weights, gate, down, down), (x, ids, weights, gate, up, gate), (x, ids, weights, plain, up, down),
                 (x, ids, weights, G(plain, tensor_type=gate.tensor_type, tensor_shape=(6 * 768, 512)), up, down), (x, ids[:, :0], weights[:, :0], gate, up, down),
                 (x, ids, weights, G(plain[:-144], tensor_type=gate.tensor_type, tensor_shape=(6, 768, 512)), up, down),
                 (x.repeat(30, 1), ids.repeat(30, 1), weights.repeat(30, 1), gate, up, down), (x, ids.repeat(1, 9), weights.repeat(1, 9), gate, up, down)):
        with pytest.raises(no):
            M.moe_experts(*args)
    with pytest.raises(no):
        M.moe_experts(x, ids, weights, gate, up, down, activation="relu")
    with pytest.raises(no, match="autograd"):
        M.moe_experts(x.clone().requires_grad_(), ids, weights, gate, up, down)
    r = torch.zeros(6, 512, device=DEV, dtype=torch.float16)
    for args in ((x, r, 7), (x, r, 0), (x, r[:, :256], 2), (x.float(), r, 2), (x, r.bfloat16(), 2), (x[:, :4].contiguous(), r[:, :4].contiguous(), 2), (x, r.repeat(100, 1), 2)):
        with pytest.raises(no):
            M.route(*args)
