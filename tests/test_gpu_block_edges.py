"""The block operators (norms, int8, moe and their layers) at the edges of what their documentation allows."""
import copy

import numpy as np
import pytest
import torch

from test_gpu_linear import ALL
from test_gpu_moe import DT, Stack, U, _act, _close, _want

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ---- the router

@pytest.mark.parametrize("experts", [9, 40])                    # one launch, and two
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("wide", [False, True])
def test_one_score_that_is_no_number(pkg, experts, renormalize, wide):
    """softmax over scores of which one is NaN or +inf has no number in it: all of the token's weights are NaN, also where that expert is not among the chosen."""
    g = torch.Generator(device=DEV)
    g.manual_seed(91)
    x = torch.randn(3, 64, device=DEV, generator=g).bfloat16()
    w = torch.randn(experts, 64, device=DEV, generator=g).to(torch.float32 if wide else torch.bfloat16)
    x[1, 5], x[2, 5] = 0.0, 0.0
    x[1, 6] = x[1, 7] = 1.0
    bad = w.clone()
    bad[2, 5] = float("nan")                                    # NaN times 0 is NaN too
    ids, weights = pkg.moe.route(x, bad, 6, renormalize=renormalize)
    assert bool(weights.isnan().all())
    assert not bool((ids == 2).any())                           # it comes last
    bad = w.clone()
    bad[2, 6], bad[2, 7] = float("inf"), float("-inf")          # inf - inf: one token's score only, where both meet the same sign
    ids, weights = pkg.moe.route(x[1:2], bad, 6, renormalize=renormalize)
    assert bool(weights.isnan().all()) and not bool((ids == 2).any())
    bad[2, 7] = w[2, 7]
    ids, weights = pkg.moe.route(x[1:2], bad, 6, renormalize=renormalize)          # +inf
    assert int(ids[0, 0]) == 2 and bool(weights.isnan().all())
    bad[2, 6] = float("-inf")                                   # -inf: probability 0, the others as without it
    ids, weights = pkg.moe.route(x[1:2], bad, 6, renormalize=renormalize)
    rest = torch.cat((w[:2], w[3:]))
    same, share = pkg.moe.route(x[1:2], rest, 6, renormalize=renormalize)
    assert torch.equal(ids, same + (same >= 2).int()) and bool((weights - share).abs().max() <= 2 * U)


def test_a_layer_whose_router_holds_a_nan(pkg):
    """NaN through the kernels and through the experts one by one alike."""
    g = torch.Generator(device=DEV)
    g.manual_seed(92)
    gate, up, down = (Stack(pkg, "Q8_0", s, "bf16", 3 + i, shrink=0.25).tensor for i, s in enumerate(((6, 64, 64), (6, 64, 64), (6, 64, 64))))
    router = torch.randn(6, 64, device=DEV, generator=g)
    router[4, 3] = float("nan")
    x = torch.randn(65, 64, device=DEV, generator=g).bfloat16()
    layer = pkg.ops.GGMLMoE(router, gate, up, down, top_k=2)
    assert bool(layer(x[:64]).isnan().all()) and bool(layer(x).isnan().all())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("experts", [8, 48])
@pytest.mark.parametrize("wide", [False, True])
def test_scores_that_cancel(pkg, kind, experts, wide):
    """Each expert's score is a small number beside terms of 2^24 that cancel exactly: every sum of these terms is exact in 64 bits in any order (31 bits), and in
    32 bits the small numbers are lost.  Equal scores from different columns tie to the lower expert."""
    g = np.random.default_rng(17)
    dim = 1024
    small = g.permutation(experts) // 2                         # each value twice: ties
    w = np.zeros((experts, dim // 4, 4))
    for e in range(experts):
        fours = g.permutation(dim // 4)[:8]
        w[e, fours[:4], 0], w[e, fours[4:], 0] = 4096.0, -4096.0
        w[e, fours[g.integers(8)], 1 + e % 3] = small[e] * 2.0 ** -17                        # in the same four as a large one
    x = torch.full((2, dim), 4096.0, dtype=DT[kind], device=DEV)
    x[1] = -4096.0
    router = torch.from_numpy(w.reshape(experts, dim)).to(torch.float32 if wide else DT[kind]).to(DEV)
    exact = (x.double() @ router.double().T).cpu().numpy()
    top = 8
    ids, weights = pkg.moe.route(x, router, top)
    for t in range(2):
        order = np.argsort(-exact[t], kind="stable")[:top]
        assert ids[t].tolist() == order.tolist()
        p = np.exp(exact[t][order] - exact[t][order[0]])
        assert np.abs(weights[t].cpu().numpy() / (p / p.sum()) - 1).max() <= 640 * U


def test_scores_of_products_that_32_bits_do_not_hold(pkg):
    """An fp32 router: products of 24 x 8 bits whose neighbours are equal once rounded to fp32."""
    for experts in (8, 48):
        order = np.random.default_rng(5).permutation(experts)
        w = torch.zeros(experts, 16, device=DEV)
        # 1.99 ... + e 2^-23 times 1.0078125: neighbours are 2^-23 apart, fp32 has steps of 2^-22 there
        w[:, 0] = torch.from_numpy((np.float32(1.9921875) + order.astype(np.float32) * np.float32(2.0 ** -23)).astype(np.float32)).to(DEV)
        w[:, 8] = -2.0
        x = torch.zeros(1, 16, device=DEV, dtype=torch.bfloat16)
        x[0, 0], x[0, 8] = 1.0078125, 1.0
        ids, _ = pkg.moe.route(x, w, 8)
        assert ids[0].tolist() == np.argsort(-order, kind="stable")[:8].tolist()


# ---- hidden values

@pytest.mark.parametrize("tokens,experts,top_k", [(1, 3, 2), (20, 4, 2), (64, 3, 2)])
@pytest.mark.parametrize("names", [("Q8_0", "Q8_0"), ("Q4_K", "Q6_K"), ("Q5_0", "IQ4_NL")])
def test_fp16_hidden_values_beyond_fp16(pkg, tokens, experts, top_k, names):
    """Hidden values up to 1e7 and beyond, where every result is far inside fp16; beside them tokens whose values are small, unchanged by the others.
    A hidden value above 65504 is kept to 19 bits: 2^-19 of it, weighted, joins the bound."""
    g = torch.Generator(device=DEV)
    g.manual_seed(95)
    dtype, dim, ff = torch.float16, 256, 512
    gate, up = (Stack(pkg, names[0], (experts, ff, dim), "f16", 60 + i, shrink=0.25) for i in range(2))
    down = Stack(pkg, names[1], (experts, dim, ff), "f16", 62, shrink=2.0 ** -9)
    x = torch.randn(tokens, dim, device=DEV, generator=g) * 0.5
    scale = 4000.0 / float((gate.dense[0] @ x[0].double()).abs().max())          # gate and up values of thousands
    x[::2] *= scale
    x = x.to(dtype)
    ids = torch.stack([torch.randperm(experts, device=DEV, generator=g)[:top_k] for _ in range(tokens)]).int()
    weights = torch.rand(tokens, top_k, device=DEV, generator=g)
    weights[::2] *= 2.0 ** -6
    want, bound = _want(x, ids, weights, gate.dense, up.dense, down.dense, "silu", dtype)
    most = 0.0
    for t in range(tokens):
        for s in range(top_k):
            i = int(ids[t, s])
            h = _act(gate.dense[i] @ x[t].double(), "silu") * (up.dense[i] @ x[t].double())
            most = max(most, float(h.abs().max()))
            bound[t] += 2.0 ** -19 * float(weights[t, s]) * (down.dense[i].abs() @ (h.abs() * (h.abs() > 65000)))
    assert most > 1e6 and float(want.abs().max()) < 30000
    y = pkg.moe.moe_experts(x, ids, weights, gate.tensor, up.tensor, down.tensor)
    _close(y, want, bound, dtype)
    if tokens > 1:                                              # the tokens between: bit for bit what they are without the large ones
        calm = x.clone()
        calm[::2] = 0
        assert torch.equal(pkg.moe.moe_experts(calm, ids, weights, gate.tensor, up.tensor, down.tensor)[1::2], y[1::2])


@pytest.mark.parametrize("name", ALL)
def test_fp16_hidden_values_beyond_fp16_in_every_format(pkg, name):
    """The same for the down projection's formats, with short last spans in the 32-element ones; the shares bring the results back into fp16."""
    g = torch.Generator(device=DEV)
    g.manual_seed(96)
    dtype = torch.float16
    dim, ff = (192, 320) if pkg.qtypes.block_geometry(pkg.qtypes.Q[name])[0] == 32 else (256, 768)
    gate, up = (Stack(pkg, "Q8_0", (3, ff, dim), "f16", 70 + i, shrink=0.25) for i in range(2))
    down = Stack(pkg, name, (3, dim, ff), "f16", 72, shrink=0.25)
    x = (torch.randn(5, dim, device=DEV, generator=g) * (3000.0 / (gate.dense.abs().mean() * dim ** 0.5).float())).to(dtype)
    ids = torch.tensor([[0, 1], [1, 1], [2, 0], [-1, 2], [0, 2]], device=DEV, dtype=torch.int32)
    most, bound, reach = 0.0, torch.zeros(5, dim, dtype=torch.float64, device=DEV), 0.0
    for t in range(5):
        for i in ids[t].tolist():
            if i >= 0:
                h = _act(gate.dense[i] @ x[t].double(), "silu") * (up.dense[i] @ x[t].double())
                most, reach = max(most, float(h.abs().max())), max(reach, float((down.dense[i] @ h).abs().max()))
                bound[t] += 2.0 ** -19 * (down.dense[i].abs() @ (h.abs() * (h.abs() > 65000)))
    share = 2.0 ** float(np.floor(np.log2(10000.0 / reach)))
    assert most > 1e6
    weights = torch.full((5, 2), share, device=DEV)
    want, base = _want(x, ids, weights, gate.dense, up.dense, down.dense, "silu", dtype)
    y = pkg.moe.moe_experts(x, ids, weights, gate.tensor, up.tensor, down.tensor)
    _close(y, want, base + share * bound, dtype)


def test_fp16_hidden_values_beyond_fp16_one_by_one(pkg):
    """More than 64 tokens take the experts one by one: the same hidden values, in fp16 products.  Gate, up, activation, hidden and output are rounded to fp16: a few steps
    of the largest magnitudes, as where nothing overflows.  Tokens that are in range get the bits that they get without the others."""
    g = torch.Generator(device=DEV)
    g.manual_seed(97)
    gate, up = (Stack(pkg, "Q8_0", (3, 512, 256), "f16", 60 + i, shrink=0.25) for i in range(2))
    down = Stack(pkg, "Q8_0", (3, 256, 512), "f16", 62, shrink=2.0 ** -13)
    router = torch.randn(3, 256, device=DEV, generator=g) * 0.01
    x = torch.randn(70, 256, device=DEV, generator=g)
    x = x * (3000.0 / float((gate.dense[0] @ x[0].double()).abs().max()))
    x[1::2] *= 2.0 ** -6
    x = x.half()
    layer = pkg.ops.GGMLMoE(router, gate.tensor, up.tensor, down.tensor, top_k=2)
    hidden = _act(gate.dense[0] @ x[0].double(), "silu") * (up.dense[0] @ x[0].double())
    assert float(hidden.abs().max()) > 1e6
    slow, fast = layer(x), layer(x[:64])
    assert bool(slow.isfinite().all()) and bool(fast.isfinite().all())
    assert float((slow[:64].double() - fast.double()).norm() / fast.double().norm()) < 8 * torch.finfo(torch.float16).eps
    calm = x.clone()
    calm[::2] *= 2.0 ** -6
    f = torch.nn.functional
    want, same = torch.zeros(70, 256, device=DEV), layer(calm)
    ids, p = pkg.moe.route(calm, router, 2)
    for e in range(3):
        token, place = torch.nonzero(ids == e, as_tuple=True)
        w = [s.dense[e].half() for s in (gate, up, down)]
        want = want.index_add(0, token, f.linear(f.silu(f.linear(calm[token], w[0])) * f.linear(calm[token], w[1]), w[2]).float() * p[token, place][:, None])
    assert torch.equal(same, want.half())


# ---- refusals

def _small_mixture(pkg, experts=6):
    g = torch.Generator(device=DEV)
    g.manual_seed(98)
    return (torch.randn(experts, 256, device=DEV, generator=g), *(Stack(pkg, "Q4_K", (experts, 256, 256), "f16", 80 + i, shrink=0.25).tensor for i in range(3)))


def test_the_layer_refuses_before_it_launches(pkg, monkeypatch):
    """What moe_experts refuses of the stacks, moe_layer refuses before the router has run."""
    router, gate, up, down = _small_mixture(pkg)
    x = torch.ones(3, 256, device=DEV, dtype=torch.float16)
    pkg.moe._bind()

    def launched(*args):
        raise AssertionError("the router was launched")
    monkeypatch.setattr(pkg.moe, "_route_call", launched)
    with pytest.raises(AssertionError):
        pkg.moe.moe_layer(x, router, gate, up, down, top_k=2)
    G = pkg.ops.GGMLTensor
    short = G(down.as_subclass(torch.Tensor)[:-144], tensor_type=down.tensor_type, tensor_shape=down.tensor_shape)
    patched = G(down.as_subclass(torch.Tensor), tensor_type=down.tensor_type, tensor_shape=down.tensor_shape, patches=[1])
    for stacks, kw in (((gate, up, short), {}), ((gate, up, patched), {}), ((gate, up, down.cpu()), {}), ((gate, up, gate.as_subclass(torch.Tensor)), {}), ((gate, up, down), {"activation": "relu"})):
        with pytest.raises(pkg.dequant.GGQUnsupported):
            pkg.moe.moe_layer(x, router, *stacks, top_k=2, **kw)


def test_a_router_of_other_experts_than_the_stacks(pkg):
    """Ids beyond the stacks add nothing in moe_experts; a layer whose router has more (or fewer) experts than its stacks is a mistake."""
    router, gate, up, down = _small_mixture(pkg)
    x = torch.ones(3, 256, device=DEV, dtype=torch.float16)
    for other in (router[:5], torch.cat((router, router))):
        with pytest.raises(pkg.dequant.GGQUnsupported, match="router"):
            pkg.moe.moe_layer(x, other, gate, up, down, top_k=2)
        with pytest.raises(ValueError, match="router"):
            pkg.ops.GGMLMoE(other, gate, up, down, top_k=2)


def test_the_layers_under_transforms(pkg):
    """Forward-mode gradients and vmap take the layers' torch operations: the tangent of an 8-bit linear is F.linear of the tangent, bit for bit; the calls themselves refuse."""
    from torch.autograd import forward_ad
    g = torch.Generator(device=DEV)
    g.manual_seed(99)
    no = pkg.dequant.GGQUnsupported
    layer = pkg.ops.GGMLInt8Linear(torch.randn(48, 64, device=DEV, generator=g).half(), torch.randn(48, device=DEV, generator=g).half())
    x, v = (torch.randn(3, 5, 64, device=DEV, generator=g).half() for _ in range(2))
    dense = (layer.weight.float() * layer.weight_scale[:, None]).half()
    f = torch.nn.functional
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, v)
        y = forward_ad.unpack_dual(layer(dual))
        assert torch.equal(y.primal, f.linear(x, dense, layer.bias)) and torch.equal(y.tangent, f.linear(v, dense))
        for call in (lambda: pkg.norms.block_norm(dual), lambda: pkg.norms.block_norm(x, scale=dual[0, 0]), lambda: pkg.int8.quantize_rows(dual), lambda: pkg.int8.linear_int8(x, layer.weight, layer.weight_scale, dual[0, 0, :48]),
                     lambda: pkg.moe.route(dual[0], x[1, :3], 2)):
            with pytest.raises(no, match="forward"):
                call()
        pkg.norms.block_norm(x)                                 # nothing in this one
    _, tangent = torch.func.jvp(layer, (x,), (v,))
    assert torch.equal(tangent, f.linear(v, dense))
    torch.testing.assert_close(torch.vmap(layer)(x), f.linear(x, dense, layer.bias), rtol=2.0 ** -10, atol=2.0 ** -8)          # a batched product's sums in fp32, and two roundings

    router, gate, up, down = _small_mixture(pkg)
    mix = pkg.ops.GGMLMoE(router, gate, up, down, top_k=2)
    x, v = (torch.randn(4, 3, 256, device=DEV, generator=g).half() * 0.5 for _ in range(2))
    slow = torch.stack([mix._one_by_one(t) for t in x]).double()
    near = 8 * torch.finfo(torch.float16).eps
    assert float((torch.vmap(mix)(x).double() - slow).norm() / slow.norm()) < near
    value, tangent = torch.func.jvp(mix, (x,), (v,))
    assert float((value.double() - slow).norm() / slow.norm()) < near
    leaf = x.clone().requires_grad_()
    back, = torch.autograd.grad(mix(leaf).float().sum(), leaf)
    pairs = back.double() * v.double()
    assert abs(float(tangent.double().sum() - pairs.sum())) < 16 * torch.finfo(torch.float16).eps * (float(pairs.norm()) + float(tangent.double().norm()) * 4)


@pytest.mark.parametrize("rows", [1, 20])
def test_the_fused_linears_under_transforms(pkg, rows):
    """The same for a packed linear with the fused kernels on: unpack + F.linear carries tangents and batches."""
    from torch.autograd import forward_ad
    g = torch.Generator(device=DEV)
    g.manual_seed(100)
    ops, q = pkg.ops, pkg.qtypes.Q.Q8_0
    packed = torch.from_numpy(pkg.synth.make_tensor_bytes(q, (64, 256), seed=3, mode="signed")).to(DEV)
    layer = ops.GGMLLinear(ops.GGMLTensor(packed, tensor_type=q, tensor_shape=(64, 256)))
    layer.fuse_small_m, layer.fuse_mfma_max_m = True, 256
    dense = pkg.dequant.dequantize_tensor(layer.weight, torch.float16)
    x, v = (torch.randn(rows, 256, device=DEV, generator=g).half() for _ in range(2))
    with torch.no_grad(), forward_ad.dual_level():
        y = forward_ad.unpack_dual(layer(forward_ad.make_dual(x, v)))
    f = torch.nn.functional
    assert torch.equal(y.primal, f.linear(x, dense)) and torch.equal(y.tangent, f.linear(v, dense))
    batch = torch.stack((x, v, x - v))
    got, want = torch.vmap(layer)(batch), f.linear(batch.double(), dense.double())
    assert float((got.double() - want).norm() / want.norm()) < 2 * torch.finfo(torch.float16).eps


# ---- layers that are cast, moved, copied and saved

def _int8_layer(pkg, k=200):
    g = torch.Generator(device=DEV)
    g.manual_seed(101)
    layer = pkg.ops.GGMLInt8Linear(torch.randn(40, k, device=DEV, generator=g), torch.randn(40, device=DEV, generator=g))
    x = torch.randn(6, k, device=DEV, generator=g)
    return layer, x


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_an_8_bit_layer_that_is_cast(pkg, dtype):
    """Its scales stay in 32 bits and its result that of linear_int8: only the bias is cast."""
    layer, x = _int8_layer(pkg)
    want = pkg.int8.linear_int8(x.to(dtype), layer.weight, layer.weight_scale, layer.bias)
    scale = layer.weight_scale.clone()
    for cast in (lambda m: m.to(dtype), lambda m: m.half() if dtype is torch.float16 else m.bfloat16(), lambda m: m.to(DEV, dtype), lambda m: torch.nn.Sequential(m).to(dtype)[0]):
        m = cast(copy.deepcopy(layer))
        assert m.weight_scale.dtype is torch.float32 and torch.equal(m.weight_scale, scale) and m.bias.dtype is dtype
        assert torch.equal(m(x.to(dtype)), want)


def test_an_8_bit_layer_that_is_moved_copied_and_saved(pkg, monkeypatch):
    """The layout that linear_int8 reads without a copy (rows of 200 bytes, 208 apart) survives; where it cannot, the result does."""
    layer, x = _int8_layer(pkg)
    want = layer(x)
    elsewhere = layer.cpu()
    assert elsewhere.weight.device.type == "cpu" and torch.equal(elsewhere(x.cpu()), torch.nn.functional.linear(x.cpu(), elsewhere.weight.float() * elsewhere.weight_scale[:, None], elsewhere.bias))
    back = elsewhere.to(DEV)
    copies = [back, copy.deepcopy(back), back.float()]
    loaded, _ = _int8_layer(pkg)
    loaded.weight.zero_()
    loaded.load_state_dict(back.state_dict())
    copies.append(loaded)
    made = []
    zeros = torch.zeros
    monkeypatch.setattr(pkg.int8.torch, "zeros", lambda *a, **k: made.append(a) or zeros(*a, **k))
    for m in copies:
        assert m.weight.shape == (40, 200) and m.weight.stride() == (208, 1) and m.weight.dtype is torch.int8
        assert torch.equal(m(x), want)
    assert not made                                             # nothing was copied on a call
    loaded.load_state_dict({k: v.contiguous() for k, v in back.state_dict().items()}, assign=True)
    assert torch.equal(loaded(x), want)


def test_layers_whose_weights_are_on_another_device(pkg):
    """As with GGMLLayer, weights that are kept elsewhere come to the input: the result is what it is with the weights in place, in the kernels and one by one."""
    G = pkg.ops.GGMLTensor
    router, *stacks = _small_mixture(pkg)
    away = [G(s.as_subclass(torch.Tensor).cpu(), tensor_type=s.tensor_type, tensor_shape=s.tensor_shape) for s in stacks]
    here, there = pkg.ops.GGMLMoE(router, *stacks, top_k=2), pkg.ops.GGMLMoE(router.cpu(), *away, top_k=2)
    g = torch.Generator(device=DEV)
    g.manual_seed(102)
    for tokens in (1, 64, 70):
        x = torch.randn(tokens, 256, device=DEV, generator=g).half() * 0.5
        assert torch.equal(there(x), here(x))
    leaf = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(there(leaf).float().sum(), leaf)[0], torch.autograd.grad(here(leaf).float().sum(), leaf)[0])
    layer, x = _int8_layer(pkg)
    want = layer(x)
    assert torch.equal(copy.deepcopy(layer).cpu()(x), want)
    dense = layer.weight.float() * layer.weight_scale[:, None]
    assert torch.equal(layer(x.cpu()), torch.nn.functional.linear(x.cpu(), dense.cpu(), layer.bias.cpu()))


@pytest.mark.parametrize("tokens", [64, 65])
def test_a_layer_whose_scores_cancel(pkg, tokens, monkeypatch):
    """The experts one by one are the experts that the kernels choose: scores that 32 bits do not tell apart, as in the router's own test."""
    router, gate, up, down = _small_mixture(pkg, experts=8)
    order = np.random.default_rng(6).permutation(8)
    w = torch.zeros(8, 64, 4, device=DEV)
    for e in range(8):
        w[e, e, 0], w[e, 63 - e, 0] = 2.0 ** 18, -2.0 ** 18
        w[e, e, 1] = float(order[e]) * 2.0 ** -9                 # products of 2^24 beside up to 7 * 2^-3
    x = torch.full((tokens, 256), 64.0, device=DEV, dtype=torch.float16)
    chosen = [int(i) for i in np.argsort(-order)[:2]]
    layer = pkg.ops.GGMLMoE(w.view(8, 256), gate, up, down, top_k=2, renormalize=False)
    ids, share = pkg.moe.route(x, w.view(8, 256), 2, renormalize=False)
    assert ids.tolist() == [chosen] * tokens
    ran, expert = set(), layer._expert
    monkeypatch.setattr(layer, "_expert", lambda stack, e, *a: ran.add(e) or expert(stack, e, *a))
    layer._one_by_one(x)
    assert ran == set(chosen)


# ---- more rows than one launch has threads for

def test_quantized_rows_beyond_a_launch(pkg):
    """2^26 rows and more, a wave each: the same as in two halves."""
    rows, k = (1 << 26) + 5, 16
    x = (torch.arange(rows, device=DEV, dtype=torch.int32) % 251).to(torch.bfloat16)[:, None] * torch.tensor([1.0, -0.5] * 8, device=DEV, dtype=torch.bfloat16)
    x[:, 3] += 7
    q, scale = pkg.int8.quantize_rows(x)
    half = rows // 2
    for part in (slice(0, half), slice(half, rows)):
        a, b = pkg.int8.quantize_rows(x[part])
        assert torch.equal(q[part], a) and torch.equal(scale[part], b)


def test_products_beyond_a_launch(pkg):
    """A weight of 2^27 rows for one row and for 20, x of 2^30 rows and more for one row of the weight: every 16 rows (64, with the tiles) took a workgroup."""
    n = 1 << 27
    w = torch.zeros(n, 16, dtype=torch.int8, device=DEV)
    w[:, 0] = (torch.arange(n, device=DEV, dtype=torch.int32) % 127).to(torch.int8)
    w[:, 5] = 1
    scale = torch.ones(n, device=DEV)
    x = torch.zeros(20, 16, device=DEV, dtype=torch.float16)
    x[:, 0], x[:, 5] = 127, 3
    x[7, 0] = 0
    part = pkg.int8.linear_int8(x, w[:254], scale[:254])
    for m in (1, 20):
        y = pkg.int8.linear_int8(x[:m], w, scale)
        assert y.shape == (m, n)
        whole = n // 127 * 127
        assert torch.equal(y[:, :whole].view(m, -1, 127), part[:m, None, :127].expand(m, whole // 127, 127)) and torch.equal(y[:, whole:], part[:m, :n - whole])
    del y, w, scale
    m = (1 << 30) + 70
    q = torch.zeros(m, 16, dtype=torch.int8, device=DEV)
    q[:, 2] = 5
    q[-1, 2], q[1 << 30, 2] = 9, 11
    y = pkg.int8.linear_int8(q, torch.full((1, 16), 2, dtype=torch.int8, device=DEV), torch.ones(1, device=DEV), x_scale=torch.ones(m, device=DEV), out_dtype=torch.float16)
    assert y.shape == (m, 1) and float(y[-1]) == 18 and float(y[1 << 30]) == 22
    y[-1] = y[1 << 30] = 10
    assert bool((y == 10).all())


def test_norms_of_more_rows_than_32_bits_count(pkg):
    rows = (1 << 32) + 6
    x = torch.ones(rows, 1, device=DEV, dtype=torch.bfloat16)
    x[-3:] = -2.0
    x[1 << 32] = 0.0
    r, y = pkg.norms.block_norm(x, scale=torch.full((1,), 2.0, device=DEV), eps=0.0625)
    assert r.data_ptr() == x.data_ptr()
    at = [0, (1 << 32) - 1, 1 << 32, (1 << 32) + 1, rows - 3, rows - 1]
    want = [3 / 1.0625 ** 0.5] * 2 + [0.0, 3 / 1.0625 ** 0.5] + [-6 / 4.0625 ** 0.5] * 2
    got = torch.stack([y[i, 0] for i in at]).double().cpu()
    assert bool(((got - torch.tensor(want, dtype=torch.float64)).abs() <= 2.0 ** -8 * torch.tensor(want, dtype=torch.float64).abs()).all())
    y[-3:], y[1 << 32] = y[0], y[0]
    assert bool((y == y[0]).all())


@pytest.mark.parametrize("rows,dim", [(5000, 256), (3000, 2432), (700, 4097), (40, 16384)])
def test_outputs_on_the_inputs_at_the_c_entry(pkg, rows, dim):
    """stream_out on stream and y on branch, or the other way round: what the call gives in arrays of their own."""
    import ctypes
    n = pkg._native
    g = torch.Generator(device=DEV)
    g.manual_seed(103)
    stream, branch = (torch.randn(rows, dim, device=DEV, generator=g).bfloat16() for _ in range(2))
    want_r, want_y = pkg.norms.block_norm(stream, branch, post_norm="layer", norm="rms")
    for swap in (False, True):
        s, b = stream.clone(), branch.clone()
        out, y = (b, s) if swap else (s, b)
        d = n.ggq_norm_desc(stream=s.data_ptr(), branch=b.data_ptr(), stream_out=out.data_ptr(), y=y.data_ptr(), rows=rows, dim=dim, rows_per_mod=rows, dtype=n.BF16, norm=1, post_norm=2, eps=1e-6)
        assert n.lib().ggq_block_norm(ctypes.byref(d), torch.cuda.current_stream().cuda_stream) == n.GGQ_OK
        assert torch.equal(out, want_r) and torch.equal(y, want_y)


# ---- many tokens over many spans

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,experts,top_k", [(20, 8, 2), (33, 4, 2), (48, 8, 2), (64, 8, 2), (64, 16, 4)])
@pytest.mark.parametrize("up_name,down_name,dim,ff", [("Q4_K", "Q6_K", 2048, 1280), ("Q8_0", "Q5_0", 2112, 1216)])
def test_more_tokens_on_an_expert_than_columns_in_registers(pkg, kind, tokens, experts, top_k, up_name, down_name, dim, ff):
    """Evenly spread routes, and all tokens on one expert, over as many pieces of k as every wave takes several of: the sums of the columns that the registers have no room for
    are kept in LDS, for one matrix and for two."""
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(104)
    gate, up = (Stack(pkg, up_name, (experts, ff, dim), kind, 90 + i, shrink=0.125) for i in range(2))
    down = Stack(pkg, down_name, (experts, dim, ff), kind, 92, shrink=0.125)
    x = (torch.randn(tokens, dim, device=DEV, generator=g) * 0.25).to(dtype)
    spread = torch.stack([torch.randperm(experts, device=DEV, generator=g)[:top_k] for _ in range(tokens)]).int()
    one = spread.clone()
    one[:, 0] = 1
    one[:, 1] = torch.where(one[:, 1] == 1, -1, one[:, 1])
    one[5:, 1:] = -1
    weights = torch.rand(tokens, top_k, device=DEV, generator=g) + 0.25
    for ids in (spread, one):
        y = pkg.moe.moe_experts(x, ids, weights, gate.tensor, up.tensor, down.tensor)
        want, bound = _want(x, ids, weights, gate.dense, up.dense, down.dense, "silu", dtype)
        assert bool(want.isfinite().all()) and float(want.abs().max()) < 60000
        _close(y, want, bound, dtype)


# ---- calls that stand for themselves

def _q8_rows(pkg, values):
    """A Q8_0 stack of one expert whose row j holds values[j] in column 0 (at most 127, whole) and values2[j] in column 1."""
    first, second = values
    rows = first.numel()
    b = np.zeros((rows, 2, 34), dtype=np.uint8)
    b[:, :, :2] = np.array([1.0], dtype=np.float16).view(np.uint8)
    b[:, 0, 2] = first.numpy().astype(np.int8).view(np.uint8)
    b[:, 0, 3] = second.numpy().astype(np.int8).view(np.uint8)
    return pkg.ops.GGMLTensor(torch.from_numpy(b.reshape(-1)).to(DEV), tensor_type=pkg.qtypes.Q.Q8_0, tensor_shape=(1, rows, 64))


def test_every_size_of_an_fp16_hidden_value(pkg):
    """One hidden value per result: silu(g) u with g >= 40, where silu(g) is g to 2^-57.  g and u are products of two numbers of 11 bits, so exact in fp32; h is one fp32 product (and
    the activation's reciprocal: 4 u), kept to 2^-22, or to 2^-19 beyond 65504, and y is half a step of share * h.  Values on both sides of 65520, where fp16 begins to
    round to infinity, and up to 2^45, of either sign."""
    g = torch.tensor([1, 2, 47, 61, 64, 100, 120, 127] * 8, dtype=torch.float32)
    u = torch.tensor([1] * 8 + [-1] * 8 + [2] * 8 + [-3] * 8 + [16] * 8 + [-64] * 8 + [127] * 8 + [-127] * 8, dtype=torch.float32)
    none = torch.zeros(64)
    gate, up = _q8_rows(pkg, (g, none)), _q8_rows(pkg, (none, u))
    b = np.zeros((64, 2, 34), dtype=np.uint8)
    b[:, :, :2] = np.array([1.0], dtype=np.float16).view(np.uint8)
    for i in range(64):
        b[i, i // 32, 2 + i % 32] = 1
    down = pkg.ops.GGMLTensor(torch.from_numpy(b.reshape(-1)).to(DEV), tensor_type=pkg.qtypes.Q.Q8_0, tensor_shape=(1, 64, 64))
    x = torch.zeros(9, 64)
    x[:, 0] = torch.tensor([1394.0, 546.0, 512.0, 40.0, 16384.0, 60000.0, 1071.0, 1092.0, 515.0])
    x[:, 1] = torch.tensor([1.0, 1.0, 1.0, 1.0, 16384.0, 60000.0, 1.0, 0.5, 0.25])
    want = (x[:, :1].double() * g.double()) * (x[:, 1:2].double() * u.double())
    assert {65518.0, 65520.0, 65536.0} <= set(want.abs().flatten().tolist()) and float(want.abs().max()) > 2.0 ** 45
    for share in (2.0 ** -31, 2.0 ** -12, 1.0):
        y = pkg.moe.moe_experts(x.half().to(DEV), torch.zeros(9, 1, dtype=torch.int32, device=DEV), torch.full((9, 1), share, device=DEV), gate, up, down)
        t = (share * want).abs()
        fits = t < 65000
        tol = t * (2.0 ** -11 + torch.where(want.abs() > 65504, 2.0 ** -19, 2.0 ** -22) + 8 * U) + 2.0 ** -25
        err = (y.double().cpu() - share * want).abs()
        assert bool((err <= tol)[fits].all()), float((err / tol)[fits].max())
        assert torch.equal(y.cpu()[t > 66000], torch.sign(want[t > 66000]).half() * float("inf"))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_layer_of_many_experts_in_a_graph(pkg, kind):
    """The router's two launches and its scratch, hidden values beyond fp16: captured once, replayed on other inputs between eager calls."""
    dtype = DT[kind]
    gate, up = (Stack(pkg, "Q4_K", (40, 256, 256), kind, 110 + i).tensor for i in range(2))
    down = Stack(pkg, "Q6_K", (40, 256, 256), kind, 112, shrink=2.0 ** -10).tensor
    g = torch.Generator(device=DEV)
    g.manual_seed(105)
    router = torch.randn(40, 256, device=DEV, generator=g) * 0.05
    layer = pkg.ops.GGMLMoE(router, gate, up, down, top_k=3)
    static = torch.randn(7, 256, device=DEV, generator=g).to(dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(static)
    for i in range(5):
        new = (torch.randn(7, 256, device=DEV, generator=g) * (1.0, 30.0, 0.01, 100.0, 1.0)[i]).to(dtype)
        static.copy_(new)
        graph.replay()
        kept = out.clone()
        assert torch.equal(kept.nan_to_num(1.5), layer(new).nan_to_num(1.5)) and torch.equal(kept.isnan(), layer(new).isnan())
        torch.cuda.synchronize()


def test_the_longest_sums_in_every_kernel(pkg):
    """131071 columns at the extremes, for few rows and for many: |sum| = 127 * 128 * 131071 = 0.99 * 2^31, the integers exact."""
    k = 131071
    for m, n in ((16, 5), (17, 70), (300, 260)):
        q = torch.full((m, k), 127, dtype=torch.int8, device=DEV)
        w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
        w[1::2] = 127
        w[0, :7] = 1
        y = pkg.int8.linear_int8(q, w, torch.ones(n, device=DEV), x_scale=torch.ones(m, device=DEV), out_dtype=torch.float32)
        want = w.long().sum(1).mul(127).float()
        assert torch.equal(y, want[None].expand(m, n))


@pytest.mark.parametrize("experts", [5, 20])
def test_routes_of_as_many_tokens_as_a_call_takes(pkg, experts):
    g = torch.Generator(device=DEV)
    g.manual_seed(106)
    x, w = torch.randn(65535, 8, device=DEV, generator=g).bfloat16(), torch.randn(experts, 8, device=DEV, generator=g).bfloat16()
    ids, weights = pkg.moe.route(x, w, 3)
    scores = x.double() @ w.double().t()                        # 8 exact products; their sums in 64 bits differ by the order of adding at most, 2^-50 of the terms
    p, order = torch.sort(torch.softmax(scores, -1), dim=-1, descending=True, stable=True)
    top = torch.sort(scores, dim=-1, descending=True)[0]
    clear = (top.diff(dim=-1).abs()[:, :3] > 2.0 ** -49 * (x.double().abs() @ w.double().abs().t()).amax(-1, keepdim=True)).all(-1)
    assert int(clear.sum()) > 65000 and torch.equal(ids[clear].long(), order[clear, :3])
    want = p[:, :3] / p[:, :3].sum(-1, keepdim=True)
    # |difference of scores| u for its rounding to fp32 (8 products of normal values: below 40), and 16 u for exp, reciprocal, sum and product
    assert bool(((weights.double() - want).abs() <= want * 64 * U)[clear].all())
    with pytest.raises(pkg.dequant.GGQUnsupported):
        pkg.moe.route(torch.cat((x, x[:1])), w, 3)
