"""The block operators at the edges of what their documentation allows, as far as that is decided without a GPU."""
import pytest
import torch


def _stacks(experts=3, ff=8, dim=4):
    return torch.ones(experts, ff, dim), torch.ones(experts, ff, dim), torch.ones(experts, dim, ff)


@pytest.mark.parametrize("bad", [dict(activation="relu"), dict(activation="gelu"), dict(activation=None), dict(top_k=0), dict(top_k=4), dict(top_k=-1)])
def test_a_mixture_that_is_not_one_is_refused_when_it_is_made(pkg, bad):
    """Not when it runs: the experts one by one would take any activation for gelu, and any number of places for as many as there are experts."""
    with pytest.raises(ValueError):
        pkg.ops.GGMLMoE(torch.zeros(3, 4), *_stacks(), **{"top_k": 2, **bad})
    layer = pkg.ops.GGMLMoE(torch.zeros(3, 4), *_stacks(), top_k=3, activation="gelu_tanh")
    x = torch.full((2, 4), 0.25)
    torch.testing.assert_close(layer(x), torch.full((2, 4), 8 * float(torch.nn.functional.gelu(torch.tensor(1.0), approximate="tanh"))))


def test_tensors_that_a_launch_cannot_see_are_refused(pkg):
    """A dual tensor's requires_grad is false; inside vmap a tensor has no memory of its own.  Others in the same call are what they were."""
    from torch.autograd import forward_ad
    refuse, no = pkg.norms._refuse_grad, pkg.dequant.GGQUnsupported
    x = torch.ones(3, 4)
    with torch.no_grad(), forward_ad.dual_level():
        refuse("call", x, None, x[0])
        for args in ((forward_ad.make_dual(x, x),), (x, None, forward_ad.make_dual(x, x))):
            with pytest.raises(no, match="forward"):
                refuse("call", *args)

    def inside(v, alone=False):
        if not alone:                                             # inside jvp the results of a call would be wrapped too
            refuse("call", x)
        with pytest.raises(no, match="transform"):
            refuse("call", x, v)
        with pytest.raises(no, match="transform"):
            pkg.norms.block_norm(v)
        return v
    torch.vmap(inside)(x)
    torch.func.jvp(lambda v: inside(v, True), (x,), (x,))
    refuse("call", x)


def test_experts_one_by_one_under_transforms(pkg):
    """Forward-mode gradients against backward ones (in fp32: sums of up to 8 x 4 x 8 terms in another order, 2^-17), vmap against a loop."""
    from torch.autograd import forward_ad
    g = torch.Generator().manual_seed(5)
    stacks = [torch.randn(s, generator=g) * 0.4 for s in ((3, 8, 4), (3, 8, 4), (3, 4, 8))]
    layer = pkg.ops.GGMLMoE(torch.randn(3, 4, generator=g), *stacks, top_k=2)
    x, v = torch.randn(5, 4, generator=g), torch.randn(5, 4, generator=g)
    y, back = torch.autograd.functional.vjp(layer, x, torch.ones(5, 4))
    with forward_ad.dual_level():
        dual = forward_ad.unpack_dual(layer(forward_ad.make_dual(x, v)))
    value, tangent = torch.func.jvp(layer, (x,), (v,))
    for t in (dual.tangent, tangent):
        assert abs(float(t.sum()) - float((back * v).sum())) <= 2.0 ** -17 * float((back * v).abs().sum())
    assert torch.equal(dual.primal, y)
    torch.testing.assert_close(value, y, rtol=2.0 ** -17, atol=2.0 ** -20)
    many = torch.randn(6, 5, 4, generator=g)
    torch.testing.assert_close(torch.vmap(layer)(many), torch.stack([layer(m) for m in many]), rtol=2.0 ** -17, atol=2.0 ** -20)


def test_patched_parameters_are_refused_everywhere(pkg):
    """A LoRA patch on a norm's weight, a router or a bias is not dropped either: get_weight applies those (ops.py:183-190), the kernels do not."""
    G, no = pkg.ops.GGMLTensor, pkg.dequant.GGQUnsupported
    f32, q8 = pkg.qtypes.Q.F32, pkg.qtypes.Q.Q8_0
    plain = G(torch.ones(64), tensor_type=f32, tensor_shape=(64,))
    patched = G(torch.ones(64), tensor_type=f32, tensor_shape=(64,), patches=[("lora", "key")])
    packed = torch.from_numpy(pkg.synth.make_tensor_bytes(q8, (1, 64), seed=1))
    for good in (plain, torch.ones(64)):
        v, is32 = pkg.norms._vector(good, 64, torch.float16, torch.device("cpu"), "weight")
        assert type(v) is torch.Tensor and is32
        assert pkg.norms._per_sample(good, (2, 3), 64, torch.float16, torch.device("cpu"), "gate", 1)[0].shape == (1, 64)
    for bad in (patched, G(packed, tensor_type=q8, tensor_shape=(1, 64), patches=[("lora", "key")])):
        with pytest.raises(no, match="patch"):
            pkg.norms._vector(bad, 64, torch.float16, torch.device("cpu"), "weight")
    with pytest.raises(no, match="patch"):
        pkg.norms._per_sample(patched, (2, 3), 64, torch.float16, torch.device("cpu"), "gate", 1)
    with pytest.raises(no, match="patch"):
        pkg.norms._plain(patched)
    router = G(torch.zeros(3, 4), tensor_type=f32, tensor_shape=(3, 4), patches=[("lora", "key")])
    with pytest.raises(ValueError, match="patch"):
        pkg.ops.GGMLMoE(router, *_stacks(), top_k=2)
    with pytest.raises(ValueError, match="patch"):
        pkg.ops.GGMLInt8Linear(torch.ones(64, 8), patched)


def test_more_rows_than_a_launch_takes_are_refused(pkg):
    """At the C entries, before anything is launched (addresses that are never followed): fewer than 2^32 threads are one launch."""
    import ctypes
    n, A = pkg._native, 0x10000
    L = n.lib()

    def norm(**kw):
        return L.ggq_block_norm(ctypes.byref(n.ggq_norm_desc(**{**dict(stream=A, y=A, rows=1 << 22, dim=8200, rows_per_mod=4, dtype=n.F16, norm=1, post_norm=0, eps=1e-6), **kw})), None)
    assert norm() == n.GGQ_ERR_ARG and norm(dim=4097) == n.GGQ_ERR_ARG and norm(dim=32768, rows=1 << 40) == n.GGQ_ERR_ARG
    for cols, stride, rows in ((8200, 8208, 1 << 22), (4105, 8208, 1 << 22), (32768, 32768, 1 << 33)):
        assert L.ggq_quantize_rows(A, rows, cols, A, stride, A, n.F16, None) == n.GGQ_ERR_ARG
    for m, rows in ((1 << 31, 1), (1, 1 << 31), ((1 << 32) - 1, 1), (1 << 25, 1 << 24), ((1 << 31) - 1, 257)):
        assert L.ggq_linear_int8(A, 64, A, m, A, 64, A, rows, 64, None, A, n.F16, None) == n.GGQ_ERR_ARG, (m, rows)
    assert L.ggq_linear_int8_few(A, 1, A, 64, A, 16 * ((1 << 23) - 1), 64, None, A, n.F16, None) == n.GGQ_ERR_ARG


def test_rows_beyond_32_bits_per_modulation_vector(pkg):
    """One vector for all rows is read for all of them, however many; the descriptor's field has 32 bits."""
    per = pkg.norms._rows_per_vector
    assert per(6, 1) == 6 and per(6, 3) == 2 and per(0, 1) == 1 and per(2, 2) == 1
    assert per((1 << 32) - 1, 1) == (1 << 32) - 1
    assert per(5 << 32, 1) == (1 << 32) - 1
    assert per(5 << 32, 5 << 3) == 1 << 29
    with pytest.raises(pkg.dequant.GGQUnsupported):
        per(5 << 32, 5)


def test_eight_bit_rows_do_not_go_over_the_inputs(pkg):
    """y may be branch where its rows lie on branch's own; 8-bit rows do not, and another workgroup's would be gone before they are read."""
    import ctypes
    n, A = pkg._native, 0x100000
    base = dict(stream=A, branch=2 * A, stream_out=A, y=3 * A, y_scale=4 * A, rows=4, dim=64, rows_per_mod=4, y_stride=64, dtype=n.F16, norm=1, post_norm=0, eps=1e-6)

    def call(**kw):
        return n.lib().ggq_block_norm(ctypes.byref(n.ggq_norm_desc(**{**base, **kw})), None)
    row = 64 * 2
    for y in (A, 2 * A, A + row, 2 * A + 3 * row, A - 64, 2 * A - 3 * 64, 2 * A - 64 - 48):
        assert call(y=y) == n.GGQ_ERR_ARG, hex(y)
    assert call(branch=None, stream_out=None, y=A) == n.GGQ_ERR_ARG
    assert n.lib().ggq_quantize_rows(A, 4, 64, A, 64, 4 * A, n.F16, None) == n.GGQ_ERR_ARG
    assert n.lib().ggq_quantize_rows(A, 4, 64, A + 3 * row, 64, 4 * A, n.F16, None) == n.GGQ_ERR_ARG
    # 16-bit rows: on the input's own rows or apart from it, nothing between
    for y in (A + row, 2 * A + row, 2 * A - 3 * row, A + 2, 2 * A + 16):
        assert call(y=y, y_scale=None) == n.GGQ_ERR_ARG, hex(y)
    for out in (A + row, 2 * A + row, 2 * A + 16):
        assert call(stream_out=out) == n.GGQ_ERR_ARG, hex(out)
    assert call(y=A, y_scale=None) == n.GGQ_ERR_ARG and call(y=5 * A, stream_out=5 * A, y_scale=None) == n.GGQ_ERR_ARG          # y on the stream that is stored


def test_experts_in_torch_are_chosen_by_scores_in_64_bits(pkg):
    """Small scores beside terms of 2^24 that cancel: 32 bits do not tell them apart.  Each expert's result is its own number."""
    order = torch.tensor([3, 0, 7, 5, 1, 6, 2, 4])
    router = torch.zeros(8, 64)
    for e in range(8):
        router[e, 4 * e], router[e, 63 - 4 * e], router[e, 4 * e + 1] = 2.0 ** 24, -2.0 ** 24, float(order[e]) * 2.0 ** -3
    gate, up = torch.full((8, 1, 64), 1.0), torch.full((8, 1, 64), 1.0)
    down = torch.arange(1.0, 9.0).view(8, 1, 1).expand(8, 64, 1)
    x = torch.ones(2, 64)
    y = pkg.ops.GGMLMoE(router, gate, up, down, top_k=1)(x)
    assert torch.equal(y, torch.full((2, 64), 64.0 * 64.0 * 3))          # silu(64) is 64 in fp32; the third expert has the largest score
