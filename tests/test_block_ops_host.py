"""Host side of the block operators without a GPU: refusals of the python entry points, and of the C entry points before anything is launched."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused(pkg):
    no = pkg.dequant.GGQUnsupported
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(no):
        pkg.norms.block_norm(x)
    with pytest.raises(no):
        pkg.int8.quantize_rows(x)
    with pytest.raises(no):
        pkg.int8.linear_int8(x, torch.zeros(4, 64, dtype=torch.int8), torch.ones(4))
    with pytest.raises(no):
        pkg.moe.route(x, x, 1)
    with pytest.raises(no):
        pkg.moe.moe_experts(x, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1), x, x, x)


def test_layers_do_not_drop_patches(pkg):
    Q, ops = pkg.qtypes.Q, pkg.ops
    packed = torch.from_numpy(pkg.synth.make_tensor_bytes(Q.Q8_0, (2 * 64, 64), seed=1))
    stack = ops.GGMLTensor(packed, tensor_type=Q.Q8_0, tensor_shape=(2, 64, 64), patches=[("lora", "key")])
    x = torch.ones(3, 64)
    with pytest.raises(ValueError, match="patch"):
        ops.GGMLMoE(torch.zeros(2, 64), stack, stack, stack, 1)(x)
    with pytest.raises(ValueError, match="patch"):
        ops.GGMLInt8Linear(ops.GGMLTensor(packed, tensor_type=Q.Q8_0, tensor_shape=(128, 64), patches=[("lora", "key")]))
    with pytest.raises(pkg.dequant.GGQUnsupported):
        pkg.moe.moe_layer(torch.tensor(1.0), torch.zeros(2, 64), stack, stack, stack, top_k=1)


def test_layer_with_stacks_that_are_not_packed(pkg):
    """Equal experts, equal scores: each token's result is one expert's, every value a small integer or a half (exact in fp32)."""
    g = torch.Generator().manual_seed(2)
    one = [torch.randint(-1, 2, s, generator=g).float() for s in ((32, 16), (32, 16), (16, 32))]
    stacks = [w[None].expand(2, *w.shape) for w in one]
    x = torch.randint(-2, 3, (5, 16), generator=g).float()
    layer = pkg.ops.GGMLMoE(torch.zeros(2, 16), *stacks, 2, activation="silu")
    want = (torch.nn.functional.silu(x @ one[0].t()) * (x @ one[1].t())) @ one[2].t()
    torch.testing.assert_close(layer(x), want, rtol=2.0 ** -20, atol=2.0 ** -12)


def _lib(pkg):
    return pkg._native.lib()


# addresses that are never followed: every call below has to be answered before a launch
A = 0x10000


def test_block_norm_arguments_at_the_c_entry(pkg):
    n, L = pkg._native, _lib(pkg)

    def call(**kw):
        base = dict(stream=A, y=A, rows=4, dim=64, rows_per_mod=4, dtype=n.F16, norm=1, post_norm=0, eps=1e-6)
        base.update(kw)
        return L.ggq_block_norm(ctypes.byref(n.ggq_norm_desc(**base)), None)
    assert L.ggq_block_norm(None, None) == n.GGQ_ERR_ARG
    assert call(rows=0) == n.GGQ_OK
    for bad in (dict(dtype=3), dict(dtype=-1), dict(norm=3), dict(post_norm=-1), dict(dim=0), dict(rows_per_mod=0), dict(stream=None), dict(branch=A), dict(y=None),
                dict(y_scale=A, y_stride=63), dict(y_scale=A, y_stride=72), dict(y_scale=A, y=None, branch=A, stream_out=A, y_stride=64), dict(dim=32769)):
        assert call(**bad) == n.GGQ_ERR_ARG, bad
    for bad in (dict(stream=A + 1), dict(y=A + 1), dict(y_scale=A, y_stride=64, y=A + 8), dict(weight=A + 1), dict(weight=A + 2, params_f32=4), dict(dtype=n.F32, stream=A + 2)):
        assert call(**bad) == n.GGQ_ERR_ALIGN, bad


def test_quantize_and_product_arguments_at_the_c_entry(pkg):
    n, L = pkg._native, _lib(pkg)
    q = lambda x=A, rows=4, cols=64, to=A, stride=64, s=A, dt=n.F16: L.ggq_quantize_rows(x, rows, cols, to, stride, s, dt, None)  # noqa: E731
    assert q(rows=0) == n.GGQ_OK
    for rc in (q(x=None), q(to=None), q(s=None), q(cols=0), q(stride=48), q(stride=65), q(dt=3), q(cols=32769, stride=32784)):
        assert rc == n.GGQ_ERR_ARG
    assert q(to=A + 8) == n.GGQ_ERR_ALIGN and q(x=A + 1) == n.GGQ_ERR_ALIGN
    p = lambda x=A, xs=64, sx=A, m=4, w=A, ws=64, sw=A, rows=4, k=64, b=None, y=A, dt=n.F16: L.ggq_linear_int8(x, xs, sx, m, w, ws, sw, rows, k, b, y, dt, None)  # noqa: E731
    assert p(m=0) == n.GGQ_OK and p(rows=0) == n.GGQ_OK
    for rc in (p(x=None), p(sx=None), p(w=None), p(sw=None), p(y=None), p(xs=48), p(xs=72), p(ws=48), p(k=65), p(k=0), p(k=131072, xs=1 << 20, ws=1 << 20), p(dt=3), p(m=(1 << 32) - 1, rows=(1 << 32) - 1)):
        assert rc == n.GGQ_ERR_ARG
    for rc in (p(x=A + 8), p(w=A + 8), p(y=A + 1), p(dt=n.F32, y=A + 2), p(b=A + 1), p(sx=A + 2), p(sw=A + 2)):
        assert rc == n.GGQ_ERR_ALIGN


def test_few_rows_arguments_at_the_c_entry(pkg):
    n, L = pkg._native, _lib(pkg)
    p = lambda x=A, m=2, w=A, ws=64, sw=A, rows=4, k=64, b=None, y=A, dt=n.F16: L.ggq_linear_int8_few(x, m, w, ws, sw, rows, k, b, y, dt, None)  # noqa: E731
    assert p(m=0) == n.GGQ_OK and p(rows=0) == n.GGQ_OK
    for rc in (p(x=None), p(w=None), p(sw=None), p(y=None), p(m=17), p(k=0), p(k=60), p(m=2, k=8200, ws=8208), p(ws=48), p(ws=72), p(dt=3)):
        assert rc == n.GGQ_ERR_ARG
    for rc in (p(x=A + 8), p(w=A + 8), p(y=A + 1)):
        assert rc == n.GGQ_ERR_ALIGN


def test_expert_arguments_at_the_c_entry(pkg):
    n, L = pkg._native, _lib(pkg)
    r = lambda x=A, w=A, t=4, d=64, e=8, k=2, ids=A, out=A, dt=n.F16, rt=n.F16, ws=A, size=1 << 20: L.ggq_moe_route(x, w, t, d, e, k, 1, ids, out, dt, rt, ws, size, None)  # noqa: E731
    assert r(t=0) == n.GGQ_OK
    for rc in (r(x=None), r(w=None), r(ids=None), r(out=None), r(d=0), r(d=60), r(e=0), r(e=513, k=2), r(k=0), r(k=9), r(k=17, e=64), r(dt=n.F32), r(rt=n.BF16), r(t=65536), r(e=17, ws=None), r(e=17, size=4 * 17 * 8 - 1)):
        assert rc == n.GGQ_ERR_ARG
    assert r(x=A + 2) == n.GGQ_ERR_ALIGN and r(ids=A + 2) == n.GGQ_ERR_ALIGN and r(e=17, ws=A + 4) == n.GGQ_ERR_ALIGN
    assert L.ggq_moe_route_workspace(4, 16) == 0 and L.ggq_moe_route_workspace(4, 17) == 4 * 17 * 8

    def call(**kw):
        base = dict(x=A, ids=A, weights=A, gate=A, up=A, down=A, y=A, workspace=A, workspace_bytes=1 << 30, tokens=4, top_k=2, experts=8, dim=256, ff=512, up_qtype=12, down_qtype=14,
                    act=0, dtype=n.F16)
        base.update(kw)
        return L.ggq_moe_experts(ctypes.byref(n.ggq_moe_desc(**base)), None)
    assert L.ggq_moe_experts(None, None) == n.GGQ_ERR_ARG
    assert call(tokens=0) == n.GGQ_OK
    assert call(up_qtype=16) == n.GGQ_ERR_QTYPE and call(down_qtype=0) == n.GGQ_ERR_QTYPE
    for bad in (dict(x=None), dict(ids=None), dict(weights=None), dict(gate=None), dict(up=None), dict(down=None), dict(y=None), dict(workspace=None), dict(workspace_bytes=L.ggq_moe_workspace(4, 2, 256, 512) - 1),
                dict(tokens=65), dict(top_k=0), dict(top_k=17), dict(experts=0), dict(experts=513), dict(dim=192), dict(dim=0), dict(ff=320), dict(ff=0), dict(act=2), dict(dtype=n.F32)):
        assert call(**bad) == n.GGQ_ERR_ARG, bad
    for bad in (dict(x=A + 8), dict(gate=A + 8), dict(workspace=A + 8), dict(ids=A + 2), dict(y=A + 4)):
        assert call(**bad) == n.GGQ_ERR_ALIGN, bad
    assert L.ggq_moe_workspace(64, 16, 1 << 20, 1 << 20) == (64 * 16 * 4 << 20) + (64 * 4 << 20)       # hidden values, and one part of y
    assert L.ggq_moe_workspace(3, 2, 256, 512) == 3 * 2 * 512 * 4 + 8 * 3 * 256 * 4
