"""int8.quantize_rows / int8.linear_int8 (include/ggq.h) on an MI355X.

Quantization of 16-bit rows is exact: q = rint(127 x / max|x|) has to be the same integer as in rational arithmetic, half-way values to the even one.  The
product's integer sum is exact; float(sum), the product of the scales, their product and the bias are four fp32 roundings (u = 2^-24), then half a step e of
the result's type: e |y| + 4 u (|sum sx sw| + |bias|)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _quants(x):
    """rint(127 x / max|x|) of a 16-bit matrix in integers: x = n 2^e exactly."""
    v = x.double().cpu().numpy()
    top = np.abs(v).max(-1, keepdims=True)
    num = v * 254                                              # exact: 11 + 8 bits
    twice = np.floor(num / np.where(top > 0, top, 1) + 1)      # floor(2 t + 1); doubles divide 19 by 11 bits: whole results are exact, others are >= 2^-19 away
    q = np.floor(twice / 2)
    tie = (num + top == 2 * q * top) & (np.mod(q, 2) == 1)     # t + 1/2 == q exactly
    return np.where(top > 0, q - tie, 0).astype(np.int64)


def _scales(x):
    """max|x| / 127, correctly rounded: numpy divides (torch multiplies by a rounded 1 / 127)."""
    return x.float().abs().amax(-1).cpu().numpy() / np.float32(127)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (7, 33), (2050, 520), (5, 24576), (260, 2432)])
def test_quantized_rows_are_exact(pkg, kind, shape):
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    x = torch.randn(*shape, device=DEV, generator=g).to(DT[kind])
    x[0, shape[1] // 2:] = x[0, 0] / 2                         # half of the maximum: 63.5 steps where x[0, 0] is the largest
    x[:, 0] *= 8
    if shape[0] > 2:
        x[2] = 0
    q, scale = pkg.int8.quantize_rows(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and q.stride(0) % 16 == 0 and scale.shape == shape[:1]
    assert np.array_equal(q.cpu().numpy().astype(np.int64), _quants(x))
    assert np.array_equal(scale.cpu().numpy(), _scales(x))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_quantization_of_every_bit_pattern(pkg, kind):
    """Every finite 16-bit value, in rows of random order: subnormals, the largest values, both zeros."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(DT[kind])
    x = x[x.isfinite()]
    x = x[torch.from_numpy(np.random.default_rng(4).permutation(x.numel()))]
    x = x[:x.numel() // 64 * 64].view(-1, 64)
    x = torch.cat((x, torch.sort(x.flatten().float().abs())[0].to(DT[kind]).view(-1, 64)))           # and of similar sizes: ties among small numbers
    q, scale = pkg.int8.quantize_rows(x.to(DEV))
    assert np.array_equal(q.cpu().numpy().astype(np.int64), _quants(x))


def test_quantization_of_fp32_rows_and_rows_without_a_form(pkg):
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    x = torch.randn(300, 777, device=DEV, generator=g)
    q, scale = pkg.int8.quantize_rows(x)
    t = x.double() * 127 / x.double().abs().amax(-1, keepdim=True)
    assert bool(((q.double() - t).abs() <= 0.5 + 2.0 ** -16).all())       # |t| < 128 rounded to fp32 before rint: 2^-18, and fp64's own
    assert np.array_equal(scale.cpu().numpy(), _scales(x))
    x[1, 5], x[2, 6], x[3] = float("nan"), float("-inf"), 0.0
    q, scale = pkg.int8.quantize_rows(x)
    assert bool(scale[1:3].isnan().all()) and float(scale[3]) == 0 and not bool(q[1:4].any())
    y = pkg.int8.linear_int8(x[:4, :776], q[:50, :776], torch.ones(50, device=DEV))          # few rows: quantized in the product itself
    assert bool(y[1:3].isnan().all()) and not bool(y[3].any()) and bool(y[0].isfinite().all())
    y = pkg.int8.linear_int8(x, q[:50], torch.ones(50, device=DEV))
    assert bool(y[1:3].isnan().all()) and not bool(y[3].any()) and bool(y[0].isfinite().all())


def _weight(n, k, g, stride=None):
    q = torch.randint(-128, 128, (n, stride or (k + 15) // 16 * 16), device=DEV, generator=g, dtype=torch.int8)      # whatever lies behind column k has no effect
    return q[:, :k], torch.rand(n, device=DEV, generator=g) + 0.5


def _check(y, q, sx, w, sw, bias, dtype):
    acc = q.double() @ w.double().T
    part = acc * sx.double()[:, None] * sw.double()
    want = part if bias is None else part + bias.double()
    tol = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 8 * U) + 4 * U * (part.abs() + (0 if bias is None else bias.double().abs())) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = (y.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


SIZES = [(1, 1, 1), (1, 17, 64), (3, 100, 1001), (16, 48, 4096), (17, 33, 129), (64, 65, 127), (65, 130, 2432), (128, 128, 128), (129, 257, 384), (333, 1501, 1001), (300, 70, 16),
         (1, 10240, 4096), (2, 5, 20000), (1100, 1030, 640), (4100, 4099, 160), (31, 16384, 48), (700, 5000, 200), (1, 100, 16384), (2, 33, 8192), (16, 40, 1024), (5, 20, 8), (4, 64, 4104), (13, 50, 72)]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_against_64_bits(pkg, m, n, k, kind):
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(m + n + k)
    w, sw = _weight(n, k, g)
    x = (torch.randn(m, k, device=DEV, generator=g) * 3).to(dtype)
    bias = torch.randn(n, device=DEV, generator=g).to(dtype) if (m + n) % 2 else None
    q, sx = pkg.int8.quantize_rows(x)
    y = pkg.int8.linear_int8(x, w, sw / (100 * k ** 0.5), bias)
    assert y.shape == (m, n) and y.dtype == dtype
    _check(y, q, sx, w, sw / (100 * k ** 0.5), bias, dtype)
    again = pkg.int8.linear_int8(q, w, sw / (100 * k ** 0.5), bias, x_scale=sx, out_dtype=dtype)
    assert torch.equal(again, y)                                          # the same rows, quantized before


def test_integer_sums_are_exact(pkg):
    """Scales of 1 and fp32 results below 2^24: every output is the integer itself, at the extreme values too."""
    g = torch.Generator(device=DEV)
    g.manual_seed(21)
    for m, n, k in ((1, 64, 1000), (40, 200, 1040), (270, 300, 1000)):
        q = torch.randint(-127, 128, (m, (k + 15) // 16 * 16), device=DEV, generator=g, dtype=torch.int8)[:, :k]
        w, _ = _weight(n, k, g)
        q[0], w[0] = 127, -128
        y = pkg.int8.linear_int8(q, w, torch.ones(n, device=DEV), x_scale=torch.ones(m, device=DEV), out_dtype=torch.float32)
        assert torch.equal(y.double(), q.double() @ w.double().T)
    k = 131071                                                            # the longest sums: 127 * 127 * k = 0.98 * 2^31
    q = torch.full((2, k), 127, dtype=torch.int8, device=DEV)
    y = pkg.int8.linear_int8(q, torch.cat((q, -q)), torch.ones(4, device=DEV), x_scale=torch.ones(2, device=DEV), out_dtype=torch.float32)
    s = float(np.float32(127 * 127 * k))
    assert y.tolist() == [[s, s, -s, -s]] * 2


def test_layouts(pkg):
    """Leading dimensions, non-contiguous x, weights and rows whose layout has to be copied, a bias of another type, empty inputs, a wide stride."""
    g = torch.Generator(device=DEV)
    g.manual_seed(23)
    L = pkg.int8.linear_int8
    x = torch.randn(2, 5, 3, 200, device=DEV, generator=g).bfloat16()
    w, sw = _weight(40, 200, g)
    bias = torch.randn(40, device=DEV, generator=g)
    y = L(x, w, sw, bias)
    q, sx = pkg.int8.quantize_rows(x)
    assert y.shape == (2, 5, 3, 40) and q.shape == x.shape and sx.shape == (2, 5, 3)
    _check(y.view(30, 40), q.reshape(30, 200), sx.view(30), w, sw, bias.bfloat16(), torch.bfloat16)
    assert torch.equal(L(x.transpose(0, 2), w, sw, bias), y.transpose(0, 2))
    tight = w.contiguous()                                                # rows of 200 bytes: copied
    odd = torch.empty(40 * 200 + 3, dtype=torch.int8, device=DEV)[3:].view(40, 200).copy_(w)
    wide = torch.zeros(40, 512, dtype=torch.int8, device=DEV)
    wide[:, 96:296] = w
    for other in (tight, odd, wide[:, 96:296], w.t().contiguous().t()):
        assert torch.equal(L(x, other, sw, bias), y)
    assert torch.equal(L(q, w, sw, bias, x_scale=sx, out_dtype=torch.bfloat16), y)
    dirty = torch.full((30, 208), 99, dtype=torch.int8, device=DEV)       # 8-bit rows of the caller's own, with something behind column 200
    dirty[:, :200] = q.reshape(30, 200)
    assert torch.equal(L(dirty[:, :200], w, sw, bias, x_scale=sx.view(30), out_dtype=torch.bfloat16), y.view(30, 40))
    assert L(x[:0], w, sw).shape == (0, 5, 3, 40) and L(x, w[:0], sw[:0]).shape == (2, 5, 3, 0)
    assert L(x, w, sw, out_dtype=torch.float32).dtype == torch.float32


def test_refusals_on_the_gpu(pkg):
    L, no = pkg.int8.linear_int8, pkg.dequant.GGQUnsupported
    x = torch.zeros(2, 64, device=DEV, dtype=torch.float16)
    w, s = torch.zeros(8, 64, dtype=torch.int8, device=DEV), torch.ones(8, device=DEV)
    q, sx = pkg.int8.quantize_rows(x)
    for args, kw in (((x, w.half(), s), {}), ((x, w[0], s), {}), ((x, w, s[:7]), {}), ((x, w, s.half()), {}), ((x[:, :32], w, s), {}), ((x, w, s, s[:7]), {}), ((q, w, s), {}),
                     ((q, w, s), {"x_scale": sx}), ((q, w, s), {"x_scale": sx[:1], "out_dtype": x.dtype}), ((x, w, s), {"x_scale": sx}), ((x.double(), w, s), {}),
                     ((x, w, s), {"out_dtype": torch.float64}), ((x, w.cpu(), s), {}), ((x.cpu(), w, s), {}), ((x, w, s.cpu()), {})):
        with pytest.raises(no):
            L(*args, **kw)
    with pytest.raises(no, match="autograd"):
        L(x.clone().requires_grad_(), w, s)
    with pytest.raises(no):
        pkg.int8.quantize_rows(torch.zeros(2, 32769, device=DEV))


def test_the_layer(pkg):
    """GGMLInt8Linear from a packed weight: its 8-bit weight is within half a step of the unpacked one, forward is linear_int8, autograd takes F.linear."""
    Q, ops = pkg.qtypes.Q, pkg.ops
    blocks = pkg.synth.make_tensor_bytes(Q.Q4_K, (96, 1024), seed=3)
    w = ops.GGMLTensor(torch.from_numpy(blocks).to(DEV), tensor_type=Q.Q4_K, tensor_shape=(96, 1024))
    bias = torch.randn(96, device=DEV).half()
    layer = ops.GGMLInt8Linear(w, bias)
    dense = pkg.dequant.dequantize_tensor(w, torch.float16).double()
    # half a step, and the scale's own rounding times at most 127 steps: 0.5 s + 127 s 2^-24 < 0.5 s (1 + 2^-16)
    assert bool(((layer.weight.double() * layer.weight_scale.double()[:, None] - dense).abs() <= 0.5 * layer.weight_scale.double()[:, None] * (1 + 2.0 ** -16)).all())
    x = torch.randn(2, 40, 1024, device=DEV).half()
    assert torch.equal(layer(x), pkg.int8.linear_int8(x, layer.weight, layer.weight_scale, bias))
    x.requires_grad_()
    y = layer(x)
    y.sum().backward()
    values = (layer.weight.float() * layer.weight_scale[:, None]).half()
    assert torch.equal(x.grad, torch.autograd.grad(torch.nn.functional.linear(x, values, bias).sum(), x)[0])
