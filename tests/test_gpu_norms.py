"""norms.block_norm (include/ggq.h ggq_block_norm) on an MI355X, against the formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32) and e half a step of the result's type: r is one fp32 product and one sum, then rounded: e |r| + 2 u (|s| + |g h|).
A mean or a mean square adds dim positive terms in fp32, at most 64 in a lane, 6 steps over the wave, 8 over the waves and one product: 80 u of the sum
of magnitudes.  The norm's factor carries half of the mean square's error, the division and the root: 45 u; a layer norm's centred elements carry the
mean's 80 u mean|v| and one rounding.  Two norms (before and after) double that.  The modulation is four more roundings of its terms."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _norm64(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / (v.square().mean(-1, keepdim=True) + eps).sqrt()


def _formula(stream, branch, p, norm, post, eps):
    """(r, bound on r's error before rounding, y, bound on y's)."""
    s = stream.double()
    zero = torch.zeros_like(s)
    h, dh = (zero, zero) if branch is None else (branch.double(), zero)
    if post:
        mag = h.abs().mean(-1, keepdim=True)
        rms = (h.square().mean(-1, keepdim=True) + eps).sqrt() if post == "rms" else ((h - h.mean(-1, keepdim=True)).square().mean(-1, keepdim=True) + eps).sqrt()
        h = _norm64(h, post, eps)
        dh = 130 * U * h.abs() + (82 * U * mag / rms if post == "layer" else 0)
        if "post_weight" in p:
            h, dh = h * p["post_weight"].double(), dh * p["post_weight"].double().abs() + U * (h * p["post_weight"].double()).abs()
    if "gate" in p:
        h, dh = h * p["gate"].double(), dh * p["gate"].double().abs() + U * (h * p["gate"].double()).abs()
    r = s + h
    dr = dh + 2 * U * (s.abs() + h.abs())
    if norm is None:
        return r, dr, None, None
    mag = r.abs().mean(-1, keepdim=True)
    centred = r - r.mean(-1, keepdim=True) if norm == "layer" else r
    rms = (centred.square().mean(-1, keepdim=True) + eps).sqrt()
    y = centred / rms
    # an error of the rows moves the mean square by at most twice its own root mean square over the rows'
    dy = dr / rms + y.abs() * (130 * U + 2 * dr.square().mean(-1, keepdim=True).sqrt() / rms) + ((82 * U * mag + dr.mean(-1, keepdim=True)) / rms if norm == "layer" else 0)
    for name in ("weight", "bias", "scale", "shift"):
        if name in p:
            v = p[name].double()
            if name == "weight":
                y, dy = y * v, dy * v.abs()
            elif name == "scale":
                y, dy = y * (1 + v), dy * (1 + v).abs() + 2 * U * (y * (1 + v)).abs() + U * y.abs() * (1 + v.abs())
            else:
                y, dy = y + v, dy + U * v.abs()
            dy = dy + 2 * U * y.abs()
    return r, dr, y, dy


def _close(got, want, bound, dtype):
    e = torch.finfo(dtype).eps / 2
    tol = bound + e * (want.abs() + bound) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


CASES = [
    # batch, seq, dim, norm, post, parameters, which of them hold fp32
    (1, 1, 4096, "rms", None, ("weight",), ("weight",)),
    (2, 3, 2432, "layer", None, ("gate", "scale", "shift"), ()),
    (1, 2049, 256, "rms", "rms", ("gate", "post_weight", "weight"), ("post_weight", "weight")),         # a row per wave
    (3, 700, 513, "layer", "layer", ("gate", "scale", "shift", "post_weight", "weight", "bias"), ("bias", "gate")),
    (1, 5, 1, "rms", "rms", ("weight",), ()),
    (1, 7, 7, "layer", None, ("weight", "bias", "scale"), ("scale",)),
    (2, 2, 24576, "rms", None, ("weight", "shift"), ()),                                                # rows in LDS, the longest below
    (2, 3, 32768, "layer", "layer", ("gate", "weight", "bias", "scale"), ("weight", "gate")),
    (1, 9, 8193, "rms", "rms", ("gate", "post_weight"), ("post_weight",)),
    (5, 1001, 200, "rms", None, ("gate", "scale", "shift"), ()),                                        # a team's rows cross from sample to sample
    (900, 7, 1032, "layer", None, ("gate", "shift", "weight"), ()),
    (1, 300, 4097, "layer", None, (), ()),
    (1, 4, 1000, None, None, ("gate",), ()),                                                            # only the stream
    (2, 260, 5001, "layer", None, ("gate", "scale", "bias"), ("gate",)),                                # an odd length beyond the registers
    (1, 2500, 4100, "rms", None, ("gate", "weight"), ("weight",)),                                      # more than a wave's registers hold
]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_block_norm_against_the_formula(pkg, case, kind):
    batch, seq, dim, norm, post, names, wide = CASES[case]
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(100 + case)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    stream, branch = (2 * rand(batch, seq, dim) + 0.5).to(dtype), (rand(batch, seq, dim) - 0.25).to(dtype)
    mod = (0.5 * rand(batch, 3 * dim)).chunk(3, dim=-1)                       # strided, as chunks of one linear's output are
    mod16 = torch.cat(mod, -1).to(dtype).chunk(3, dim=-1)
    p = {}
    for i, n in enumerate(("gate", "scale", "shift")):
        if n in names:
            p[n] = (mod if n in wide else mod16)[i].unsqueeze(1)
    for n in ("weight", "bias", "post_weight"):
        if n in names:
            p[n] = (1 + 0.2 * rand(dim)).to(torch.float32 if n in wide else dtype)
    eps = 1e-5
    r, y = pkg.norms.block_norm(stream, branch, post_norm=post, norm=norm, eps=eps, **p)
    want_r, dr, want_y, dy = _formula(stream, branch, p, norm, post, eps)
    assert r.dtype == dtype and r.shape == stream.shape
    _close(r, want_r, dr, dtype)
    if norm is None:
        assert y is None
        return
    _close(y, want_y, dy, dtype)
    # without a branch: the stream itself, normed
    q = {k: v for k, v in p.items() if k not in ("gate", "post_weight")}
    same, y = pkg.norms.block_norm(stream, norm=norm, eps=eps, **q)
    assert same.data_ptr() == stream.data_ptr()
    _, _, want, d = _formula(stream, None, q, norm, None, eps)
    _close(y, want, d, dtype)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", [(1, 4096), (5, 33), (2100, 128), (3, 1), (300, 5000), (2, 24576)])
def test_eight_bit_rows_are_the_normed_rows(pkg, kind, shape):
    """q * q_scale is y to half a step of the row's grid (and y's own error), the padding behind the columns is zero."""
    dtype = DT[kind]
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    stream, branch = (torch.randn(*shape, device=DEV, generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.1 * torch.randn(shape[1], device=DEV, generator=g))
    r, (q, scale) = pkg.norms.block_norm(stream, branch, weight=w, quantize=True)
    assert q.dtype == torch.int8 and q.shape == stream.shape and scale.shape == stream.shape[:-1] and q.stride(0) % 16 == 0
    want_r, dr, want, d = _formula(stream, branch, {"weight": w}, "rms", None, 1e-6)
    _close(r, want_r, dr, dtype)
    top = want.abs().amax(-1, keepdim=True)
    d_top = d.amax(-1, keepdim=True)
    step = top / 127
    err = (q.double() * scale.double()[:, None] - want).abs()
    assert bool((err <= 0.5 * step * (1 + 4 * U) + 2 * d + 2 * d_top + 4 * U * top).all())
    assert bool(((scale.double()[:, None] - step).abs() <= d_top + 2 * U * step).all())
    pad = q.as_strided((shape[0], q.stride(0)), (q.stride(0), 1))[:, shape[1]:]
    assert not bool(pad.any())


def test_rows_of_their_own_kind(pkg):
    """Zeros, an infinity, a NaN, a row whose square overflows fp16: each row by itself, the others as if they were not there."""
    g = torch.Generator(device=DEV)
    g.manual_seed(9)
    x = torch.randn(6, 640, device=DEV, generator=g).half()
    x[1] = 0
    x[2, 17] = float("inf")
    x[3, 600] = float("nan")
    x[4] = 60000.0
    want = _norm64(x.double(), "rms", 1e-6)
    _, y = pkg.norms.block_norm(x)
    for i in (0, 5):
        _close(y[i], want[i], 200 * U * want[i].abs(), torch.float16)
    assert not bool(y[1].any()) and bool(y[3].isnan().all())
    assert bool(y[2, 17].isnan()) and not bool(y[2, :17].any())               # inf / inf, and finite / inf
    assert torch.equal(y[4], torch.ones_like(y[4]))
    _, (q, scale) = pkg.norms.block_norm(x, quantize=True)
    assert float(scale[1]) == 0 and not bool(q[1].any())
    assert bool(scale[2:4].isnan().all()) and not bool(q[2:4].any())
    assert bool((q[4] == 127).all()) and abs(float(scale[4]) * 127 - 1) < 1e-5


def test_layouts_that_are_not_the_usual_ones(pkg):
    """Non-contiguous stream and branch, per-token modulation, one vector for a batch, empty batches, a base that is not 16-byte aligned."""
    g = torch.Generator(device=DEV)
    g.manual_seed(11)
    big = torch.randn(4, 6, 2 * 320, device=DEV, generator=g).bfloat16()
    stream, branch = big[..., :320], big[..., 320:]
    gate = torch.randn(4, 6, 320, device=DEV, generator=g).bfloat16()
    shift = torch.randn(320, device=DEV, generator=g)
    r, y = pkg.norms.block_norm(stream, branch, gate=gate, shift=shift)
    want_r, dr, want, d = _formula(stream, branch, {"gate": gate, "shift": shift}, "rms", None, 1e-6)
    _close(r, want_r, dr, torch.bfloat16)
    _close(y, want, d, torch.bfloat16)
    flat = torch.randn(33 * 321 + 1, device=DEV, generator=g).half()[1:].view(33, 321)
    _, y = pkg.norms.block_norm(flat, norm="layer")
    _, _, want, d = _formula(flat, None, {}, "layer", None, 1e-6)
    _close(y, want, d, torch.float16)
    r, y = pkg.norms.block_norm(stream[:0], branch[:0])
    assert r.shape == y.shape == (0, 6, 320)
    r, (q, s) = pkg.norms.block_norm(stream[:, :0], branch[:, :0], quantize=True)
    assert q.shape == (4, 0, 320) and s.shape == (4, 0)


def test_refusals_on_the_gpu(pkg):
    B, no = pkg.norms.block_norm, pkg.dequant.GGQUnsupported
    x = torch.zeros(2, 3, 64, device=DEV, dtype=torch.float16)
    for bad in (dict(gate=x), dict(post_norm="rms"), dict(norm=None), dict(norm="batch"), dict(norm=None, weight=x[0, 0], branch=x), dict(branch=x.float()), dict(branch=x[:1]),
                dict(weight=x[0]), dict(branch=x, gate=x[0, :, :32]), dict(branch=x, gate=x[0]), dict(branch=x, gate=x, scale=x[:, :1]), dict(post_weight=x[0, 0], branch=x)):
        with pytest.raises(no):
            B(x, **bad)
    for other in (x.double(), x.cpu(), torch.zeros(2, 0, device=DEV), torch.zeros(1, 32769, device=DEV)):
        with pytest.raises(no):
            B(other)
    with pytest.raises(no, match="autograd"):
        B(x.clone().requires_grad_())
    with torch.no_grad():
        B(x.clone().requires_grad_())
