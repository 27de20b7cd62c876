"""The block operators together, as a transformer block on quantized weights runs them: residual + gate + norm into 8-bit rows, the integer product, the norm
behind it, the experts -- eagerly, captured into a graph and replayed, on a stream of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _stack(pkg, name, shape, seed):
    q = pkg.qtypes.Q[name]
    n = shape[0] * shape[1] * shape[2]
    b = pkg.synth.device_blocks(q, n // pkg.qtypes.block_geometry(q)[0], DEV, seed, mode="signed")
    return pkg.ops.GGMLTensor(b, tensor_type=q, tensor_shape=shape)


class Block:
    def __init__(self, pkg, dim=512, ff=768, experts=5):
        g = torch.Generator(device=DEV)
        g.manual_seed(71)
        self.pkg, self.dim = pkg, dim
        q = pkg.qtypes.Q.Q4_K
        w = pkg.ops.GGMLTensor(pkg.synth.device_blocks(q, dim * dim // 256, DEV, 5), tensor_type=q, tensor_shape=(dim, dim))
        self.proj = pkg.ops.GGMLInt8Linear(w)
        self.norm1, self.norm2 = (1 + 0.1 * torch.randn(dim, device=DEV, generator=g) for _ in range(2))
        self.experts = pkg.ops.GGMLMoE(torch.randn(experts, dim, device=DEV, generator=g) * 0.1, _stack(pkg, "Q4_K", (experts, ff, dim), 6), _stack(pkg, "Q4_K", (experts, ff, dim), 7),
                                       _stack(pkg, "Q6_K", (experts, dim, ff), 8), top_k=2)

    def __call__(self, stream, branch, mod):
        N, shift, scale, gate = self.pkg.norms.block_norm, *[m.unsqueeze(1) for m in mod.chunk(3, dim=-1)]
        stream, (q, s) = N(stream, branch, gate=gate, weight=self.norm1, scale=scale, shift=shift, quantize=True)
        h = self.pkg.int8.linear_int8(q, self.proj.weight, self.proj.weight_scale, x_scale=s, out_dtype=stream.dtype)
        stream, y = N(stream, h, gate=gate, post_norm="rms", weight=self.norm2)
        return N(stream, self.experts(y), gate=gate, norm=None)[0]


def _inputs(batch, seq, dim, dtype, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return [torch.randn(batch, seq, dim, device=DEV, generator=g).to(dtype) for _ in range(2)] + [(0.3 * torch.randn(batch, 3 * dim, device=DEV, generator=g)).to(dtype)]


def _plain(block, stream, branch, mod):
    """The same block in fp32 torch operations on the unpacked weights; 8-bit rows stay 8-bit rows."""
    pkg, f = block.pkg, torch.float32
    shift, scale, gate = [m.unsqueeze(1).float() for m in mod.chunk(3, dim=-1)]
    rms = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    r = stream.float() + gate * branch.float()
    y = rms(r) * block.norm1 * (1 + scale) + shift
    a = y.abs().amax(-1, keepdim=True)
    q = torch.round(127 * y / a)
    h = (q @ block.proj.weight.float().T) * (a / 127) * block.proj.weight_scale
    r = r + gate * rms(h)
    y = rms(r) * block.norm2
    return r + gate * block.experts._one_by_one(y)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,seq", [(1, 1), (3, 5), (2, 32), (1, 100)])
def test_the_block_against_torch(pkg, dtype, batch, seq):
    block = Block(pkg)
    args = _inputs(batch, seq, 512, dtype, 80 + seq)
    got, want = block(*args), _plain(block, *args)
    # the stream is rounded three times on its way, 8-bit steps flip where values were rounded to 16 bits before: relative to the whole, ten steps of the type
    assert float((got.float() - want).norm() / want.norm()) < 10 * torch.finfo(dtype).eps


def test_the_block_in_a_graph(pkg):
    """Captured once, replayed on new inputs with eager work between: every replay gives what an eager call gives, bit for bit; two graphs of one block do not
    disturb each other."""
    block = Block(pkg)
    static = [_inputs(2, 7, 512, torch.bfloat16, 1), _inputs(1, 20, 512, torch.bfloat16, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            block(*s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(*s)
        graphs.append(graph)
        outs.append(out)
    for round_ in range(4):
        for i, (b, n) in enumerate(((2, 7), (1, 20))):
            new = _inputs(b, n, 512, torch.bfloat16, 10 + 2 * round_ + i)
            for dst, src in zip(static[i], new):
                dst.copy_(src)
            graphs[i].replay()
            kept = outs[i].clone()
            assert torch.equal(block(*new), kept)
        torch.cuda.synchronize()


def test_the_block_on_another_stream(pkg):
    block = Block(pkg)
    args = _inputs(2, 9, 512, torch.float16, 3)
    want = block(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block(*args)
    side.synchronize()
    assert torch.equal(got, want)


def test_two_streams_at_once(pkg):
    """Calls that overlap on two streams do not share scratch memory: each gives what it gives alone."""
    block = Block(pkg)
    args = [_inputs(2, 9, 512, torch.float16, 3), _inputs(1, 30, 512, torch.float16, 4)]
    want = [block(*a) for a in args]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(block(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_under_torch_compile(pkg):
    """A compiled caller runs the same kernels (the calls are graph breaks) and gets the same bits."""
    block = Block(pkg)
    args = _inputs(2, 9, 512, torch.bfloat16, 3)
    want = block(*args)
    torch._dynamo.reset()
    got = torch.compile(lambda *a: block(*a), backend="eager")(*args)
    assert torch.equal(got, want)


def test_no_rows_and_rows_that_had_to_be_copied(pkg):
    norm = pkg.norms.block_norm
    none = torch.empty(0, 5, 64, device=DEV, dtype=torch.bfloat16)
    r, y = norm(none, none, scale=torch.empty(0, 1, 64, device=DEV), shift=torch.empty(0, 64, device=DEV))
    assert r.shape == y.shape == none.shape
    r, (q, s) = norm(torch.empty(2, 0, 64, device=DEV, dtype=torch.float16), gate=None, scale=torch.ones(2, 1, 64, device=DEV), quantize=True)
    assert q.shape == (2, 0, 64) and s.shape == (2, 0)
    x = torch.randn(64, 6, device=DEV, dtype=torch.bfloat16).t()
    r, y = norm(x)
    assert r is x and torch.equal(y, norm(x.contiguous())[1])
    assert pkg.int8.linear_int8(torch.empty(0, 64, device=DEV, dtype=torch.float16), *pkg.int8.quantize_rows(torch.ones(8, 64, device=DEV))).shape == (0, 8)
