"""The operators that a transformer block runs beside its quantized linears: what each computes, on which sizes it is timed.

    norm    the norms before and after a block, fused with the block's gate and the residual sum (norms.block_norm)
    int8    the product of 8-bit integers with a scale per token and per output channel (int8.linear_int8), also straight from the norm that
            precedes it ("chain")
    moe     a whole mixture-of-experts layer on packed GGUF expert weights, for a few tokens (moe.moe_layer)

With ``own`` false, run() computes them in elementary torch operations in 32 bits; with ``own`` true it calls the package.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
# ggml type id, elements per block, bytes per block
FORMATS = {"Q4_0": (2, 32, 18), "Q5_0": (6, 32, 22), "Q8_0": (8, 32, 34), "Q4_K": (12, 256, 144), "Q6_K": (14, 256, 210)}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one token of a text encoder of width 4096: the latency of a small call
        {"name": "norm one token", "op": "norm", "batch": 1, "seq": 1, "dim": 4096, "kind": "rms", "post": False, "modulated": False, "dtype": "bf16"},
        # a joint text / image block of width 2432, two samples with a modulation vector each, an odd number of tokens
        {"name": "norm joint block", "op": "norm", "batch": 2, "seq": 333, "dim": 2432, "kind": "layer", "post": False, "modulated": True, "dtype": "f16"},
        # image tokens of two samples through a block with a norm on either side and a gate
        {"name": "norm image block", "op": "norm", "batch": 2, "seq": 4608, "dim": 4096, "kind": "rms", "post": True, "modulated": True, "dtype": "bf16"},
        # a feed-forward projection for one token
        {"name": "int8 one token", "op": "int8", "m": 1, "n": 10240, "k": 4096, "bias": False, "dtype": "bf16"},
        # a text prompt of 77 tokens through a projection of width 2432
        {"name": "int8 short prompt", "op": "int8", "m": 77, "n": 9728, "k": 2432, "bias": True, "dtype": "f16"},
        # sizes that divide nothing
        {"name": "int8 ragged", "op": "int8", "m": 333, "n": 1501, "k": 1001, "bias": True, "dtype": "bf16"},
        # 512 text tokens through the feed-forward projection of width 4096
        {"name": "int8 text encoder", "op": "int8", "m": 512, "n": 10240, "k": 4096, "bias": False, "dtype": "bf16"},
        # image tokens through a feed-forward projection of width 2432
        {"name": "int8 image", "op": "int8", "m": 4608, "n": 9728, "k": 2432, "bias": True, "dtype": "bf16"},
        # residual, gate, norm and the projection behind them for the tokens of one image
        {"name": "norm into int8", "op": "chain", "batch": 1, "seq": 4608, "dim": 4096, "n": 10240, "kind": "rms", "post": False, "modulated": True, "dtype": "bf16"},
        # one token through two of eight wide experts
        {"name": "moe one token", "op": "moe", "tokens": 1, "experts": 8, "top_k": 2, "dim": 4096, "ff": 10240, "up": "Q4_K", "down": "Q6_K", "dtype": "bf16"},
        # a handful of sequences, one token each, through eight of 64 narrow experts
        {"name": "moe many experts", "op": "moe", "tokens": 7, "experts": 64, "top_k": 8, "dim": 2048, "ff": 1024, "up": "Q4_K", "down": "Q4_K", "dtype": "bf16"},
        # a short prompt through two of four experts whose widths are no multiples of 256, in the 32-element formats
        {"name": "moe short prompt", "op": "moe", "tokens": 33, "experts": 4, "top_k": 2, "dim": 2432, "ff": 6848, "up": "Q8_0", "down": "Q5_0", "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "int8", "int8", "moe", "moe"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "norm":
        dim = _log(rng, 64, 8192)
        dim = dim if rng.random() < 0.4 else max(8, dim // 8 * 8)
        batch = rng.choice([1, 1, 2, 3])
        return {"op": op, "batch": batch, "seq": max(1, min(_log(rng, 1, 4608), 2 * 4608 * 4096 // (batch * dim))), "dim": dim, "kind": rng.choice(["rms", "layer"]),
                "post": rng.random() < 0.5, "modulated": rng.random() < 0.6, "dtype": dtype}
    if op == "int8":
        n, k = _log(rng, 64, 16384), _log(rng, 64, 12288)
        k = k if rng.random() < 0.3 else max(32, k // 32 * 32)
        return {"op": op, "m": max(1, min(_log(rng, 1, 4608), 4608 * 9728 * 2432 // (n * k))), "n": n, "k": k, "bias": rng.random() < 0.5, "dtype": dtype}
    legacy = rng.random() < 0.4
    unit = 64 if legacy else 256
    dim, ff = max(1, _log(rng, 512, 4096) // unit) * unit, max(1, _log(rng, 512, 8192) // unit) * unit
    experts = min(_log(rng, 2, 64), 8 * 4096 * 10240 // (dim * ff))
    names = ["Q4_0", "Q5_0", "Q8_0"] if legacy else ["Q4_K", "Q6_K"]
    return {"op": "moe", "tokens": min(_log(rng, 1, 64), 64), "experts": experts, "top_k": rng.randint(1, min(8, experts)), "dim": dim, "ff": ff,
            "up": rng.choice(names), "down": rng.choice(names), "dtype": dtype}


def work(c):
    if c["op"] in ("norm", "chain"):
        rows = c["batch"] * c["seq"]
        if c["op"] == "norm":           # stream and block output in, stream and normed rows out
            return {"bytes": 8 * rows * c["dim"] + 6 * c["batch"] * c["dim"] * c["modulated"] + 4 * c["dim"], "flops": 10 * rows * c["dim"]}
        return {"bytes": 6 * rows * c["dim"] + c["n"] * c["dim"] + 2 * rows * c["n"], "flops": 2 * rows * c["dim"] * c["n"]}
    if c["op"] == "int8":
        return {"bytes": 2 * c["m"] * c["k"] + c["n"] * c["k"] + 2 * c["m"] * c["n"], "flops": 2 * c["m"] * c["n"] * c["k"]}
    # an expert's weights are read once where any token chose it: so many of them with routers that choose evenly
    busy = c["experts"] * (1 - (1 - c["top_k"] / c["experts"]) ** c["tokens"])
    per = lambda name: FORMATS[name][2] / FORMATS[name][1]  # noqa: E731
    packed = c["dim"] * c["ff"] * (2 * per(c["up"]) + per(c["down"]))
    return {"bytes": busy * packed + 2 * c["experts"] * c["dim"] + 4 * c["tokens"] * c["dim"],
            "flops": 2 * c["tokens"] * (c["top_k"] * 3 * c["dim"] * c["ff"] + c["experts"] * c["dim"])}


# ------------------------------------------------------------------------------------------------------------------ the inputs

def _packed(name, shape, std, g):
    """Packed blocks of random quants whose values have mean 0 and about the standard deviation `std`, as a byte tensor that says what it holds."""
    type_id, block, size = FORMATS[name]
    n = shape[0] * shape[1] * shape[2] // block
    b = torch.randint(0, 256, (n, size), dtype=torch.uint8, device=DEV, generator=g)
    spread = {"Q4_0": 4.6, "Q5_0": 9.2, "Q8_0": 74.0, "Q4_K": 240.0, "Q6_K": 1365.0}[name]
    d = ((0.75 + 0.5 * torch.rand(n, device=DEV, generator=g)) * (std / spread)).half()
    at = 208 if name == "Q6_K" else 0
    b[:, at:at + 2] = d.view(torch.uint8).view(n, 2)
    if name == "Q4_K":
        b[:, 2:4] = (7.5 * d.float()).half().view(torch.uint8).view(n, 2)       # the mins undo the mean of unsigned quants
    w = b.view(-1)
    w.tensor_type, w.tensor_shape = type_id, torch.Size(shape)
    return w


def _weight8(n, k, g):
    """An 8-bit weight as int8.quantize_rows lays it out: rows of k values, 16 bytes apart where k is odd."""
    q = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=DEV)
    q[:, :k] = (torch.randn(n, k, device=DEV, generator=g) * 36).round().clamp(-127, 127).to(torch.int8)
    return q[:, :k], (0.5 + torch.rand(n, device=DEV, generator=g)) * (1 / (36 * math.sqrt(k)))


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DT[c["dtype"]]
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    s = {"case": c}
    if c["op"] in ("norm", "chain"):
        b, d = c["batch"], c["dim"]
        s["stream"], s["branch"] = (rand(b, c["seq"], d) * 2).to(dt), rand(b, c["seq"], d).to(dt)
        s["weight"] = 1 + 0.1 * rand(d)                                             # norm weights are kept in 32 bits in GGUF files
        s["post_weight"] = 1 + 0.1 * rand(d) if c["post"] else None
        mod = (0.3 * rand(b, 3 * d)).to(dt)                                         # one modulation linear's output, cut in three
        s["gate"], s["shift"], s["scale"] = [m.unsqueeze(1) for m in mod.chunk(3, dim=-1)] if c["modulated"] else (None, None, None)
        if c["op"] == "chain":
            s["w8"], s["w8_scale"] = _weight8(c["n"], d, g)
    elif c["op"] == "int8":
        s["x"] = (rand(c["m"], c["k"]) * torch.exp(0.5 * rand(c["m"], 1))).to(dt)
        s["w8"], s["w8_scale"] = _weight8(c["n"], c["k"], g)
        s["bias"] = (0.1 * rand(c["n"])).to(dt) if c["bias"] else None
    else:
        e, d, ff = c["experts"], c["dim"], c["ff"]
        s["x"] = rand(c["tokens"], d).to(dt)
        s["router"] = (rand(e, d) * (1.5 / math.sqrt(d))).to(dt)
        s["w_gate"], s["w_up"] = (_packed(c["up"], (e, ff, d), 1 / math.sqrt(d), g) for _ in range(2))
        s["w_down"] = _packed(c["down"], (e, d, ff), 1 / math.sqrt(ff), g)
    return s


# ------------------------------------------------------------------------------------------------------------------ the plain forms

def _norm(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _block_norm(s, c):
    """(new residual stream, normed and modulated rows), both in 32 bits."""
    h = s["branch"].float()
    if c["post"]:
        h = _norm(h, c["kind"]) * s["post_weight"]
    if c["modulated"]:
        h = h * s["gate"].float()
    r = s["stream"].float() + h
    y = _norm(r, c["kind"]) * s["weight"]
    if c["modulated"]:
        y = y * (1 + s["scale"].float()) + s["shift"].float()
    return r, y


def _linear8(x, w8, w8_scale, bias):
    """x in 8 bits, one scale per row, times w8.  A row's quotients are formed in 64 bits: half-way values are common in 16-bit rows."""
    amax = x.abs().amax(-1, keepdim=True)
    q = torch.round(x.double() * 127 / amax.double().clamp_min(1e-300)).float()
    y = (q @ w8.float().T) * (amax.float() / 127) * w8_scale
    return y if bias is None else y + bias.float()


def _halves(b):
    return b.contiguous().view(torch.float16)


def _decode(w):
    """The fp16 values of a packed weight, in the formats' own operations: each product and difference is rounded to fp16."""
    shape = tuple(w.tensor_shape)
    name = next(n for n, f in FORMATS.items() if f[0] == w.tensor_type)
    b = w.view(-1, FORMATS[name][2])
    n = b.shape[0]
    if name == "Q8_0":
        v = _halves(b[:, :2]) * b[:, 2:].contiguous().view(torch.int8).half()
    elif name in ("Q4_0", "Q5_0"):
        d, qs = _halves(b[:, :2]), b[:, -16:]
        q = torch.cat((qs & 15, qs >> 4), 1)
        if name == "Q5_0":
            bits = (b[:, 2:6, None] >> torch.arange(8, dtype=torch.uint8, device=b.device)) & 1
            q = q | (bits.reshape(n, 32) << 4)
        v = d * (q.half() - (8 if name == "Q4_0" else 16))
    elif name == "Q4_K":
        d, dmin, s = _halves(b[:, 0:2]), _halves(b[:, 2:4]), b[:, 4:16]
        lo, mid, hi = s[:, 0:4], s[:, 4:8], s[:, 8:12]
        sc = torch.cat((lo & 63, (hi & 15) | ((lo >> 6) << 4)), 1).half()
        mn = torch.cat((mid & 63, (hi >> 4) | ((mid >> 6) << 4)), 1).half()
        qs = b[:, 16:].view(n, 4, 1, 32)
        q = torch.cat((qs & 15, qs >> 4), 2).view(n, 8, 32).half()
        v = (d * sc).view(n, 8, 1) * q - (dmin * mn).view(n, 8, 1)
    else:
        ql, qh = b[:, :128].view(n, 2, 2, 32), b[:, 128:192].view(n, 2, 1, 32)
        sc, d = b[:, 192:208].contiguous().view(torch.int8).half(), _halves(b[:, 208:210])
        q = torch.cat((ql & 15, ql >> 4), 2) | (((qh >> torch.tensor([0, 2, 4, 6], dtype=torch.uint8, device=b.device).view(1, 1, 4, 1)) & 3) << 4)
        v = (d * sc).view(n, 16, 1) * (q.view(n, 16, 16).half() - 32)
    return v.reshape(shape)


def _moe(s, c):
    x, dt = s["x"].float(), s["x"].dtype
    e, ff, d = c["experts"], c["ff"], c["dim"]
    # the choice is made in 64 bits, equal scores to the lower expert
    logits = s["x"].double() @ s["router"].double().T
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    top, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    top, ids = top[:, :c["top_k"]], ids[:, :c["top_k"]]
    top = (top / top.sum(-1, keepdim=True)).float()
    share = ((ids[:, :, None] == torch.arange(e, device=x.device)) * top[:, :, None]).sum(1)        # [tokens, experts]
    # a packed weight stands for its fp16 values in the type of the activations
    w_gate, w_up, w_down = (_decode(w).to(dt).float() for w in (s["w_gate"], s["w_up"], s["w_down"]))
    a = x @ w_gate.view(e * ff, d).T
    h = a / (1 + torch.exp(-a)) * (x @ w_up.view(e * ff, d).T)
    h = h.view(-1, e, ff) * share[:, :, None]
    return h.view(-1, e * ff) @ w_down.transpose(1, 2).reshape(e * ff, d)


def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    dt = DT[c["dtype"]]
    if c["op"] == "norm":
        r, y = _block_norm(s, c)
        return {"stream": r.to(dt), "y": y.to(dt)}
    if c["op"] == "chain":
        r, y = _block_norm(s, c)
        return {"stream": r.to(dt), "y": _linear8(y, s["w8"], s["w8_scale"], None).to(dt)}
    if c["op"] == "int8":
        return {"y": _linear8(s["x"], s["w8"], s["w8_scale"], s["bias"]).to(dt)}
    return {"y": _moe(s, c).to(dt)}


# ------------------------------------------------------------------------------------------------------------------ the package's calls

def _run_own(s, c):
    from ggq_pkg import load_package
    pkg = load_package()
    if c["op"] in ("norm", "chain"):
        r, y = pkg.norms.block_norm(s["stream"], s["branch"], gate=s["gate"], post_norm=c["kind"] if c["post"] else None, post_weight=s["post_weight"], norm=c["kind"],
                                    weight=s["weight"], scale=s["scale"], shift=s["shift"], eps=EPS, quantize=c["op"] == "chain")
        if c["op"] == "chain":
            y = pkg.int8.linear_int8(y[0], s["w8"], s["w8_scale"], x_scale=y[1], out_dtype=r.dtype)
        return {"stream": r, "y": y}
    if c["op"] == "int8":
        return {"y": pkg.int8.linear_int8(s["x"], s["w8"], s["w8_scale"], s["bias"])}
    return {"y": pkg.moe.moe_layer(s["x"], s["router"], s["w_gate"], s["w_up"], s["w_down"], top_k=c["top_k"])}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits

def _exact_norm(v, kind):
    centre = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
    v = v - centre
    return v / ((v.square().sum(-1, keepdim=True) / v.shape[-1]) + EPS).sqrt()


def _exact_linear8(x, w8, w8_scale, bias):
    top = x.abs().max(-1, keepdim=True).values
    # round half to even of 127 x / top, from whole numbers of half steps
    steps = 254 * x / torch.where(top > 0, top, torch.ones_like(top))
    below = torch.floor((steps + 1) / 2)
    q = below - ((steps == 2 * below - 1) & (torch.remainder(below, 2) == 1)).double()
    out = torch.matmul(q, w8.double().t()) * (top / 127) * w8_scale.double()[None, :]
    return out if bias is None else out + bias.double()


def _exact_values(raw, name):
    """float64 values of packed blocks [n, size]: bit by bit, one position of the block after the other."""
    i = raw.to(torch.int64)
    f16 = lambda lo: (i[:, lo] + 256 * i[:, lo + 1]).to(torch.int16).view(torch.float16).double()  # noqa: E731
    r16 = lambda v: v.half().double()  # noqa: E731
    s8 = lambda v: v - 256 * (v > 127)  # noqa: E731
    out = []
    if name == "Q8_0":
        return torch.stack([r16(f16(0) * s8(i[:, 2 + k])) for k in range(32)], 1)
    if name == "Q4_0":
        return torch.stack([r16(f16(0) * ((i[:, 2 + k % 16] // (16 if k >= 16 else 1)) % 16 - 8)) for k in range(32)], 1)
    if name == "Q5_0":
        fifth = i[:, 2] + (i[:, 3] << 8) + (i[:, 4] << 16) + (i[:, 5] << 24)
        return torch.stack([r16(f16(0) * ((i[:, 6 + k % 16] // (16 if k >= 16 else 1)) % 16 + 16 * ((fifth >> k) & 1) - 16)) for k in range(32)], 1)
    if name == "Q4_K":
        for sub in range(8):
            if sub < 4:
                sc, mn = i[:, 4 + sub] % 64, i[:, 8 + sub] % 64
            else:
                sc, mn = i[:, 8 + sub] % 16 + 16 * (i[:, sub] // 64), i[:, 8 + sub] // 16 + 16 * (i[:, 4 + sub] // 64)
            q = (i[:, 16 + 32 * (sub // 2):48 + 32 * (sub // 2)] // (16 if sub % 2 else 1)) % 16
            out.append(r16(r16(r16(f16(0) * sc)[:, None] * q) - r16(f16(2) * mn)[:, None]))
        return torch.cat(out, 1)
    for group in range(8):                                                                        # Q6_K: eight groups of 32
        half, part = group // 4, group % 4
        low = (i[:, 64 * half + 32 * (part % 2):][:, :32] // (16 if part >= 2 else 1)) % 16
        high = (i[:, 128 + 32 * half:][:, :32] // 4 ** part) % 4
        scale = s8(i[:, 192 + 2 * group:194 + 2 * group]).repeat_interleave(16, dim=1)
        out.append(r16(r16(f16(208)[:, None] * scale) * (low + 16 * high - 32)))
    return torch.cat(out, 1)


def _exact_weight(w, name, expert, dt):
    e, rows, cols = w.tensor_shape
    _, block, size = FORMATS[name]
    per = rows * cols // block
    v = _exact_values(w.view(e, per, size)[expert], name).reshape(rows, cols)
    return v.to(dt).double()


def exact(c, seed):
    s = prepare(c, seed)
    dt = DT[c["dtype"]]
    if c["op"] in ("norm", "chain"):
        f = {k: s[k].double() if s[k] is not None else None for k in ("stream", "branch", "weight", "post_weight", "gate", "shift", "scale")}
        h = f["branch"]
        if c["post"]:
            h = f["post_weight"] * _exact_norm(h, c["kind"])
        r = f["stream"] + (h if f["gate"] is None else f["gate"] * h)
        y = f["weight"] * _exact_norm(r, c["kind"])
        if f["scale"] is not None:
            y = y + f["scale"] * y + f["shift"]
        return {"stream": r, "y": y if c["op"] == "norm" else _exact_linear8(y.view(-1, c["dim"]), s["w8"], s["w8_scale"], None).view(c["batch"], c["seq"], c["n"])}
    if c["op"] == "int8":
        return {"y": _exact_linear8(s["x"].double(), s["w8"], s["w8_scale"], s["bias"])}
    x = s["x"].double()
    scores = torch.softmax((x[:, None, :] * s["router"].double()[None]).sum(-1), -1)
    order = torch.argsort(scores, dim=-1, descending=True, stable=True)[:, :c["top_k"]]
    share = scores.gather(1, order)
    share = share / share.sum(1, keepdim=True)
    y = torch.zeros(c["tokens"], c["dim"], dtype=torch.float64, device=x.device)
    for expert in sorted(set(order.flatten().tolist())):
        token, slot = torch.nonzero(order == expert, as_tuple=True)
        a = x[token] @ _exact_weight(s["w_gate"], c["up"], expert, dt).t()
        h = a * torch.sigmoid(a) * (x[token] @ _exact_weight(s["w_up"], c["up"], expert, dt).t())
        y.index_add_(0, token, share[token, slot][:, None] * (h @ _exact_weight(s["w_down"], c["down"], expert, dt).t()))
    return {"y": y}
