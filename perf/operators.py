"""Measured cases of the 16/32-bit operators around the 8-bit linears: layer norm, rotary positions and cross attention.

Each case is one pass through one operator as a program calls it. `run` computes the operator from elementary torch
operations in float32, or, with `own` set, through the functions of q8_kernels_amd.functional:

    layer_norm.layer_norm(x, weight, bias, eps)                            differentiable in x, weight and bias
    rotary.apply_rotary(q, k, positions, inv_freq, layout=, factor=)       differentiable in q and k
    cross_attention.cross_attention(q, k, v, kv_lens=, key_mask=)          differentiable in q, k and v

`exact` gives the same outputs in float64, from the definitions (gradients by automatic differentiation).
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the norm in front of a layer while one token of one sequence is decoded: a call's latency
        {"name": "norm, one token", "op": "norm", "type": "bf16", "wtype": "fp32", "rows": 1, "dim": 2048, "train": False},
        # a training step over two samples of 6144 tokens of the transformer block (hidden size 2048), float32 parameters
        {"name": "norm, train 12288x2048", "op": "norm", "type": "bf16", "wtype": "fp32", "rows": 12288, "dim": 2048, "train": True},
        # a float32 model of an odd width, ragged batch flattened to tokens: rows that start at any 4-byte address
        {"name": "norm, train 4099x1155 fp32", "op": "norm", "type": "fp32", "wtype": "fp32", "rows": 4099, "dim": 1155, "train": True},
        # decoding a batch of 16 sequences, far positions of a context stretched by a factor of 8
        {"name": "rotary, 16 single tokens", "op": "rotary", "type": "fp16", "batch": 16, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary_dim": 128, "layout": "half", "stretch": 8.0, "start": 90000, "train": False},
        # queries and keys of two samples of 6144 tokens, 32 heads of 64, as they leave their projections (token-major)
        {"name": "rotary, 2x6144 tokens", "op": "rotary", "type": "bf16", "batch": 2, "tokens": 6144, "heads": 32, "kv_heads": 32, "dim": 64,
         "rotary_dim": 64, "layout": "interleaved", "stretch": 1.0, "start": 0, "train": False},
        # a training step where half of each head is rotated, shared key heads, an odd number of tokens
        {"name": "rotary, train 4099 partial", "op": "rotary", "type": "bf16", "batch": 2, "tokens": 4099, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary_dim": 64, "layout": "half", "stretch": 4.0, "start": 1000, "train": True},
        # one decoder token of one sequence against 128 text states: a call's latency
        {"name": "attention, one token", "op": "attention", "type": "bf16", "batch": 1, "heads": 32, "kv_heads": 32, "queries": 1, "keys": 128, "dim": 64,
         "mask": "none", "train": False},
        # one decoder token of 8 sequences against long encoder states of ragged lengths, shared key heads
        {"name": "attention, 8 tokens, 8192 keys", "op": "attention", "type": "bf16", "batch": 8, "heads": 32, "kv_heads": 8, "queries": 1, "keys": 8192, "dim": 128,
         "mask": "lens", "train": False},
        # the block's cross attention: 6144 video tokens against 128 text states of ragged lengths
        {"name": "attention, 6144x128", "op": "attention", "type": "bf16", "batch": 2, "heads": 32, "kv_heads": 32, "queries": 6144, "keys": 128, "dim": 64,
         "mask": "lens", "train": False},
        # a prompt against the states of a long recording with dropped frames: odd lengths, a mask with holes
        {"name": "attention, 4099x1501 masked", "op": "attention", "type": "fp16", "batch": 2, "heads": 16, "kv_heads": 4, "queries": 4099, "keys": 1501, "dim": 128,
         "mask": "holes", "train": False},
        # a training step of the block's cross attention against 256 text states of ragged lengths
        {"name": "attention, train 6144x256", "op": "attention", "type": "bf16", "batch": 2, "heads": 32, "kv_heads": 32, "queries": 6144, "keys": 256, "dim": 64,
         "mask": "lens", "train": True},
        # a training step over long sequences on both sides, heads of 128, shared key heads: the largest
        {"name": "attention, train 4096x4096", "op": "attention", "type": "bf16", "batch": 2, "heads": 16, "kv_heads": 4, "queries": 4096, "keys": 4096, "dim": 128,
         "mask": "none", "train": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "rotary", "attention", "attention"))
    if op == "norm":
        kind = rng.choice(("bf16", "fp16", "fp32"))
        dim = _spread(rng, 17, 8192)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        rows = _spread(rng, 1, 16384)
        while rows * dim > 12288 * 4096:
            rows //= 2
        return {"op": op, "type": kind, "wtype": rng.choice(("fp32", kind)), "rows": rows, "dim": dim, "train": rng.random() < 0.6}
    if op == "rotary":
        dim = rng.choice((32, 48, 64, 80, 96, 128))
        kv_heads = rng.choice((1, 2, 4, 8))
        case = {"op": op, "type": rng.choice(("bf16", "fp16", "fp32")), "batch": _spread(rng, 1, 32), "tokens": _spread(rng, 1, 8192),
                "heads": kv_heads * rng.choice((1, 2, 4)), "kv_heads": kv_heads, "dim": dim, "rotary_dim": rng.choice((dim, dim, dim // 2)),
                "layout": rng.choice(("half", "interleaved")), "stretch": rng.choice((1.0, 2.0, 8.0, 32.0)), "start": _spread(rng, 1, 120000),
                "train": rng.random() < 0.5}
        while case["batch"] * case["tokens"] * (case["heads"] + kv_heads) * dim > 12288 * 64 * 128:
            case["batch" if case["batch"] > 1 else "tokens"] //= 2
        return case
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"op": op, "type": rng.choice(("bf16", "fp16")), "batch": _spread(rng, 1, 16), "heads": kv_heads * rng.choice((1, 2, 4, 8)), "kv_heads": kv_heads,
            "queries": rng.choice((1, _spread(rng, 1, 32), _spread(rng, 17, 8192), _spread(rng, 17, 8192))), "keys": _spread(rng, 1, 16384),
            "dim": rng.choice((32, 64, 64, 80, 96, 128, 128)), "mask": rng.choice(("none", "lens", "lens", "holes")), "train": False}
    if case["queries"] > 1 and rng.random() < 0.5:
        case["train"], case["keys"] = True, max(16, case["keys"])  # with a single key every score's gradient is zero
    while case["batch"] * case["heads"] * case["queries"] * case["keys"] * case["dim"] > 2 * 16 * 4096 * 4096 * 128 // 2:
        big = max(("batch", "queries", "keys"), key=lambda n: case[n] * (64 if n == "batch" else 1))
        case[big] //= 2
    return case


# ------------------------------------------------------------------------------------------------ inputs

def _frequencies(case):
    """Radians per position of each rotated pair, float64, and the factor of the rotated values: a context stretched by a factor keeps the fast pairs,
    interpolates the slow ones and blends those between, as a model's configuration says."""
    n = case["rotary_dim"] // 2
    f = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    s = case["stretch"]
    if s == 1.0:
        return f, 1.0
    turns = 4096.0 * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return f * keep + f / s * (1 - keep), 0.1 * math.log(s) + 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    dt = _TYPES[case["type"]]
    st = dict(case)
    train = case["train"]
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        # hidden states: some channels are much larger than the others, the mean is not zero
        size = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.01, 20.0, 1.0)
        st["x"] = ((normal(rows, dim) + 0.1 * normal(dim)) * size).to(dt).requires_grad_(train)
        wt = _TYPES[case["wtype"]]
        st["weight"] = (1.0 + 0.1 * normal(dim)).to(wt).requires_grad_(train)
        st["bias"] = (0.1 * normal(dim)).to(wt).requires_grad_(train)
        st["grad"] = normal(rows, dim).to(dt) if train else None
    elif case["op"] == "rotary":
        b, t, h, hk, d = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim"))
        # projections are token-major: the heads are a view of them
        st["q"], st["k"] = ((normal(b, t, n, d).to(dt).transpose(1, 2)).requires_grad_(train) for n in (h, hk))
        st["dq"], st["dk"] = ((normal(b, t, n, d).to(dt).transpose(1, 2)) if train else None for n in (h, hk))
        start = torch.randint(0, case["start"] + 1, (b, 1), generator=g, device="cuda")
        st["positions"] = start + torch.arange(t, device="cuda")
        freq, st["factor"] = _frequencies(case)
        st["inv_freq"] = freq.cuda()
    else:
        b, h, hk, m, n, d = (case[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
        st["q"] = normal(b, m, h, d).to(dt).transpose(1, 2).requires_grad_(train)
        st["k"] = normal(b, n, hk, d).to(dt).transpose(1, 2).requires_grad_(train)
        st["v"] = normal(b, n, hk, d).to(dt).transpose(1, 2).requires_grad_(train)
        st["grad"] = normal(b, m, h, d).to(dt).transpose(1, 2) if train else None
        st["kv_lens"] = st["key_mask"] = None
        if case["mask"] == "lens":
            st["kv_lens"] = torch.randint((n + 7) // 8, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        elif case["mask"] == "holes":
            st["key_mask"] = torch.rand((b, n), generator=g, device="cuda") < 0.9
    return st


# ------------------------------------------------------------------------------------------------ plain forms

def _norm(st):
    x, w, b = (st[n].detach().float() for n in ("x", "weight", "bias"))
    c = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    xh = c * rstd
    y = (xh * w + b).to(st["x"].dtype)
    if not st["train"]:
        return y
    g = st["grad"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return y, dx.to(st["x"].dtype), (g * xh).sum(0).to(st["weight"].dtype), g.sum(0).to(st["bias"].dtype)


def _rotate(x, c, s, layout):
    """c, s [B, 1, T, pairs]; the part of the head behind the pairs stays as it is."""
    n = c.shape[-1]
    f = x.detach().float()
    if layout == "half":
        a, b = f[..., :n], f[..., n:2 * n]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = f[..., 0:2 * n:2], f[..., 1:2 * n:2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((r, f[..., 2 * n:]), -1).to(x.dtype)


def _rotary(st):
    angle = (st["positions"].double()[:, None, :, None] * st["inv_freq"])
    c, s = (angle.cos() * st["factor"]).float(), (angle.sin() * st["factor"]).float()
    lay = st["layout"]
    out = _rotate(st["q"], c, s, lay), _rotate(st["k"], c, s, lay)
    if st["train"]:
        out += _rotate(st["dq"], c, -s, lay), _rotate(st["dk"], c, -s, lay)
    return out


def _attention(st):
    q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    b, h, m, d = q.shape
    hk, n = k.shape[1], k.shape[2]
    scale = d ** -0.5
    valid = None
    if st["kv_lens"] is not None:
        valid = (torch.arange(n, device=q.device) < st["kv_lens"][:, None])[:, None, None, :]
    elif st["key_mask"] is not None:
        valid = st["key_mask"][:, None, None, :]
    qf = q.float().reshape(b, hk, h // hk * m, d)  # the query heads that share a key head, one after the other
    kf, vf = k.float().contiguous(), v.float().contiguous()
    s = torch.matmul(qf, kf.transpose(2, 3)) * scale
    if valid is not None:
        s = torch.where(valid, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del s
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    of = torch.matmul(p, vf)
    o = of.reshape(b, h, m, d).to(q.dtype)
    if not st["train"]:
        return o
    g = st["grad"].float().reshape(qf.shape)
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = torch.matmul(g, vf.transpose(2, 3))
    ds = p * (ds - (g * of).sum(-1, keepdim=True)) * scale
    dq, dk = torch.matmul(ds, kf), torch.matmul(ds.transpose(2, 3), qf)
    return o, dq.reshape(q.shape).to(q.dtype), dk.to(k.dtype), dv.to(v.dtype)


# ------------------------------------------------------------------------------------------------ the framework's operators

def _own_norm(st):
    from q8_kernels_amd import functional as Q8F
    y = Q8F.layer_norm.layer_norm(st["x"], st["weight"], st["bias"], _EPS)
    if not st["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["grad"])


def _own_rotary(st):
    from q8_kernels_amd import functional as Q8F
    q, k = Q8F.rotary.apply_rotary(st["q"], st["k"], st["positions"], st["inv_freq"], layout=st["layout"], factor=st["factor"])
    if not st["train"]:
        return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))


def _own_attention(st):
    from q8_kernels_amd import functional as Q8F
    o = Q8F.cross_attention.cross_attention(st["q"], st["k"], st["v"], kv_lens=st["kv_lens"], key_mask=st["key_mask"])
    if not st["train"]:
        return o
    return (o.detach(),) + torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["grad"])


def run(state):
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "attention": _own_attention}[state["op"]](state)
    return {"norm": _norm, "rotary": _rotary, "attention": _attention}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = 4 if case["type"] == "fp32" else 2
    if case["op"] == "norm":
        n, w = case["rows"] * case["dim"], case["dim"] * (4 if case["wtype"] == "fp32" else 2)
        # forward: x in, y out; training adds the gradient in, dx out and the parameters' gradients
        return {"bytes": (4 if case["train"] else 2) * n * e + (4 if case["train"] else 2) * w, "flops": (20 if case["train"] else 8) * n}
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": (4 if case["train"] else 2) * n * e + 8 * case["batch"] * case["tokens"], "flops": (6 if case["train"] else 3) * n}
    b, h, hk, m, n, d = (case[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
    live = {"none": 1.0, "lens": 0.5625, "holes": 0.9}[case["mask"]] * n  # the keys that count, on average
    q, kv = b * h * m * d * e, b * hk * live * d * e
    # forward: q, k, v in, o out; training adds the gradient in and dq, dk, dv out, and five products to the two
    return {"bytes": (4 * q + 4 * kv) if case["train"] else (2 * q + 2 * kv), "flops": (14 if case["train"] else 4) * b * h * m * live * d}


# ------------------------------------------------------------------------------------------------ float64

def exact(case, seed):
    st = prepare(case, seed)
    train = case["train"]
    if case["op"] == "norm":
        x, w, b = (st[n].detach().double().requires_grad_(train) for n in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / (var + _EPS).sqrt() * w + b
        if not train:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), st["grad"].double())
    if case["op"] == "rotary":
        turn = torch.polar(torch.full((), st["factor"], dtype=torch.float64, device="cuda"),
                           st["positions"].double()[:, None, :, None] * st["inv_freq"])
        n = case["rotary_dim"] // 2

        def rotated(x, by):
            x = x.detach().double().contiguous()
            if case["layout"] == "half":
                z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * by
                return torch.cat((z.real, z.imag, x[..., 2 * n:]), -1)
            z = torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * by
            return torch.cat((torch.view_as_real(z).flatten(-2), x[..., 2 * n:]), -1)

        out = rotated(st["q"], turn), rotated(st["k"], turn)
        if train:
            out += rotated(st["dq"], turn.conj()), rotated(st["dk"], turn.conj())
        return out
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    b, h, m, d = q.shape
    each = h // k.shape[1]
    n = k.shape[2]
    o, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for i in range(b):
        if st["kv_lens"] is not None:
            at = torch.arange(int(st["kv_lens"][i]), device="cuda")
        elif st["key_mask"] is not None:
            at = st["key_mask"][i].nonzero()[:, 0]
        else:
            at = torch.arange(n, device="cuda")
        if not len(at):
            continue  # nothing to attend to: zeros
        for j in range(h):
            x, y, z = (t.clone().requires_grad_(train) for t in (q[i, j], k[i, j // each][at], v[i, j // each][at]))
            r = torch.softmax(x @ y.T / math.sqrt(d), -1) @ z
            o[i, j] = r.detach()
            if train:
                gx, gy, gz = torch.autograd.grad(r, (x, y, z), st["grad"][i, j].double())
                dq[i, j] = gx
                dk[i, j // each].index_add_(0, at, gy)
                dv[i, j // each].index_add_(0, at, gz)
    return (o, dq, dk, dv) if train else o
