"""16-bit cross attention against its definition in float64, forward and gradients.

Tolerances, element by element, from the kernels' roundings. u = half a step of the type (2^-8 bf16, 2^-11 fp16); t = 2^-25 for
fp16, whose values below 2^-14 round to multiples of 2^-24 (0 for bf16). Scores are fp32 sums of D exact products: relative
error of p = exp(s) at most es = D 2^-23 scale sum|q k| + 2^-18 (the exponent's own fp32 rounding at |c s| below 2^4, exp2, and
the row sum) + N 2^-24; the probabilities entering a product round by u. With p normalised and l >= 1 the unnormalised sum:
  o:  (u + 2 es) sum_j p |v_j| + t sum_j |v_j| + half a step of o                           =: eo
  dv: (u + 2 es) sum_i p |g_i| + t sum_i |g_i| + half a step
  ds: |ds| (u + 2 es) + p (D 2^-23 sum|g v| + sum_d |g| eo + D 2^-23 sum|g o|) + t          =: eds
  dq: scale (sum_j eds |k_j| + N 2^-24 sum_j |ds k_j|) + half a step;  dk with the sums over the rows
Where at most 32 keys can count, delta is corrected by what the ds of its row add up to, which leaves the errors of that sum,
sum_j (es |ds_j| + p_j D 2^-23 sum|g v_j|), and 2 es of the correction itself, in the place of sum_d |g| eo + D 2^-23 sum|g o|."""
import pytest
import torch

from q8_kernels_amd import _C, functional as Q8F

pytestmark = pytest.mark.gpu
attend = Q8F.cross_attention.cross_attention
TYPES = [torch.bfloat16, torch.float16]


def reference(q, k, v, g, scale, valid, exact=False):
    """((o, dq, dk, dv), their tolerances) in float64; valid bool [B, N]"""
    b, h, m, d = q.shape
    hk, n = k.shape[1], k.shape[2]
    u = torch.finfo(q.dtype).eps / 2
    t = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134
    live = valid[:, None, :, None]
    q6, g6 = (x.double().reshape(b, hk, h // hk * m, d) for x in (q, g))
    k6, v6 = (torch.where(live, x.double(), 0.0) for x in (k, v))
    s = q6 @ k6.transpose(2, 3) * scale
    s = torch.where(valid[:, None, None, :], s, float("-inf"))
    top = s.amax(-1, keepdim=True) if n else torch.zeros_like(q6[..., :1])
    p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    es = 2 * (d * 2.0 ** -23 * scale * (q6.abs() @ k6.abs().transpose(2, 3)) + 2.0 ** -18 + n * 2.0 ** -24)
    half = lambda x: x.abs() * u + tiny  # noqa: E731
    o = p @ v6
    eo = (p * (u + es)) @ v6.abs() + t * v6.abs().sum(2, keepdim=True)
    eo = eo + half(o) + u * eo
    dv = p.transpose(2, 3) @ g6
    edv = (p * (u + es)).transpose(2, 3) @ g6.abs() + t * g6.abs().sum(2, keepdim=True)
    dp = g6 @ v6.transpose(2, 3)
    ds = p * (dp - (g6 * o).sum(-1, keepdim=True))
    edp = d * 2.0 ** -23 * (g6.abs() @ v6.abs().transpose(2, 3))
    edelta = (g6.abs() * (eo + d * 2.0 ** -23 * o.abs())).sum(-1, keepdim=True)
    if exact:
        edelta = (es * ds.abs() + p * edp).sum(-1, keepdim=True) + edelta * (es * (p > 0)).amax(-1, keepdim=True)
    eds = ds.abs() * (u + es) + p * (edp + edelta) + t
    dq, dk = scale * (ds @ k6), scale * (ds.transpose(2, 3) @ q6)
    edq = scale * (eds @ k6.abs() + n * 2.0 ** -24 * (ds.abs() @ k6.abs()))
    edk = scale * (eds.transpose(2, 3) @ q6.abs() + q6.shape[2] * 2.0 ** -24 * (ds.abs().transpose(2, 3) @ q6.abs()))
    edq, edk, edv = edq * (1 + u) + half(dq), edk * (1 + u) + half(dk), edv * (1 + u) + half(dv)
    edk, edv = torch.where(live, edk, 0.0), torch.where(live, edv, 0.0)
    back = lambda x: x.reshape(b, h, m, d)  # noqa: E731
    return (back(o), back(dq), dk, dv), (back(eo), back(edq), edk, edv)


def close(got, want, tol, what):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert (off <= tol).all(), "%s: off by %g where %g is allowed" % (what, (off - tol).max() + tol[off > tol].min(), tol[off > tol].min())


def check(q, k, v, scale=None, lens=None, mask=None, seed=0, grads=True, exact=False):
    b, n = k.shape[0], k.shape[2]
    valid = torch.ones(b, n, dtype=torch.bool, device=q.device)
    if lens is not None:
        valid = valid & (torch.arange(n, device=q.device) < lens[:, None])
    if mask is not None:
        valid = valid & mask
    gen = torch.Generator(device=q.device).manual_seed(seed)
    g = torch.randn(q.shape, generator=gen, device=q.device).to(q.dtype)
    want, tol = reference(q, k, v, g, scale if scale is not None else q.shape[-1] ** -0.5, valid, exact)
    out = attend(q, k, v, scale, lens, mask)
    assert out.dtype == q.dtype
    close(out, want[0], tol[0], "o")
    if not grads:
        return out
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = attend(*leaves, scale, lens, mask)
    assert torch.equal(o, out)
    got = torch.autograd.grad(o, leaves, g)
    for name, x, w, e in zip(("dq", "dk", "dv"), got, want[1:], tol[1:]):
        assert x.dtype == q.dtype
        close(x, w, e, name)
    dead = ~valid[:, None, :, None].expand(k.shape)
    assert (got[1][dead] == 0).all() and (got[2][dead] == 0).all()
    return out


def make(dev, b, h, hk, m, n, d, dtype, seed=0, token_major=True):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def one(heads, t):
        shape = (b, t, heads, d) if token_major else (b, heads, t, d)
        x = torch.randn(shape, generator=gen, device=dev).to(dtype)
        return x.transpose(1, 2) if token_major else x

    return one(h, m), one(hk, n), one(hk, n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 24, 32, 40, 64, 72, 80, 96, 104, 128])
def test_head_sizes(dev, dtype, d):
    check(*make(dev, 2, 4, 2, 70, 150, d, dtype, seed=d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (2, 31), (31, 1), (33, 32), (127, 129), (128, 128), (129, 127), (300, 257), (257, 700)])
def test_lengths(dev, dtype, m, n):
    check(*make(dev, 2, 2, 2, m, n, 64, dtype, seed=m * 1000 + n))


@pytest.mark.parametrize("b,h,hk,m,n,d", [(1, 1, 1, 1, 5000, 128), (3, 8, 1, 1, 3001, 64), (8, 32, 8, 1, 777, 128), (1, 6, 2, 18, 3000, 96), (2, 5, 5, 2999, 20, 64),
                                          (1, 16, 2, 640, 1100, 128), (1, 7, 7, 5, 4097, 32), (16, 4, 4, 3, 16, 64), (2, 24, 3, 100, 90, 80)])
def test_shared_heads_and_divided_walks(dev, b, h, hk, m, n, d):
    check(*make(dev, b, h, hk, m, n, d, torch.bfloat16, seed=n))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(1, 200), (1, 3000), (150, 200), (40, 3000)])
def test_lengths_of_keys(dev, dtype, m, n):
    q, k, v = make(dev, 7, 4, 2, m, n, 64, dtype, seed=3)
    lens = torch.tensor([0, 1, n, 64, 65, n - 1, n + 50], dtype=torch.int32, device=dev)
    out = check(q, k, v, lens=lens, seed=4)
    assert (out[0] == 0).all()
    close(out[1].double(), v[1, :, :1].repeat_interleave(2, 0).expand(4, m, 64).double(), torch.zeros(4, m, 64, device=dev, dtype=torch.float64), "one key: its value")
    neg = lens.clone()
    neg[0] = -5
    assert torch.equal(attend(q, k, v, None, neg), out)


@pytest.mark.parametrize("m,n", [(1, 130), (1, 4000), (90, 333)])
def test_masks_with_holes(dev, m, n):
    gen = torch.Generator(device=dev).manual_seed(n)
    q, k, v = make(dev, 4, 4, 2, m, n, 128, torch.bfloat16, seed=5)
    mask = torch.rand((4, n), generator=gen, device=dev) < 0.5
    mask[1] = False                                     # a row that leaves nothing
    mask[2] = False
    mask[2, n - 1] = True                               # only the last key
    out = check(q, k, v, mask=mask, seed=6)
    assert (out[1] == 0).all()
    lens = torch.tensor([n // 2, n, n - 1, 3], dtype=torch.int32, device=dev)
    out = check(q, k, v, lens=lens, mask=mask, seed=7)
    assert (out[2] == 0).all()
    wide = torch.zeros(4, 2 * n + 3, dtype=torch.bool, device=dev)   # rows at odd addresses, and every second byte
    wide[:, 1:n + 1] = mask
    assert torch.equal(attend(q, k, v, None, lens, wide[:, 1:n + 1]), out)
    wide[:, 0:2 * n:2] = mask
    assert torch.equal(attend(q, k, v, None, lens, wide[:, 0:2 * n:2]), out)
    check(q, k, v, mask=mask[:1].expand(4, n), seed=8)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 6e4])
def test_what_stands_in_keys_that_do_not_count(dev, bad):
    for m, n in ((1, 2100), (70, 190)):
        q, k, v = make(dev, 2, 4, 2, m, n, 64, torch.float16, seed=9)
        lens = torch.tensor([n - 37, 5], dtype=torch.int32, device=dev)
        mask = torch.ones(2, n, dtype=torch.bool, device=dev)
        mask[0, 3:40] = False
        clean = check(q, k, v, lens=lens, mask=mask, seed=10)
        dead = ~(mask & (torch.arange(n, device=dev) < lens[:, None]))[:, None, :, None].expand(k.shape)
        k2, v2 = k.masked_fill(dead, bad), v.masked_fill(dead, bad)
        g = torch.randn_like(q)
        one, two = ([x.detach().requires_grad_() for x in (q, *kv)] for kv in ((k, v), (k2, v2)))
        r1, r2 = ((o, *torch.autograd.grad(o, x, g)) for x in (one, two) for o in (attend(*x, None, lens, mask),))
        assert torch.equal(r1[0], clean) and all(torch.equal(a, c) for a, c in zip(r1, r2))


def test_scores_far_from_zero(dev):
    """Large scores of both signs: the maximum moves, and whole rows sit far below zero. |c s| stays below 2^7, where the
    exponent's fp32 rounding is 2^-17 (allowed: 2 * 2^-18)."""
    q, k, v = make(dev, 2, 2, 2, 100, 500, 64, torch.bfloat16, seed=11)
    for shift in (-30.0, 30.0):
        bias = torch.zeros_like(k)
        bias[..., 0] = shift
        q2 = q.clone()
        q2[..., 0] = 1.0
        check(q2, (k * 2 + bias).to(k.dtype), v, seed=12)
    rising = (k * torch.linspace(0.0, 4.0, 500, device=dev)[None, None, :, None]).to(k.dtype)
    check(q, rising, v, seed=13)
    check(q, k, v, scale=0.7, seed=14)


def test_nan_in_a_key_that_counts(dev):
    q, k, v = make(dev, 1, 1, 1, 40, 100, 64, torch.bfloat16, seed=15)
    k[0, 0, 70, 3] = float("nan")
    assert attend(q, k, v).isnan().all()
    assert not attend(q, k, v, None, torch.tensor([70], dtype=torch.int32, device=dev)).isnan().any()
    q[0, 0, 5, 1] = float("nan")
    out = attend(q, k, v, None, torch.tensor([70], dtype=torch.int32, device=dev))
    assert out[0, 0, 5].isnan().all() and not out[0, 0, :5].isnan().any() and not out[0, 0, 6:].isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_orders(dev, dtype):
    gen = torch.Generator(device=dev).manual_seed(16)
    rnd = lambda *s: torch.randn(s, generator=gen, device=dev).to(dtype)  # noqa: E731
    q = rnd(2, 4, 50, 64)
    kv = rnd(2, 90, 2, 4, 64)                                       # one projection of keys and values, token-major
    check(q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2))
    qkv = rnd(2, 60, 3, 4, 64)
    check(*(qkv[:, :, i].transpose(1, 2) for i in range(3)))
    wide = rnd(2, 4, 90, 72)
    check(q, wide[..., 8:], wide[..., 3:67])                        # the second off 16 bytes: copied
    check(q, rnd(2, 4, 64, 90).transpose(2, 3), rnd(2, 4, 90, 128)[..., ::2])
    check(q[:1].expand(2, 4, 50, 64), rnd(1, 4, 90, 64).expand(2, 4, 90, 64), rnd(2, 1, 90, 64).expand(2, 4, 90, 64))  # broadcast
    flat = rnd(2 * 4 * 90 * 64 + 4)[4:].view(2, 4, 90, 64)
    check(q, flat, flat)
    out = attend(qkv[:, :, 0].transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2))
    assert out.transpose(1, 2).is_contiguous()                      # the memory order of q


def test_gradients_of_broadcast_inputs(dev):
    q, k, v = make(dev, 3, 2, 2, 20, 40, 64, torch.bfloat16, seed=17)
    one = k[:1].detach().requires_grad_()
    o = attend(q, one.expand_as(k), v)
    (dk,) = torch.autograd.grad(o, one, torch.ones_like(o))
    each = one.detach().expand_as(k).contiguous().requires_grad_()
    o2 = attend(q, each, v)
    (dk2,) = torch.autograd.grad(o2, each, torch.ones_like(o2))
    # the sum of the three batch elements' gradients, rounded at each of two additions and once at the end
    assert ((dk.double() - dk2.double().sum(0, keepdim=True)).abs() <= 3 * 2.0 ** -8 * dk2.double().abs().sum(0, keepdim=True)).all()


def test_offsets_beyond_32_bits(dev):
    """Keys 2^23 elements apart: 300 of them reach 2.5e9 elements, 5e9 bytes."""
    buf = torch.empty(300 * 2 ** 23, dtype=torch.float16, device=dev)
    q, k, v = make(dev, 1, 2, 1, 9, 300, 64, torch.float16, seed=18)
    far = buf.as_strided((1, 1, 300, 64), (0, 64, 2 ** 23, 1))
    far.copy_(k)
    check(q, far, v)
    far.copy_(v)
    check(q, k, far)


def test_nothing_to_attend_and_nothing_to_do(dev):
    for b, h, m, n in ((2, 4, 5, 0), (2, 4, 0, 7), (0, 4, 5, 7), (1, 2, 0, 0)):
        q, k, v = (x.detach().requires_grad_() for x in make(dev, b, h, h, m, n, 64, torch.bfloat16))
        o = attend(q, k, v)
        grads = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
        assert (o == 0).all() and all(x.shape == g.shape and (g == 0).all() for x, g in zip((q, k, v), grads))


def test_same_bits_every_time(dev):
    q, k, v = make(dev, 2, 4, 2, 600, 900, 128, torch.bfloat16, seed=19)
    g = torch.randn_like(q)
    o, lse = _C.cross_attention(q, k, v, 0.1)
    first = _C.cross_attention_backward(g, q, k, v, o, lse, 0.1)
    for _ in range(3):
        o2, lse2 = _C.cross_attention(q, k, v, 0.1)
        again = _C.cross_attention_backward(g, q, k, v, o2, lse2, 0.1)
        assert torch.equal(o, o2) and torch.equal(lse, lse2) and all(torch.equal(a, b) for a, b in zip(first, again))


def test_gradient_against_differences(dev):
    """The output is linear in v: <g, f(v + d) - f(v - d)> = 2 <dv, d> up to the roundings of both (each output's and each
    gradient element's tolerance). For q and k a step of 2^-4: the same roundings, and a third-order term below
    (scale |d| |k|)^3 / 3 of the outputs' size."""
    q, k, v = make(dev, 1, 1, 1, 8, 16, 64, torch.float16, seed=20)
    d = {n: (torch.randn_like(x) * 2.0 ** -4).half() for n, x in zip("qkv", (q, k, v))}
    g = torch.randn_like(q)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(attend(*leaves), leaves, g)
    valid = torch.ones(1, 16, dtype=torch.bool, device=dev)
    for i, n in enumerate("qkv"):
        up, down = ([x + s * d[n] if j == i else x for j, x in enumerate((q, k, v))] for s in (1, -1))
        diff = (g.double() * (attend(*up).double() - attend(*down).double())).sum()
        step = (up[i].double() - down[i].double())                 # what the type made of the step
        noise = sum((g.double().abs() * reference(*x, g, 0.125, valid)[1][0]).sum() for x in (up, down))
        noise = noise + (reference(q, k, v, g, 0.125, valid)[1][i + 1] * step.abs()).sum()
        other = k if n == "q" else q
        bend = 0.0 if n == "v" else float(g.double().abs().sum() * v.double().abs().max()) * (0.125 * float(step.norm(dim=-1).max()) / 2 * float(other.double().norm(dim=-1).max())) ** 3
        assert abs(float(diff - (grads[i].double() * step).sum())) <= float(noise) + bend


def test_captured_and_replayed(dev):
    """Two graphs with workspaces of their own, replayed in turn with eager work between, against eager results."""
    sets, graphs = [make(dev, 1, 8, 2, 3, 2500, 128, torch.bfloat16, seed=s) for s in (21, 22)], []
    lens = torch.tensor([2500], dtype=torch.int32, device=dev)
    g = torch.randn_like(sets[0][0])

    def step(q, k, v):
        o, lse = _C.cross_attention(q, k, v, 0.09, lens)
        return [o, lse] + _C.cross_attention_backward(g, q, k, v, o, lse, 0.09, lens)

    for s in sets:
        step(*s)
    torch.cuda.synchronize()
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*s)
        graphs.append((graph, out))
    for turn in range(3):
        lens.fill_(2500 - 700 * turn)
        for s in sets:
            s[0].add_(0.125)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), s in zip(graphs, sets):
            assert all(torch.equal(a, b) for a, b in zip(out, step(*s)))


def test_another_stream(dev):
    q, k, v = make(dev, 1, 4, 4, 50, 3000, 64, torch.bfloat16, seed=23)
    out = attend(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [attend(q, k, v) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(out, o) for o in other)


def test_refusals(dev):
    q, k, v = make(dev, 2, 4, 2, 5, 9, 64, torch.bfloat16)
    lens, mask = torch.full((2,), 9, dtype=torch.int32, device=dev), torch.ones(2, 9, dtype=torch.bool, device=dev)
    for bad in (lambda: attend(q.float(), k.float(), v.float()), lambda: attend(q, k.half(), v), lambda: attend(q, k, v[:, :, :8]), lambda: attend(q[0], k[0], v[0]),
                lambda: attend(q[..., :60], k[..., :60], v[..., :60]), lambda: attend(q[:, :3], k, v), lambda: attend(q[:1], k, v),
                lambda: attend(q.cpu(), k.cpu(), v.cpu()), lambda: attend(q, k, v, 0.0), lambda: attend(q, k, v, -1.0), lambda: attend(q, k, v, float("inf")),
                lambda: attend(q, k, v, float("nan")), lambda: attend(q, k, v, None, lens.long()), lambda: attend(q, k, v, None, lens[:1]),
                lambda: attend(q, k, v, None, lens.cpu()), lambda: attend(q, k, v, None, None, mask.int()), lambda: attend(q, k, v, None, None, mask[:, :8]),
                lambda: attend(q, k, v, None, None, mask.float()), lambda: attend(q, k[:, :0], v[:, :0]),
                lambda: attend(*(torch.zeros(1, 1, 2, 136, dtype=torch.half, device=dev),) * 3)):
        with pytest.raises(RuntimeError):
            bad()
    x = q.detach().requires_grad_()
    (dq,) = torch.autograd.grad(attend(x, k, v), x, torch.ones_like(q), create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()


@pytest.mark.parametrize("b,h,hk,m,n,d,dtype", [(2, 32, 32, 1700, 128, 64, torch.bfloat16), (3, 16, 4, 2311, 77, 64, torch.float16), (1, 48, 48, 2100, 256, 64, torch.bfloat16),
                                                (2, 24, 24, 2050, 200, 40, torch.float16), (4, 16, 8, 1601, 1, 32, torch.bfloat16), (2, 40, 5, 1300, 129, 24, torch.bfloat16)])
def test_few_keys_and_many_rows(dev, b, h, hk, m, n, d, dtype):
    gen = torch.Generator(device=dev).manual_seed(n)
    q, k, v = make(dev, b, h, hk, m, n, d, dtype, seed=n)
    check(q, k, v, seed=1)
    lens = torch.randint(0, n + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
    lens[0] = 0 if b > 1 else n
    mask = torch.rand((b, n), generator=gen, device=dev) < 0.6
    check(q, k, v, lens=lens, seed=2, grads=False)
    out = check(q, k, v, lens=lens, mask=mask, seed=3, grads=False)
    dead = ~(mask & (torch.arange(n, device=dev) < lens[:, None]))[:, None, :, None].expand(k.shape)
    assert torch.equal(out, attend(q, k.masked_fill(dead, float("nan")), v.masked_fill(dead, float("inf")), None, lens, mask))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,n,lens", [(64, 2, None), (64, 32, None), (24, 100, [1, 2, 32]), (64, 200, [5, 0, 31]), (64, 700, [2, 3, 32]), (128, 2, None), (128, 8, None),
                                      (96, 65, [7, 32, 1]), (128, 900, [16, 2, 9])])
def test_gradients_of_few_counted_keys(dev, dtype, d, n, lens):
    q, k, v = make(dev, 3, 4, 2, 133, n, d, dtype, seed=n)
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    check(q, k, v, lens=lens, seed=5, exact=True)
    check(q, k, v, lens=lens, mask=torch.arange(n, device=dev).expand(3, n) % 3 != 1, seed=6, exact=True)


@pytest.mark.parametrize("b,h,hk,m,n,d,dtype", [(2, 16, 16, 2100, 256, 128, torch.bfloat16), (1, 20, 10, 1300, 128, 128, torch.float16), (3, 16, 4, 700, 100, 96, torch.bfloat16),
                                                (2, 32, 32, 1100, 200, 80, torch.float16), (2, 32, 8, 1025, 256, 96, torch.bfloat16), (1, 6, 2, 77, 33, 104, torch.float16),
                                                (2, 16, 16, 2050, 255, 64, torch.bfloat16), (1, 4, 4, 33, 65, 128, torch.bfloat16)])
def test_gradients_of_few_keys(dev, b, h, hk, m, n, d, dtype):
    gen = torch.Generator(device=dev).manual_seed(n)
    q, k, v = make(dev, b, h, hk, m, n, d, dtype, seed=n + 1)
    check(q, k, v, seed=1)
    lens = torch.randint(33, n + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
    mask = torch.rand((b, n), generator=gen, device=dev) < 0.7
    check(q, k, v, lens=lens, mask=mask, seed=2)
    # what stands in keys that do not count is not looked at
    dead = ~(mask & (torch.arange(n, device=dev) < lens[:, None]))[:, None, :, None].expand(k.shape)
    g = torch.randn_like(q)
    o, lse = _C.cross_attention(q, k, v, 0.1, lens, mask)
    a = _C.cross_attention_backward(g, q, k, v, o, lse, 0.1, lens, mask)
    c = _C.cross_attention_backward(g, q, k.masked_fill(dead, float("inf")), v.masked_fill(dead, float("nan")), o, lse, 0.1, lens, mask)
    assert all(torch.equal(x, y) for x, y in zip(a, c))


@pytest.mark.parametrize("n", [90, 300])
def test_rows_beyond_32_bits(dev, n):
    """Queries, outputs and their gradients 2^23 elements apart, one after the other in a buffer of 5e9 bytes: the same bits as side by side."""
    q, k, v = make(dev, 1, 2, 2, 300, n, 64, torch.bfloat16, seed=24)
    g = torch.randn_like(q)
    o, lse = _C.cross_attention(q, k, v, 0.1)
    want = _C.cross_attention_backward(g, q, k, v, o, lse, 0.1)
    far = torch.empty(300 * 2 ** 23, dtype=torch.bfloat16, device=dev).as_strided((1, 2, 300, 64), (0, 64, 2 ** 23, 1))
    for i in range(3):
        side = [q, o, g]
        far.copy_(side[i])
        side[i] = far
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(_C.cross_attention(far, k, v, 0.1), (o, lse)))
        got = _C.cross_attention_backward(side[2], side[0], k, v, side[1], lse, 0.1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
