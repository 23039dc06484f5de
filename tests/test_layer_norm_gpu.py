"""Layer norm against the definition in float64. Tolerances: the result's own rounding (half a step of its type) and the
fp32 arithmetic before it. A thread adds at most 32 elements and at most 10 more partial sums of other threads follow, so a
row sum is off by at most 42 roundings of the sum of magnitudes; E = 64 roundings covers it with the few operations around."""
import pytest
import torch

from q8_kernels_amd import _C, functional as Q8F
from q8_kernels_amd.modules import LayerNorm

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
E = 64 * 2.0 ** -24
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def half_step(t, dtype):
    return t.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype]


def reference(x, w, b, g, eps):
    """(y, dx, dw, db), their tolerances, in float64; x, g [rows, dim]"""
    x64, g64 = x.double(), g.double()
    wd = w.double() if w is not None else torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
    bd = b.double() if b is not None else torch.zeros_like(wd)
    mu = x64.mean(-1, keepdim=True)
    rs = (((x64 - mu) ** 2).mean(-1, keepdim=True) + eps) ** -0.5
    h = (x64 - mu) * rs
    y = h * wd + bd
    u = g64 * wd
    dx = rs * (u - u.mean(-1, keepdim=True) - h * (u * h).mean(-1, keepdim=True))
    dw, db = (g64 * h).sum(0), g64.sum(0)
    eh = E * (x64.abs().amax(-1, keepdim=True) * rs + h.abs())          # how far h may be off
    ey = eh * wd.abs() + E * (y.abs() + bd.abs())
    uh = (u * h).abs().mean(-1, keepdim=True)
    edx = rs * (E * (u.abs() + u.abs().mean(-1, keepdim=True) + h.abs() * uh) + eh * uh + h.abs() * (u.abs() * eh).mean(-1, keepdim=True)) + E * dx.abs()
    # the rows of a column: those of one thread, then its groups, the workgroups' sums by 32, and 32 of those; fewer than 160
    n = 160 * 2.0 ** -24
    edw = (g64.abs() * eh).sum(0) + n * (g64 * h).abs().sum(0)
    edb = n * g64.abs().sum(0)
    return (y, dx, dw, db), (ey, edx, edw, edb)


def check(x, w, b, g, eps=1e-5):
    x2, g2 = x.reshape(-1, x.shape[-1]), g.reshape(-1, x.shape[-1])
    want, tol = reference(x2, w, b, g2, eps)
    xl = x.detach().requires_grad_()
    wl, bl = (None if t is None else t.detach().clone().requires_grad_() for t in (w, b))
    y = Q8F.layer_norm.layer_norm(xl, wl, bl, eps)
    leaves = [t for t in (xl, wl, bl) if t is not None]
    grads = iter(torch.autograd.grad(y, leaves, g))
    got = [y, next(grads), next(grads) if w is not None else None, next(grads) if b is not None else None]
    assert torch.equal(y, Q8F.layer_norm.layer_norm(x, w, b, eps)), "without gradients: the same bits"
    for name, r, t, e in zip(("y", "dx", "dw", "db"), got, want, tol):
        if r is None:
            continue
        assert r.dtype == (x.dtype if name in ("y", "dx") else (w if w is not None else b).dtype)
        off = (r.detach().double().reshape(t.shape) - t).abs()
        lim = e + half_step(t, r.dtype) + half_step(e, r.dtype)
        assert (off <= lim).all(), "%s: off by %g of %g" % (name, off.max(), lim[off > lim].min())


def make(dev, rows, dim, dtype, wtype, seed=0, affine=(True, True)):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    x = (3 * rnd(rows, dim) + 5 * rnd(1, dim) + 2).to(dtype)
    w, b = (1 + 0.3 * rnd(dim)).to(wtype), rnd(dim).to(wtype)
    return x, w if affine[0] else None, b if affine[1] else None, rnd(rows, dim).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 2), (5, 7), (1, 8), (33, 64), (17, 127), (64, 128), (9, 136), (5, 511), (40, 512), (7, 1000),
                                      (6, 1155), (257, 2048), (5, 2056), (3, 4095), (12, 4096), (5, 8192), (2, 8200), (3, 16383), (2, 32768), (1, 32767)])
def test_lengths(dev, dtype, rows, dim):
    check(*make(dev, rows, dim, dtype, torch.float32, seed=rows * 131 + dim))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("affine", [(False, False), (True, False), (False, True)])
def test_missing_parameters_and_parameters_of_x_type(dev, dtype, affine):
    check(*make(dev, 50, 192, dtype, dtype, seed=5, affine=affine))
    check(*make(dev, 50, 192, dtype, dtype, seed=6))


@pytest.mark.parametrize("rows,dim", [(2500, 64), (3001, 768), (2311, 1155), (700, 12288)])
def test_many_rows(dev, rows, dim):
    check(*make(dev, rows, dim, torch.bfloat16, torch.float32, seed=rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1201, 2041), (1030, 4001), (611, 6144), (601, 6151), (530, 9001), (290, 16384), (517, 20000), (131, 30001)])
def test_many_long_rows(dev, dtype, rows, dim):
    check(*make(dev, rows, dim, dtype, torch.float32, seed=rows))


def test_long_rows_and_no_rows_or_one_gradient(dev):
    x, w, b, g = make(dev, 70, 20000, torch.bfloat16, torch.float32, seed=10)
    y, mean, rstd = _C.layer_norm(x, w, b)
    full = _C.layer_norm_backward(g, x, w, b, mean, rstd)
    for i in range(3):
        one = _C.layer_norm_backward(g, x, w, b, mean, rstd, [j == i for j in range(3)])
        assert all((one[j] is None) if j != i else torch.equal(one[j], full[j]) for j in range(3))
    none = _C.layer_norm_backward(g[:0], x[:0], w, b, mean[:0], rstd[:0])
    assert none[0].shape == (0, 20000) and (none[1] == 0).all() and (none[2] == 0).all()


def test_large_mean_does_not_cancel(dev):
    x, w, b, g = make(dev, 20, 512, torch.float32, torch.float32, seed=8)
    check(x * 1e-2 + 100.0, w, b, g)


def test_constant_rows(dev):
    x = torch.full((4, 640), 7.25, device=dev, dtype=torch.bfloat16)
    y = Q8F.layer_norm.layer_norm(x, None, torch.full((640,), 0.5, device=dev))
    assert (y == 0.5).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_odd_addresses(dev, dtype):
    wide, w, b, g = make(dev, 30, 520, dtype, torch.float32, seed=9)
    for lo, dim in ((0, 256), (8, 256), (1, 256), (3, 250)):          # a slice of a wider tensor, some of them off 16 bytes
        x = wide[:, lo:lo + dim]
        check(x, w[lo:lo + dim], b[:dim], g[:, :dim])
    x = wide[:, :512].reshape(5, 6, 512).transpose(0, 1)                # no row stride of its own: copied
    check(x, w[:512], b[:512], g[:, :512].reshape(6, 5, 512))
    check(wide[:1].expand(7, 520), w, b, g[:1].expand(7, 520))          # a broadcast input and a broadcast gradient


def test_no_rows(dev):
    x, w, b, _ = make(dev, 0, 96, torch.bfloat16, torch.float32)
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = Q8F.layer_norm.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 96) and (dw == 0).all() and (db == 0).all()


def test_only_what_is_needed(dev):
    x, w, b, g = make(dev, 60, 300, torch.float16, torch.float32, seed=11)
    y, mean, rstd = _C.layer_norm(x, w, b)
    every = _C.layer_norm_backward(g, x, w, b, mean, rstd)
    for k in range(3):
        some = _C.layer_norm_backward(g, x, w, b, mean, rstd, tuple(i == k for i in range(3)))
        assert [t is None for t in some] == [i != k for i in range(3)] and torch.equal(some[k], every[k])
    again = _C.layer_norm_backward(g, x, w, b, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(every, again))


def test_nan_and_infinity_stay_in_their_row(dev):
    x, w, b, _ = make(dev, 6, 700, torch.bfloat16, torch.float32, seed=12)
    clean = Q8F.layer_norm.layer_norm(x, w, b)
    x[2, 5], x[4, 699] = float("nan"), float("inf")
    y = Q8F.layer_norm.layer_norm(x, w, b)
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], clean[keep]) and y[2].isnan().all() and y[4].isnan().any()


def test_gradient_against_differences(dev):
    """f(x + t d) - f(x - t d) over 2 t, f = <g, layer_norm(x)>, in fp32: the values of f carry fp32 rounding (n outputs of
    size 1 with E each, divided by 2 t), and the third derivative adds t^2 of it, bounded by 6 |g| |d|^3 rstd^3 generously."""
    x, w, b, g = make(dev, 8, 320, torch.float32, torch.float32, seed=13)
    gen = torch.Generator(device=dev).manual_seed(3)
    t = 2.0 ** -6
    xl, wl, bl = (a.clone().requires_grad_() for a in (x, w, b))
    grads = torch.autograd.grad(Q8F.layer_norm.layer_norm(xl, wl, bl), (xl, wl, bl), g)
    f = lambda *a: (Q8F.layer_norm.layer_norm(*a).double() * g.double()).sum()  # noqa: E731
    y = Q8F.layer_norm.layer_norm(x, w, b)
    noise = (E * (y.abs() + w.abs() * 8 + b.abs()) * g.abs()).double().sum() / t
    for k in range(3):
        d = torch.randn(grads[k].shape, generator=gen, device=dev)
        d = d / d.norm(dim=-1, keepdim=True)
        up, down = ([a + t * d * s if i == k else a for i, a in enumerate((x, w, b))] for s in (1, -1))
        slope = (f(*up) - f(*down)) / (2 * t)
        want = (grads[k].double() * d.double()).sum()
        curve = 0.0 if k else 6 * t * t * float((g.double().norm(dim=-1) * (1 / x.double().std(-1)) ** 3).sum()) * float(w.abs().max())
        assert abs(float(slope - want)) <= float(noise) + curve


def test_captured_and_replayed(dev):
    x, w, b, g = make(dev, 300, 1024, torch.bfloat16, torch.float32, seed=14)
    y, mean, rstd = _C.layer_norm(x, w, b)
    _C.layer_norm_backward(g, x, w, b, mean, rstd)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yc, mc, rc = _C.layer_norm(x, w, b)
        out = _C.layer_norm_backward(g, x, w, b, mc, rc)
    for turn in range(3):
        x.copy_(make(dev, 300, 1024, torch.bfloat16, torch.float32, seed=20 + turn)[0])
        graph.replay()
        torch.cuda.synchronize()
        y, mean, rstd = _C.layer_norm(x, w, b)
        want = _C.layer_norm_backward(g, x, w, b, mean, rstd)
        assert torch.equal(yc, y) and all(torch.equal(p, q) for p, q in zip(out, want))


def test_another_stream(dev):
    x, w, b, g = make(dev, 500, 1024, torch.bfloat16, torch.float32, seed=15)
    y = Q8F.layer_norm.layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = Q8F.layer_norm.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ys)


def test_module(dev):
    m = LayerNorm(256, device=dev)
    x = torch.randn(4, 3, 256, device=dev, dtype=torch.bfloat16)
    m(x).float().sum().backward()
    assert m.weight.grad.shape == m.bias.grad.shape == (256,) and set(m.state_dict()) == {"weight", "bias"}
    assert list(LayerNorm(8, elementwise_affine=False).parameters()) == [] and LayerNorm(8, bias=False).bias is None


def test_refusals(dev):
    f = Q8F.layer_norm.layer_norm
    x = torch.randn(4, 64, device=dev, dtype=torch.bfloat16)
    w = torch.ones(64, device=dev)
    for bad in (lambda: f(x.to(torch.float8_e4m3fn)), lambda: f(x.double()), lambda: f(x, w.half()), lambda: f(x, w[:32]), lambda: f(x, w.cpu()),
                lambda: f(x.cpu()), lambda: f(x, w, w.bfloat16()), lambda: f(x[:, :0]), lambda: f(x, w, eps=-1.0), lambda: f(x, w, eps=float("nan")),
                lambda: f(torch.zeros(2, 32776, device=dev)), lambda: f(x, w[None])):
        with pytest.raises(RuntimeError):
            bad()
    y = f(x.requires_grad_(), w)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
