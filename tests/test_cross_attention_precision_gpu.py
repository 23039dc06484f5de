"""16-bit cross attention: how exact its gradients are where the roundings inside it could show.

Against the definition in float64, in two ways. u = half a step of the type (2^-8 bf16, 2^-11 fp16).

Element by element: scores are fp32 sums, so p = exp(s) is off by at most es = 2 (D 2^-23 scale sum|q k| + 2^-22 max(4, |c s|)
+ N 2^-24) of itself (products, exponent and its difference from the log-sum, row sum); dS is rounded once where it enters a
product, the result once at the end. delta = rowsum(dO O) has O from probabilities that were rounded for their product and are
normalised by the sum of the rounded ones, so with relative roundings r_j it is off by sum_j r_j ds_j, and O itself, kept with 8
bits more than its type has, by eo = u / 2^8 |O| (next to a tie twice that). Those are bits of its fp32 code, which cannot reach
across the step 2^-24 of float16 below 2^-14: there it is off by half that step, as O itself is.
  edelta: sum_j (u + 2 es) |ds_j| + sum_d |g| (eo + 2 es sum_j p |v|) + D 2^-23 sum_d |g o|
  ds: (u + 2 es) |ds| + p (D 2^-23 sum_d |g v| + edelta);  dq, dk: the sums of that and of fp32 additions, and half a step.

All elements together: a value x that is rounded to 16 bits is off by h(x) / sqrt(3) in the square mean, where h(x) is half its
step. dq has the roundings of its ds, of delta (u / sqrt(3) |ds_j| each, at most) and of the result. Their squares add up, for
they are independent; the sum over some 10^4 elements scatters by a few percent, so the square mean error may be 1.1 times that
root. Beside it stand the fp32 errors: a few 2^-24 of what is added up, with signs of their own, 2^-20 of p |g| |v| in a ds
and of p in a dv."""
import pytest
import torch

from q8_kernels_amd import _C, functional as Q8F

pytestmark = pytest.mark.gpu
attend = Q8F.cross_attention.cross_attention
TYPES = [torch.bfloat16, torch.float16]


def half_step(x, dtype):
    info = torch.finfo(dtype)
    e = torch.floor(torch.log2(x.abs().clamp_min(info.tiny)))
    return torch.exp2(e) * (info.eps / 2)


def definition(q, k, v, g, scale, valid):
    """dq, dk, dv: value, element tolerance, square mean error allowed; and the same of o without the last"""
    b, h, m, d = q.shape
    hk, n = k.shape[1], k.shape[2]
    dtype, u = q.dtype, torch.finfo(q.dtype).eps / 2
    live = valid[:, None, :, None]
    q6, g6 = (x.double().reshape(b, hk, h // hk * m, d) for x in (q, g))
    k6, v6 = (torch.where(live, x.double(), 0.0) for x in (k, v))
    s = q6 @ k6.transpose(2, 3) * scale
    p = torch.softmax(torch.where(valid[:, None, None, :], s, float("-inf")), -1)
    es = 2 * (d * 2.0 ** -23 * scale * (q6.abs() @ k6.abs().transpose(2, 3)) + 2.0 ** -22 * (1.45 * s.abs()).clamp_min(4.0).amax(-1, keepdim=True) + n * 2.0 ** -24)
    o, dp = p @ v6, g6 @ v6.transpose(2, 3)
    ds = p * (dp - (g6 * o).sum(-1, keepdim=True))
    dq, dk, dv = scale * (ds @ k6), scale * (ds.transpose(2, 3) @ q6), p.transpose(2, 3) @ g6

    eo = o.abs() * u / 128
    rough = 2.0 ** -25 * (o.abs() < 2.0 ** -14) * (dtype == torch.float16)
    mag = (p * (1 + es)) @ v6.abs()
    edelta = ((u + 2 * es) * ds.abs()).sum(-1, keepdim=True) + (g6.abs() * (eo + rough + 2 * es.amax(-1, keepdim=True) * mag + d * 2.0 ** -23 * o.abs())).sum(-1, keepdim=True)
    eds = ds.abs() * (u + 2 * es) + p * (d * 2.0 ** -23 * (g6.abs() @ v6.abs().transpose(2, 3)) + edelta)
    edq = scale * (eds @ k6.abs() + n * 2.0 ** -24 * (ds.abs() @ k6.abs()))
    edk = scale * (eds.transpose(2, 3) @ q6.abs() + q6.shape[2] * 2.0 ** -24 * (ds.abs().transpose(2, 3) @ q6.abs()))
    edv = (p * (u + 2 * es)).transpose(2, 3) @ g6.abs() + q6.shape[2] * 2.0 ** -24 * (p.transpose(2, 3) @ g6.abs())
    full = [e * (1 + u) + half_step(x, dtype) for e, x in zip((edq, edk, edv), (dq, dk, dv))]
    small = 2.0 ** -20 * p * (g6.norm(dim=-1, keepdim=True) * v6.norm(dim=-1).unsqueeze(2))
    fine = (scale * (small @ k6.abs()), scale * (small.transpose(2, 3) @ q6.abs()), 2.0 ** -20 * (p.transpose(2, 3) @ g6.abs()))
    third = lambda x: half_step(x, dtype).square() / 3  # noqa: E731
    # (a ds below the type's normal numbers is rounded like any other: it enters its product times a power of two)
    step = lambda x: (torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(1e-300)))) * u).square() / 3  # noqa: E731
    delta = (u * u / 3) * ds.square().sum(-1, keepdim=True) + (g6 * rough).square().sum(-1, keepdim=True) / 3
    square = [scale ** 2 * (step(ds) @ k6.square() + delta * (p @ k6).square()) + third(dq),
              scale ** 2 * (step(ds) + delta * p.square()).transpose(2, 3) @ q6.square() + third(dk),
              step(p).transpose(2, 3) @ g6.square() + third(dv)]
    mean = [1.1 * x.mean().sqrt() + e.square().mean().sqrt() for x, e in zip(square, fine)]
    return [(w.reshape(x.shape), e.reshape(x.shape), a) for w, e, a, x in zip((dq, dk, dv), full, mean, (q, k, v))]


def check(q, k, v, g, scale, lens=None, mask=None):
    b, n = k.shape[0], k.shape[2]
    valid = torch.ones(b, n, dtype=torch.bool, device=q.device)
    if lens is not None:
        valid = valid & (torch.arange(n, device=q.device) < lens[:, None])
    if mask is not None:
        valid = valid & mask
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(attend(*leaves, scale, lens, mask), leaves, g)
    for name, x, (want, tol, mean) in zip(("dq", "dk", "dv"), got, definition(q, k, v, g, scale, valid)):
        # float16 ends at 65504, and what is 65520 or more rounds to infinity: it may be that where the exact result is so large
        beyond = want.abs() + tol >= (65520.0 if q.dtype == torch.float16 else float("inf"))
        off = torch.where(beyond & (x.isinf() & (x.sign() == want.sign())), 0.0, x.double() - want)
        assert float(off.square().mean().sqrt()) <= float(mean), "%s: %g off in the square mean, %g allowed" % (name, off.square().mean().sqrt(), mean)
        assert (off.abs() <= tol).all(), "%s: off by %g" % (name, (off.abs() - tol).max())
    return got


def draw(dev, b, h, hk, m, n, d, dtype, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    one = lambda heads, t: torch.randn((b, t, heads, d), generator=gen, device=dev).transpose(1, 2)  # noqa: E731
    return tuple(x.to(dtype) for x in (one(h, m), one(hk, n), one(hk, n), one(h, m)))


# few keys and many rows (one pass over the rows, 4 or 8 waves, heads up to 64 and longer ones), long keys, divided walks
SIZES = [(2, 4, 2, 130, 100, 64), (1, 4, 4, 300, 120, 128), (2, 32, 32, 1100, 200, 64), (1, 40, 40, 1700, 250, 80), (2, 4, 2, 200, 512, 64), (1, 4, 2, 150, 700, 128),
         (1, 4, 1, 9, 3000, 64), (1, 8, 2, 3, 2100, 96)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_peaked_rows(dev, dtype, size):
    """A few keys take most of a row, and the values have a mean: what is left of dS is small beside delta."""
    q, k, v, g = draw(dev, *size, dtype, seed=1)
    check(q, k, (v.float() + 3.0).to(dtype), g, 4 * size[5] ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_long_masks_that_leave_few_keys(dev, dtype, size):
    q, k, v, g = draw(dev, *size, dtype, seed=2)
    n = size[4]
    for left in ([n - 1], [40, n - 3], [0, 33, 70]):
        mask = torch.zeros(size[0], n, dtype=torch.bool, device=dev)
        mask[:, left] = True
        dq, dk, dv = check(q, k, v, g, size[5] ** -0.5, mask=mask)
        if len(left) == 1:  # a softmax over one key has no gradient: what is left is the fp32 sums of dP and delta, of D products of about 1
            assert float(dq.float().abs().max()) < 2.0 ** -14 and float(dk.float().abs().max()) < 2.0 ** -12


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_backward_with_and_without_the_rest(dev, dtype, size):
    """o with o_low has 8 bits more, and a backward that is not given o_low forms the same one."""
    q, k, v, g = draw(dev, *size, dtype, seed=3)
    lens = torch.full((size[0],), size[4] - 1, dtype=torch.int32, device=dev)
    o, lse, low = _C.cross_attention(q, k, v, 0.1, lens, rest=True)
    assert all(torch.equal(a, b) for a, b in zip((o, lse), _C.cross_attention(q, k, v, 0.1, lens))) and torch.equal(o, attend(q, k, v, 0.1, lens))
    assert low.is_contiguous() and low.dtype == torch.int8 and low.shape == o.shape and bool((low.float().std() > 60) & (low.float().mean().abs() < 10))
    fine = (o.float().contiguous().view(torch.int32) + low.int() * (256 if dtype == torch.bfloat16 else 32)).view(torch.float32).double()
    valid = torch.arange(size[4], device=dev) < size[4] - 1
    k6, v6 = (x.double().repeat_interleave(size[1] // size[2], 1)[:, :, valid] for x in (k, v))
    s = q.double() @ k6.transpose(2, 3) * 0.1
    p = torch.softmax(s, -1)
    # o's own roundings: P (sum_j r_j p_j (v_j - o), in the square mean) and what the 8 bits leave; a rounding of o would be u / sqrt(3) |o| or so
    u = torch.finfo(dtype).eps / 2
    spread = (p.square() @ v6.square() + p.square().sum(-1, keepdim=True) * (p @ v6).square()).sqrt()
    assert float(((fine - p @ v6) / (u * (spread + (p @ v6).abs() / 128) + 2.0 ** -20)).square().mean().sqrt()) < 1.0
    one = _C.cross_attention_backward(g, q, k, v, o, lse, 0.1, lens, o_low=low)
    two = _C.cross_attention_backward(g, q, k, v, o, lse, 0.1, lens)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    assert all(torch.equal(a, b) for a, b in zip(one, torch.autograd.grad(attend(*leaves, 0.1, lens), leaves, g)))
    with pytest.raises(RuntimeError, match="o_low"):
        _C.cross_attention_backward(g, q, k, v, o, lse, 0.1, lens, o_low=low[..., :8])


def test_small_probabilities_in_float16(dev):
    """Thousands of keys that share a row evenly: probabilities below float16's normal numbers enter the products of dV times a power of two."""
    q, k, v, g = draw(dev, 1, 2, 1, 70, 50000, 64, torch.float16, seed=4)
    check(q, k, v, g, 0.02)
    q, k, v, g = draw(dev, 2, 4, 2, 40, 33, 64, torch.float16, seed=5)
    check(q, k, v, g, 2.0)                                           # few keys, some of them with next to nothing


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [60, 250, 60001])
def test_many_keys_far_below_the_largest(dev, dtype, n):
    """One key of weight 1 and n - 1 of weight 2^-18.45 each: relative to the maximum they are below float16's normal numbers, and together
    (n = 60001) a sixth as much. Each weight is rounded by u at most, the same for all: o is off by u times the sum of the parts, and half a step."""
    gen = torch.Generator(device=dev).manual_seed(6)
    d = 64
    q = torch.ones(1, 1, 5, d, device=dev)
    k = torch.zeros(1, 1, n, d, device=dev)
    k[:, :, 0] = 18.45 * 0.6931471805599453 / 8
    v = torch.randn((1, 1, n, d), generator=gen, device=dev) + 1.0
    v[:, :, 0] = 0.0
    q, k, v = (x.to(dtype) for x in (q, k, v))
    u = torch.finfo(dtype).eps / 2
    p = torch.softmax(q.double() @ k.double().transpose(2, 3) * 0.125, -1)
    want = p @ v.double()
    off = (attend(q, k, v, 0.125).double() - want).abs()
    assert (off <= (u + 2.0 ** -17) * (p @ (v.double() - want[:, :, :1]).abs()) + 2.0 ** -17 * want.abs() + half_step(want, dtype)).all(), float(off.max())


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("step", [1e-1, 1e-2, 1e-3, 1e-4])
def test_small_gradients_in_float16(dev, size, step):
    """Gradients of a mean over many elements: ds far below float16's normal numbers, between results that are not (long queries or long
    keys make them so)."""
    q, k, v, g = draw(dev, *size, torch.float16, seed=7)
    g = (g.float() * step).half()
    for a, b in ((1 / 16, 16), (16, 1 / 16)):
        check((q.float() * a).half(), (k.float() * b).half(), v, g, size[5] ** -0.5)


@pytest.mark.parametrize("size", SIZES)
def test_rows_with_gradients_of_every_size_in_float16(dev, size):
    """Rows from 2^-14 to 1, some zero: small ones beside, before and behind large ones, each exact by itself in dQ."""
    q, k, v, g = draw(dev, *size, torch.float16, seed=8)
    m, power = size[3], torch.arange(size[3], device=dev)
    for e in (power * 37 % 15, power * 14 // m, 14 - power * 14 // m):
        scale = torch.exp2(-e.float()) * (power % 11 != 5)
        check((q.float() / 16).half(), (k.float() * 16).half(), v, (g.float() * scale[:, None]).half(), size[5] ** -0.5)


@pytest.mark.parametrize("size", SIZES)
def test_large_gradients_in_float16(dev, size):
    """Gradients times a loss scale: ds above float16's largest number, between results nearly all of which are below it."""
    q, k, v, g = draw(dev, *size, torch.float16, seed=9)
    q, k, v, g = (x.float().mul(f).half() for x, f in zip((q, k, v, g), (1 / 32, 1 / 32, 96.0, 512.0)))
    lens = torch.full((size[0],), 2, dtype=torch.int32, device=dev)
    check(q, k, v, g, size[5] ** -0.5, lens=lens)
    assert all(bool(torch.isfinite(x).all()) for x in check(q, k, v, g, size[5] ** -0.5))


def test_values_that_are_not_finite_stay_in_their_rows(dev):
    """float16 gradients with a NaN or an infinity: the rows (dQ) that have it, and the others as they are without it."""
    for size in SIZES:
        q, k, v, g = draw(dev, *size, torch.float16, seed=10)
        for bad, factor in ((float("nan"), 1.0), (float("inf"), 1.0), (float("nan"), 300.0), (float("inf"), 300.0)):
            g1 = (g.float() * factor).half()
            g2 = g1.clone()
            g2[:, :, -1, 3] = bad
            o, lse, low = _C.cross_attention(q, k, v, 0.1, rest=True)
            dq, dq2 = (_C.cross_attention_backward(x, q, k, v, o, lse, 0.1, o_low=low)[0] for x in (g1, g2))
            assert not torch.isfinite(dq2[:, :, -1].float()).any(-1).any() and torch.isfinite(dq2[:, :, :-1].float()).all(), (size, bad, factor)
            assert ((dq2[:, :, :-1].float() - dq[:, :, :-1].float()).abs() <= 2 * half_step(dq[:, :, :-1].float(), torch.float16)).all()


@pytest.mark.parametrize("size", SIZES)
def test_results_that_round_to_zero(dev, size):
    """Values at the end of float16's range: the result is zero or a few steps, of either sign, and what its rounding left off is not."""
    q, k, v, g = draw(dev, *size, torch.float16, seed=11)
    for tiny in (2.0 ** -24, 2.0 ** -20, 0.0):
        o = attend(q, k, (v.sign() * tiny).half(), 0.1)
        assert bool((o == 0).any())
        check(q, k, (v.sign() * tiny).half(), g, 0.1)
