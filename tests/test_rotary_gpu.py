"""Rotary positions against a float64 rotation. Tolerance: half a step of the result's type, and the fp32 part: the rest of
the angle in turns is rounded once (2^-25 turns, 2 pi 2^-25 = 1.9e-7 radians), sine and cosine are within 2 units (2^-23
each), the factor and the two products and the sum round once each: under 2^-21 (|u| + |v|) factor."""
import math

import pytest
import torch

from q8_kernels_amd import functional as Q8F
from q8_kernels_amd.functional.rotary import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def rotated(x, positions, inv_freq, layout, factor, sign=1):
    """(the rotation, its tolerance before the last rounding), float64"""
    b, h, t, d = x.shape
    n = inv_freq.shape[0]
    p = torch.arange(t, device=x.device) if positions is None else positions
    a = p.double().reshape(-1, 1, t, 1) * inv_freq
    c, s = a.cos() * factor, a.sin() * factor * sign
    y = x.double()
    u, v = (y[..., :n], y[..., n:2 * n]) if layout == "half" else (y[..., 0:2 * n:2], y[..., 1:2 * n:2])
    ru, rv, e = u * c - v * s, v * c + u * s, (u.abs() + v.abs()) * abs(factor) * 2.0 ** -21
    join = (lambda p, q: torch.cat((p, q), -1)) if layout == "half" else (lambda p, q: torch.stack((p, q), -1).flatten(-2))
    return torch.cat((join(ru, rv), y[..., 2 * n:]), -1), torch.cat((join(e, e), torch.zeros_like(y[..., 2 * n:])), -1)


def close(got, want, what):
    want, e = want
    eps = torch.finfo(got.dtype).eps / 2
    off, lim = (got.double() - want).abs(), (want.abs() + e) * eps + e + TINY[got.dtype]
    assert (off <= lim).all(), "%s: off by %g" % (what, off.max())


def heads(dev, b, h, t, d, dtype, seed, token_major=True):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((b, t, h, d) if token_major else (b, h, t, d), generator=gen, device=dev).to(dtype)
    return x.transpose(1, 2) if token_major else x


def check(q, k, positions, inv_freq, layout, factor):
    gq, gk = torch.randn_like(q), None if k is None else torch.randn_like(k)
    ql, kl = q.detach().requires_grad_(), None if k is None else k.detach().requires_grad_()
    out = apply_rotary(ql, kl, positions, inv_freq, layout=layout, factor=factor)
    plain = apply_rotary(q, k, positions, inv_freq, layout=layout, factor=factor)
    if k is None:
        out, plain, leaves, gs = (out,), (plain,), (ql,), (gq,)
    else:
        leaves, gs = (ql, kl), (gq, gk)
    grads = torch.autograd.grad(out, leaves, gs)
    for o, p, x, g, dx, name in zip(out, plain, leaves, gs, grads, "qk"):
        assert torch.equal(o, p) and o.shape == x.shape and o.dtype == x.dtype
        close(o.detach(), rotated(x.detach(), positions, inv_freq, layout, factor), name)
        close(dx, rotated(g, positions, inv_freq, layout, factor, -1), "d" + name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", [(64, 64), (128, 128), (128, 64), (96, 96), (80, 40), (2, 2), (6, 4), (33, 10), (512, 512), (511, 510), (72, 16), (40, 24)])
def test_head_sizes(dev, dtype, layout, d, r):
    f = rotary_frequencies(r)[0].to(dev)
    check(heads(dev, 2, 3, 5, d, dtype, 1), heads(dev, 2, 1, 5, d, dtype, 2), None, f, layout, 1.0)


@pytest.mark.parametrize("b,h,hk,t", [(1, 1, 1, 1), (16, 32, 8, 1), (3, 7, 2, 33), (2, 32, 32, 300), (1, 300, 1, 3), (2, 4, 4, 2500)])
def test_batches_heads_and_lengths(dev, b, h, hk, t):
    f = rotary_frequencies(64)[0].to(dev)
    pos = torch.randint(0, 100000, (b, t), device=dev, generator=torch.Generator(device=dev).manual_seed(t))
    check(heads(dev, b, h, t, 64, torch.bfloat16, 3), heads(dev, b, hk, t, 64, torch.bfloat16, 4, token_major=False), pos, f, "half", 1.25)


def test_position_forms(dev):
    f = rotary_frequencies(32)[0].to(dev)
    q, k = heads(dev, 3, 2, 6, 32, torch.float32, 5), heads(dev, 3, 2, 6, 32, torch.float32, 6)
    row = torch.tensor([5, 0, 2 ** 31 - 1, 7, 1 << 20, 3], device=dev)
    base = apply_rotary(q, k, row, f)
    wide = torch.stack([row, -row, row, row], -1)  # a column of a wider tensor: strided
    for pos in (row.int(), row[None], row[None].expand(3, 6), row.repeat(3, 1), row.repeat(3, 1).int(), wide[:, 0], torch.stack([row] * 3, 1).t(),
                torch.cat((row.repeat(3, 1), row.repeat(3, 1)), 1)[:, :6]):
        assert all(torch.equal(a, b) for a, b in zip(base, apply_rotary(q, k, pos, f)))
    sliding = torch.arange(8, device=dev).as_strided((3, 6), (1, 1))
    check(q, k, sliding, f, "half", 1.0)
    check(q, k, -row, f, "interleaved", 1.0)


def test_far_positions_keep_their_angle(dev):
    f = torch.tensor([1.0, 0.3, 1e-3, 1e-5], dtype=torch.float64, device=dev)
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 10 ** 9 + 7, 2 ** 40 + 3], device=dev)
    # (the angle itself carries the rounding of the fp64 product: 2^40 * 2^-52, far below the tolerance)
    check(heads(dev, 1, 2, 5, 8, torch.float32, 7), None, pos, f, "half", 1.0)


def test_strides_addresses_and_broadcast(dev):
    f = rotary_frequencies(64)[0].to(dev)
    for dtype in TYPES:
        buf = heads(dev, 1, 1, 1, 2 * 9 * 3 * 5 * 70, dtype, 8).flatten()
        qkv = buf[:2 * 5 * 9 * 70].view(2, 5, 9, 70)
        for lo in (0, 1, 3):                                             # q and k as slices of one projection, off 16 bytes
            q, k = qkv[:, :, :6, lo:lo + 64].transpose(1, 2), qkv[:, :, 6:8, lo:lo + 64].transpose(1, 2)
            check(q, k, None, f, "half", 1.0)
            check(q, k, None, f, "interleaved", 1.0)
        check(qkv[:1, :, :1, :64].expand(2, 5, 4, 64).transpose(1, 2), None, None, f, "half", 1.0)
        check(qkv[..., :64].transpose(1, 2).transpose(2, 3).contiguous().transpose(2, 3), None, None, f, "half", 1.0)  # no unit last stride


def test_output_has_the_input_order(dev):
    q = heads(dev, 2, 4, 6, 64, torch.bfloat16, 9)
    out = apply_rotary(q, None, None, rotary_frequencies(64)[0].to(dev))
    assert out.stride() == q.stride() and out.transpose(1, 2).is_contiguous()


def test_gradient_of_one_output(dev):
    f = rotary_frequencies(64)[0].to(dev)
    q, k = (heads(dev, 1, 2, 9, 64, torch.float32, s).requires_grad_() for s in (10, 11))
    a, b = apply_rotary(q, k, None, f)
    g = torch.randn_like(a)
    (dq,) = torch.autograd.grad(a, q, g, retain_graph=True)
    close(dq, rotated(g, None, f, "half", 1.0, -1), "dq alone")
    (dk,) = torch.autograd.grad(b, k, g)
    close(dk, rotated(g, None, f, "half", 1.0, -1), "dk alone")
    frozen = k.detach()
    a, b = apply_rotary(q, frozen, None, f)
    (dq2,) = torch.autograd.grad((a, b), q, (g, g))
    assert torch.equal(dq, dq2)


def test_gradient_against_differences(dev):
    """The rotation is linear: <g, R(x + d)> - <g, R(x - d)> = 2 <R^T g, d> but for the rounding of its values."""
    f = rotary_frequencies(48, scaling="by_parts", stretch=4.0)[0].to(dev)
    x, d, g = (heads(dev, 2, 3, 21, 64, torch.float32, s) for s in (12, 13, 14))
    xl = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(apply_rotary(xl, None, None, f, factor=1.1), xl, g)
    r = lambda y: (apply_rotary(y, None, None, f, factor=1.1).double() * g.double()).sum()  # noqa: E731
    want = 2 * (dx.double() * d.double()).sum()
    lim = 2.0 ** -20 * 2 * 1.1 * float(((x.abs() + d.abs()) * 2 * g.abs()).double().sum())
    assert abs(float(r(x + d) - r(x - d) - want)) <= lim


def test_nothing_to_do(dev):
    f = rotary_frequencies(64)[0].to(dev)
    for shape in ((0, 4, 3, 64), (2, 4, 0, 64), (2, 0, 3, 64)):
        q = torch.zeros(shape, device=dev, dtype=torch.bfloat16).requires_grad_()
        out = apply_rotary(q, None, None, f)
        assert out.shape == shape and torch.autograd.grad(out, q, torch.zeros_like(out))[0].shape == shape


def test_captured_and_replayed(dev):
    f = rotary_frequencies(128)[0].to(dev)
    q, k = heads(dev, 4, 8, 1, 128, torch.bfloat16, 15), heads(dev, 4, 2, 1, 128, torch.bfloat16, 16)
    pos = torch.zeros(4, 1, dtype=torch.int64, device=dev)
    apply_rotary(q, k, pos, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = apply_rotary(q, k, pos, f)
    for turn in range(3):
        pos += 1000 * turn + 7
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, apply_rotary(q, k, pos, f)))


def test_same_as_the_table_rotation(dev):
    """functional.rope with tables of the same angles, interleaved: one rounding more in the tables."""
    f = rotary_frequencies(64)[0].to(dev)
    x = heads(dev, 1, 1, 40, 64, torch.bfloat16, 17, token_major=False)
    a = torch.arange(40, device=dev).double()[:, None] * f
    c, s = (t.repeat_interleave(2, -1).float().expand(1, 1, 40, 64).contiguous() for t in (a.cos(), a.sin()))
    one, two = apply_rotary(x, None, None, f, layout="interleaved"), Q8F.rope.apply_rope(x, c, s)
    mag = x.double().abs().reshape(1, 1, 40, 32, 2).sum(-1).repeat_interleave(2, -1)
    assert ((one.double() - two.double()).abs() <= 2 * (2.0 ** -8 * one.double().abs() + 2.0 ** -20 * mag)).all()


def test_refusals(dev):
    f = rotary_frequencies(64)[0].to(dev)
    q = heads(dev, 2, 4, 6, 64, torch.bfloat16, 18)
    pos = torch.arange(6, device=dev)
    for bad in (lambda: apply_rotary(q, q.float(), None, f), lambda: apply_rotary(q[0], None, None, f), lambda: apply_rotary(q, None, pos.float(), f),
                lambda: apply_rotary(q, None, pos[:5], f), lambda: apply_rotary(q, None, pos.cpu(), f), lambda: apply_rotary(q, None, pos, f.float()),
                lambda: apply_rotary(q, None, pos, f.cpu()), lambda: apply_rotary(q[..., :62], None, pos, f), lambda: apply_rotary(q, q[:1], pos, f),
                lambda: apply_rotary(q, q[:, :, :5], pos, f), lambda: apply_rotary(q.to(torch.float8_e4m3fn), None, pos, f),
                lambda: apply_rotary(q, None, pos, f[:0]), lambda: apply_rotary(q.cpu(), None, None, f),
                lambda: apply_rotary(torch.zeros(1, 1, 1, 520, device=dev), None, None, f), lambda: apply_rotary(q, None, pos.repeat(3, 1), f)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        apply_rotary(q, None, None, f, layout="other")


def test_scaled_frequencies_on_the_device(dev):
    f, factor = rotary_frequencies(64, scaling="by_parts", stretch=8.0, device=dev)
    assert f.device.type == "cuda" and math.isclose(factor, 0.1 * math.log(8.0) + 1.0)
    check(heads(dev, 1, 4, 50, 64, torch.float16, 19), None, torch.arange(30000, 30050, device=dev), f, "half", factor)
