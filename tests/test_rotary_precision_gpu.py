"""Rotary positions in float32 against the rotation in float64, all elements together: as exact as elementary operations in float32
with cosines and sines that were formed in float64 and rounded once. The kernel rounds the same values as often (each cosine and
sine, a product and the sum), so the square mean errors are alike; some 10^5 elements scatter by less than the 5 % allowed."""
import pytest
import torch

from q8_kernels_amd.functional.rotary import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("b,h,t,d,r,start", [(1, 16, 2000, 64, 64, 0), (2, 8, 1000, 128, 128, 100000), (1, 8, 500, 64, 32, 10 ** 9), (3, 16, 100, 96, 96, 4096)])
def test_float32_is_as_exact_as_rounded_tables(dev, layout, b, h, t, d, r, start):
    gen = torch.Generator(device=dev).manual_seed(t)
    x = torch.randn((b, h, t, d), generator=gen, device=dev).requires_grad_()
    g = torch.randn((b, h, t, d), generator=gen, device=dev)
    f = rotary_frequencies(r)[0].to(dev)
    pos = torch.arange(start, start + t, device=dev)
    y = apply_rotary(x, None, pos, f, layout=layout)
    (dx,) = torch.autograd.grad(y, x, g)
    angle = pos.double()[:, None] * f
    pairs = (lambda z: (z[..., :r // 2], z[..., r // 2:r])) if layout == "half" else (lambda z: (z[..., 0:r:2], z[..., 1:r:2]))

    def turned(z, sign, dtype):
        (u, v), c, s = (w.to(dtype) for w in pairs(z)), angle.cos().to(dtype), (sign * angle.sin()).to(dtype)
        return torch.stack((u * c - v * s, v * c + u * s)).double()

    for got, src, sign in ((y.detach(), x.detach(), 1), (dx, g, -1)):
        want = turned(src, sign, torch.float64)
        rms = lambda z: float((z - want).square().mean().sqrt())  # noqa: E731
        assert rms(torch.stack(pairs(got)).double()) <= 1.05 * rms(turned(src, sign, torch.float32))
        assert torch.equal(got[..., r:], src[..., r:])
