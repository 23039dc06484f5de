"""Forward-mode derivatives of the differentiable operators: refused, on the CPU before anything else is looked at, and on the GPU
with and without gradients of the other kind."""
import pytest
import torch
from torch.autograd import forward_ad

from q8_kernels_amd import functional as Q8F
from q8_kernels_amd.functional.rotary import apply_rotary, rotary_frequencies

norm, attend = Q8F.layer_norm.layer_norm, Q8F.cross_attention.cross_attention


def dual_calls(device):
    x = torch.randn(2, 2, 4, 64, device=device).to(torch.bfloat16)
    w, f = torch.ones(64, device=device), rotary_frequencies(64)[0].to(device)
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    return [lambda: norm(dual(x)), lambda: norm(x, dual(w)), lambda: norm(x, None, dual(w)),
            lambda: apply_rotary(dual(x), None, None, f), lambda: apply_rotary(x, dual(x), None, f), lambda: apply_rotary(x, None, None, dual(f)),
            lambda: attend(dual(x), x, x), lambda: attend(x, dual(x), x), lambda: attend(x, x, dual(x))]


def test_dual_tensors_are_refused_on_the_cpu():
    with forward_ad.dual_level():
        for call in dual_calls("cpu"):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_dual_tensors_are_refused(dev):
    with forward_ad.dual_level():
        for grads in (True, False):
            with torch.set_grad_enabled(grads):
                for call in dual_calls(dev):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call()
    x = torch.randn(2, 2, 4, 64, device=dev).to(torch.bfloat16)
    with forward_ad.dual_level():  # tensors without a tangent: as ever
        assert torch.equal(norm(x), norm(x.clone())) and attend(x, x, x).shape == x.shape
    with torch.inference_mode():
        assert torch.equal(norm(x.clone()), norm(x)) and torch.equal(attend(x.clone(), x, x), attend(x, x, x))
