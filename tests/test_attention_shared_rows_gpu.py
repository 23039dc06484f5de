"""Which projections of modules.Attention share one quantization of their input: all that take the codes, adapters not."""
import pytest
import torch

from q8_kernels_amd.modules import Attention, Q8Linear, Q8LinearLora
from q8_kernels_amd.modules import attention as module

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Named(Q8Linear):
    """A layer of one's own, as Q8Linear but for what it is called."""


@pytest.mark.parametrize("kind", [Q8Linear, Named])
def test_layers_that_take_codes_share_them(dev, monkeypatch, kind):
    torch.manual_seed(0)
    attn = Attention(256, 4, 64).to(dev)
    for name in ("to_q", "to_k", "to_v", "to_out"):
        setattr(attn, name, kind.from_linear(torch.nn.Linear(256, 256, bias=False, device=dev, dtype=BF16)))
    x = torch.randn(2, 50, 256, device=dev, dtype=BF16)
    seen, quantize = [], module.Q8F.fused.hadamard_quantize
    monkeypatch.setattr(module.Q8F.fused, "hadamard_quantize", lambda t: seen.append(t) or quantize(t))
    with torch.no_grad():
        shared = attn(x, mm_out_dtype=BF16, attn_type="torch")
        assert len(seen) == 1 and seen[0] is x
        attn.fuse_prologue = False
        assert torch.equal(shared, attn(x, mm_out_dtype=BF16, attn_type="torch")) and len(seen) == 1


def test_an_adapter_among_them_gets_the_values(dev):
    torch.manual_seed(0)
    attn = Attention(256, 4, 64).to(dev)
    for name in ("to_q", "to_k", "to_v", "to_out"):
        setattr(attn, name, Q8Linear.from_linear(torch.nn.Linear(256, 256, bias=False, device=dev, dtype=BF16)))
    plain = attn.to_k
    attn.to_k = Q8LinearLora.from_linear(plain, r=4)
    x = torch.randn(2, 50, 256, device=dev, dtype=BF16)
    with torch.no_grad():
        a = attn(x, mm_out_dtype=BF16, attn_type="torch")
        attn.to_k = plain                                # (a fresh adapter adds zeros)
        b = attn(x, mm_out_dtype=BF16, attn_type="torch")
    assert torch.equal(a, b)
