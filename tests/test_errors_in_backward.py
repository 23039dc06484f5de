"""What a status of the library becomes in Python: Q8Error with the status, from a call and from a backward, whose nodes run on a thread
of torch's engine."""
import pytest
import torch

from q8_kernels_amd import _lib, functional as Q8F


def test_sizes_that_a_backward_does_not_take_are_refused_by_its_workspace_query():
    L = _lib.lib()
    for query in (L.q8_cross_attn_backward_workspace, L.q8_cross_attn_train_backward_workspace):
        assert query(1 << 17, 1, 1, 1, 16640, 8) == -3 and query(1 << 20, 16, 16, 8, 300, 64) == -3 and query(1 << 16, 1, 1, 1, 16640, 8) > 0


@pytest.mark.gpu
def test_status_of_a_backward(dev):
    """One token for each of 2^17 batch elements, and 16640 keys that they share by a stride of 0, none of which counts: the forward
    takes them, the backward would need more workgroups than a launch has, and says so before it allocates anything."""
    b, n = 1 << 17, 16640
    q = torch.zeros(b, 1, 1, 8, dtype=torch.bfloat16, device=dev, requires_grad=True)
    k = torch.zeros(1, 1, n, 8, dtype=torch.bfloat16, device=dev).expand(b, 1, n, 8)
    o = Q8F.cross_attention.cross_attention(q, k, k, None, torch.zeros(b, dtype=torch.int32, device=dev))
    with pytest.raises(_lib.Q8Error, match="out of range") as caught:
        o.float().sum().backward()
    assert caught.value.status == -3 and q.grad is None
    with pytest.raises(_lib.Q8Error) as caught:
        Q8F.cross_attention.cross_attention(q.detach(), k, k, 0.0)
    assert caught.value.status == -3
    assert torch.equal(Q8F.layer_norm.layer_norm(q.detach()[:2]), q.detach()[:2])  # and calls after it work
