"""16-bit attention to the states of an encoder (or any other keys and values), differentiable: the attention of fine-tuning
and of decoders next to the fp8 inference attention of functional.flash_attention, which has no gradient and heads of 64
(the reference trains through torch's attention, q8_kernels/modules/attention.py:96-101)."""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .._C import cross_attention as cross_attention_forward, cross_attention_backward


class CrossAttention16bit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, softmax_scale, kv_lens, key_mask):
        o, lse = cross_attention_forward(q, k, v, softmax_scale, kv_lens, key_mask)
        ctx.save_for_backward(q, k, v, o, lse, kv_lens, key_mask)
        ctx.softmax_scale = softmax_scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        q, k, v, o, lse, kv_lens, key_mask = ctx.saved_tensors
        dq, dk, dv = cross_attention_backward(grad_output, q, k, v, o, lse, ctx.softmax_scale, kv_lens, key_mask)
        return dq, dk, dv, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: Optional[float] = None,
                    kv_lens: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(softmax_scale q k^T) v for q [B, H, M, D] and k, v [B, Hkv, N, D]: [B, H, M, D] in q's type and memory order.

    bfloat16 or float16; D a multiple of 8 up to 128; H a multiple of Hkv (query head h uses key head h // (H / Hkv)); any M
    and N, from one token on. Strides are read in place (`.view(B, N, Hkv, D).transpose(1, 2)` of a token-major projection)
    where the last is 1 and rows are 16-byte aligned, else the tensor is copied. softmax_scale: positive, D ** -0.5 if None.
    kv_lens: int32 [B], the keys of each batch element that count (clamped to 0 .. N); key_mask: bool [B, N], True where a key
    counts; both: keys that pass both. What stands in keys and values that do not count is not looked at, and their gradients
    are zeros. A query whose keys all do not count gets zeros. Scores, sums and the softmax are float32; the probabilities
    (and, in the backward, their gradients) are rounded to the inputs' type where they enter a product."""
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return CrossAttention16bit.apply(q, k, v, softmax_scale, kv_lens, key_mask)
    return cross_attention_forward(q, k, v, softmax_scale, kv_lens, key_mask, stats=False)[0]
