"""16-bit attention to the states of an encoder (or any other keys and values), differentiable: the attention of fine-tuning
and of decoders next to the fp8 inference attention of functional.flash_attention, which has no gradient and heads of 64
(the reference trains through torch's attention, q8_kernels/modules/attention.py:96-101)."""
from typing import Optional

import torch

from .. import _lib


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: Optional[float] = None,
                    kv_lens: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(softmax_scale q k^T) v for q [B, H, M, D] and k, v [B, Hkv, N, D]: [B, H, M, D] in q's type and memory order.

    bfloat16 or float16; D a multiple of 8 up to 128; H a multiple of Hkv (query head h uses key head h // (H / Hkv)); any M
    and N, from one token on. Strides are read in place (`.view(B, N, Hkv, D).transpose(1, 2)` of a token-major projection)
    where the last is 1 and rows are 16-byte aligned, else the tensor is copied. softmax_scale: positive, D ** -0.5 if None.
    kv_lens: int32 [B], the keys of each batch element that count (clamped to 0 .. N); key_mask: bool [B, N], True where a key
    counts; both: keys that pass both. What stands in keys and values that do not count is not looked at, and their gradients
    are zeros. A query whose keys all do not count gets zeros. Scores, sums and the softmax are float32; the probabilities
    (and, in the backward, their gradients) are rounded to the inputs' type where they enter a product, in float16 times a power
    of two that keeps small and large ones in its range. Differentiable once; a call that is differentiated keeps a byte for
    each element of the result beside what it was given. Forward-mode tangents are refused."""
    return _lib.ops().cross_attention(q, k, v, softmax_scale, kv_lens, key_mask)
