"""Layer norm over the last dimension, differentiable in the input and in both parameters. The reference has an RMSNorm
only (q8_kernels/functional/rms_norm.py:8-24), whose backward leaves the weights frozen."""
from typing import Optional

import torch

from .. import _lib


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (1 to 32768 elements), in x's type.

    x: bfloat16, float16 or float32, any shape; rows may be strided (a slice of a wider tensor is read in place). weight,
    bias: [dim], both float32 or both of x's type, each optional. Statistics and sums are float32; the parameters' gradients
    are summed over the rows in a fixed order (the same bits for the same inputs). Gradients of gradients are not formed."""
    return _lib.ops().layer_norm(x, weight, bias, eps)
