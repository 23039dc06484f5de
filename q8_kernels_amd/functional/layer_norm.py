"""Layer norm over the last dimension, differentiable in the input and in both parameters. The reference has an RMSNorm
only (q8_kernels/functional/rms_norm.py:8-24), whose backward leaves the weights frozen."""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .._C import layer_norm as layer_norm_forward, layer_norm_backward


class LayerNorm16bit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(grad_output, x, weight, bias, mean, rstd, ctx.needs_input_grad[:3])
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (1 to 32768 elements), in x's type.

    x: bfloat16, float16 or float32, any shape; rows may be strided (a slice of a wider tensor is read in place). weight,
    bias: [dim], both float32 or both of x's type, each optional. Statistics and sums are float32; their gradients are
    summed over the rows in a fixed order (the same bits for the same inputs)."""
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return LayerNorm16bit.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, stats=False)[0]
