"""Layer norm module with trainable parameters."""
import torch
import torch.nn as nn

from .. import functional as Q8F


class LayerNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, dtype=torch.float, device=device)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(dim, dtype=torch.float, device=device)) if elementwise_affine and bias else None

    def forward(self, x):
        return Q8F.layer_norm.layer_norm(x, self.weight, self.bias, self.eps)
