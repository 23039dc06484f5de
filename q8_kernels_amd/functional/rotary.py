"""Rotary positions given by the positions and the frequencies, for queries and keys of attention heads.

functional.rope rotates whole rows by tables of their shape (q8_kernels/functional/rope.py:9-44), as the video models do;
here a head, or the first part of it, turns by position * frequency, in the half or the interleaved layout, with the
frequencies of a longer context where wanted. The kernel forms the angles itself (float64), so there is no table, and no
largest position."""
import math
from typing import Optional, Tuple

import torch

from .. import _lib

LAYOUTS = ("half", "interleaved")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, stretch: float = 1.0,
                       trained_positions: int = 4096, low_turns: float = 1.0, high_turns: float = 32.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq float64 [rotary_dim / 2], factor) for apply_rotary: pair i turns by base^(-2 i / rotary_dim) radians per
    position. scaling stretches the context to `stretch` times `trained_positions`:

      None        nothing is scaled
      'linear'    positions are interpolated: every frequency divided by stretch
      'ntk'       the base grows to base * stretch^(d / (d - 2)): the slowest pair is interpolated, the fastest unchanged
      'by_parts'  pairs that turn more than high_turns times within trained_positions stay, those below low_turns are
                  interpolated, those between are blended linearly in their turns; the rotated values are multiplied by
                  factor = 0.1 ln(stretch) + 1 (YaRN, Peng et al. 2023, equations 17-22)"""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim must be even and positive, got %r" % (rotary_dim,))
    if not stretch >= 1.0 or not base > 0.0:
        raise ValueError("rotary_frequencies: stretch must be 1 or more and base positive")
    n = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("rotary_frequencies: 'ntk' needs two pairs or more")
        base = base * stretch ** (rotary_dim / (rotary_dim - 2))
    # on the CPU: a handful of values, in the same arithmetic everywhere
    f = base ** (-torch.arange(n, dtype=torch.float64) / n)
    factor = 1.0
    if scaling == "linear":
        f = f / stretch
    elif scaling == "by_parts":
        if not high_turns > low_turns:
            raise ValueError("rotary_frequencies: high_turns must be above low_turns")
        keep = ((trained_positions * f / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        f = torch.where(keep < 1.0, f / stretch + keep * (f - f / stretch), f)
        factor = 0.1 * math.log(stretch) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError("rotary_frequencies: scaling %r" % (scaling,))
    return (f if device is None else f.to(device)), factor


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: Optional[torch.Tensor], inv_freq: torch.Tensor, *,
                 layout: str = "half", factor: float = 1.0):
    """q [B, H, T, D] and k [B, Hkv, T, D] (or None), rotated: (q', k'), or q' alone without k. Differentiable in both (once).

    Any strides with unit last stride are read in place (token-major projections as `.view(B, T, H, D).transpose(1, 2)`);
    the results have the memory order of their inputs. bfloat16, float16 or float32, D up to 512. positions: int32 or
    int64 [T] or [B, T] (None: 0 .. T - 1). inv_freq: float64 [R / 2], radians per position; elements from R on are copied.
    layout 'half': pairs (i, i + R / 2); 'interleaved': pairs (2 i, 2 i + 1). factor multiplies the rotated elements.
    Angles, sines and products are formed in float64 / float32 and rounded once."""
    if layout not in LAYOUTS:
        raise ValueError("apply_rotary: layout %r (one of %s)" % (layout, ", ".join(LAYOUTS)))
    out = _lib.ops().apply_rotary(q, k, positions, inv_freq, layout == "half", factor)
    return out[0] if k is None else out
