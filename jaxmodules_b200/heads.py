"""What a model does with its query and key heads before attention: RMS norm of every head and rotary positions, in one pass.

The reference has no counterpart: its attention takes Q, K and V as they are.  Tensors are ``[B, L, H, d]`` as there, on a CUDA device.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _native as nat

_LAYOUTS = {"half": nat.BMA_ROTARY_HALF, "interleaved": nat.BMA_ROTARY_INTERLEAVED}


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0, original_length: Optional[int] = None,
                       low: float = 1.0, high: float = 32.0, device=None) -> torch.Tensor:
    """Radians per position of the ``dim / 2`` pairs of ``dim`` rotated components, float64: ``base ** (-2i / dim)``, scaled for contexts
    longer than those of training by

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: the base times ``factor ** (dim / (dim - 2))``, which divides the lowest frequency by ``factor`` and leaves the highest;
    * ``"parts"``: by the number of turns r that a pair makes within ``original_length`` positions: divided by ``factor`` where r <= ``low``, left where
      r >= ``high``, in between a mean of both that is linear in r.
    """
    if dim <= 0 or dim % 2:
        raise ValueError("dim must be positive and even")
    if not (base > 0 and factor > 0):
        raise ValueError("base and factor must be positive")
    i = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    if scaling == "base":
        if dim < 4:
            raise ValueError("scaling='base' needs dim of at least 4")
        base = base * factor ** (dim / (dim - 2))
    f = base ** -i
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if original_length is None or original_length <= 0 or not low < high:
            raise ValueError("scaling='parts' needs original_length, and low < high")
        keep = ((original_length / (2 * math.pi) * f - low) / (high - low)).clamp(0, 1)
        f = f * ((1 - keep) / factor + keep)
    elif scaling not in (None, "base"):
        raise ValueError("scaling must be None, 'linear', 'base' or 'parts'")
    return f.to(device="cuda" if device is None else device)


def layout_of(layout: str) -> int:
    if layout not in _LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved'")
    return _LAYOUTS[layout]


def rotate_heads(q: torch.Tensor, k: Optional[torch.Tensor], positions: Optional[torch.Tensor] = None, frequencies: Optional[torch.Tensor] = None, *,
                 layout: str = "half", magnitude: float = 1.0, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Queries and keys normed and rotated, ``(q, k)``, in one pass and with one rounding; differentiable in q, k and the weights.

    ``q``: ``[B, L, Hq, d]``, ``k``: ``[B, L, Hkv, d]`` or None; float32 or bfloat16, d at most 256, any strides (a tensor whose components do not lie side by
    side is copied).  The results are contiguous, of the same dtype.

    ``q_weight``, ``k_weight``: ``[d]``, float32 or bfloat16: every head x becomes ``x / sqrt(mean(x**2) + eps) * weight`` first.  None: that side has no norm.

    ``frequencies``: float64 ``[dim / 2]`` (``rotary_frequencies``): component pairs ``(i, i + dim / 2)`` (``layout="half"``) or ``(2i, 2i + 1)``
    (``"interleaved"``) of the first ``dim`` turn by the angle ``position * frequencies[i]`` and are multiplied by ``magnitude``; the other components stay.
    None: no rotation.  ``positions``: int32 or int64, ``[L]`` or ``[B, L]``, None for 0 .. L-1; the angles are as exact at position 2^30 as at 1.

    Repeated calls give the same bits, gradients included.  The gradients of the weights are sums over all tokens and heads in an order that
    the sizes of the call fix.  There are no second derivatives, none in forward mode and none in the frequencies: a backward pass with
    ``create_graph``, a dual tensor and ``frequencies`` that require a gradient are refused.  A forward and backward
    pass can be captured into a CUDA graph as long as no eager results that depend on the same leaves are held: torch's engine, for any operator, ends
    a capture that reaches a leaf which an eager graph holds.
    """
    return nat.host().rotate(q, k, positions, frequencies, layout_of(layout), magnitude, q_weight, k_weight, eps)
