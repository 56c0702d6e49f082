"""Rotary positions on q and k, half and interleaved layouts."""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import ext

_SCALINGS = (None, "linear", "ntk", "parts")


class Rotary:
    """The frequencies of rotary positions: what ``rotary()`` keeps per model.

    ``dim`` elements of a head rotate (even; the first ones), as dim / 2 pairs:
    element i with i + dim / 2 (the half layout), or 2i with 2i + 1
    (``interleaved``).  Pair i turns by ``base ** (-2i / dim)`` radians per
    position.  ``scaling`` stretches the positions for contexts ``factor``
    times as long:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: ``base`` multiplied by ``factor ** (dim / (dim - 2))``, so the
      fastest pair keeps its frequency and the slowest is divided by ``factor``;
    * ``"parts"``: a pair that turns at least ``fast`` times over ``original``
      positions keeps its frequency, one that turns at most ``slow`` times has
      it divided by ``factor``, linearly between; and cos and sin carry
      ``amplitude``, 0.1 ln(factor) + 1 unless given.

    ``turns`` holds the frequencies as full turns per position in 64 bits on
    ``device``; no table over positions is kept, so there is no largest
    position.
    """

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, scaling: Optional[str] = None,
                 factor: float = 1.0, original: int = 0, fast: float = 32.0, slow: float = 1.0,
                 amplitude: Optional[float] = None, device: Union[str, torch.device] = "cuda"):
        if dim < 2 or dim % 2:
            raise ValueError(f"Rotary: dim must be even and at least 2, got {dim}")
        if not base > 0 or not factor > 0:
            raise ValueError("Rotary: base and factor must be positive")
        if scaling not in _SCALINGS:
            raise ValueError(f"Rotary: unknown scaling {scaling!r}")
        if scaling == "ntk":
            if dim < 4:
                raise ValueError("Rotary: ntk scaling needs dim of at least 4")
            base = base * factor ** (dim / (dim - 2))
        f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
        if scaling == "linear":
            f = [x / factor for x in f]
        if scaling == "parts":
            if original < 1 or not fast > slow:
                raise ValueError("Rotary: scaling by parts needs original >= 1 and fast > slow")
            keep = [min(1.0, max(0.0, (original * x / (2 * math.pi) - slow) / (fast - slow))) for x in f]
            f = [x * w + x / factor * (1.0 - w) for x, w in zip(f, keep)]
            if amplitude is None:
                amplitude = 0.1 * math.log(factor) + 1.0
        self.dim = dim
        self.interleaved = bool(interleaved)
        self.amplitude = 1.0 if amplitude is None else float(amplitude)
        with torch.inference_mode(False):  # a plan outlives the call that made it, and training keeps it for the backward pass
            self.turns = torch.tensor([x / (2 * math.pi) for x in f], dtype=torch.float64, device=device)

    def to(self, device: Union[str, torch.device]) -> "Rotary":
        """The same plan on another device."""
        other = object.__new__(Rotary)
        other.__dict__.update(self.__dict__)
        with torch.inference_mode(False):
            other.turns = self.turns.to(device)
        return other


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], plan: Rotary,
           positions: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q [B, T, H, D] and k [B, T, Hk, D] turned to their positions, as new
    contiguous tensors (k None: q alone).  ``positions`` is [T] or [B, T], int32
    or int64 (0 .. T-1 if not given).  Elements from ``plan.dim`` on pass
    unchanged.  Gradients flow to q and k (the inverse turn).  One launch; any
    strides; float32, bfloat16 or float16, computed in 32 bits with the angle
    in 64 (sine and cosine of it to 1.5 units of 2^-24)."""
    out = ext.get_ops().rotary(q, k, plan.turns, positions, plan.dim, plan.interleaved, plan.amplitude)
    return out[0] if k is None else (out[0], out[1])


def rotary_(q: torch.Tensor, k: Optional[torch.Tensor], plan: Rotary,
            positions: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``rotary()`` in place (only the rotated part is touched); not on tensors
    that require a gradient, share memory with each other, or repeat elements
    (ValueError)."""
    ext.get_ops().rotary_inplace(q, k, plan.turns, positions, plan.dim, plan.interleaved, plan.amplitude)
    return q if k is None else (q, k)
