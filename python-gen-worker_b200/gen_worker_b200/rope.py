"""Rotary positions of queries and keys, as they come out of a block's
(quantised) qkv projection.

Pairs of each head's first ``rotary_dim`` features turn by
``positions * inv_freq``: pair i is (2 i, 2 i + 1) in the interleaved layout,
(i, rotary_dim / 2 + i) in the half layout; the other features pass through.
Positions may have several axes (image rows and columns), each with its own
share of the pairs. Angles are reduced in 64 bits, so far positions keep
their accuracy; queries and keys share one launch.
"""

from __future__ import annotations

import math
from typing import Any, Optional, Sequence, Tuple

import torch
import torch.nn as nn

from . import native
from .ops import SvdqB200Error

SCALINGS = ("none", "linear", "ntk", "by_parts")


def _call(op: str, q, k, positions, inv_freq, axis, interleaved, scale):
    if not q.is_cuda:
        raise SvdqB200Error(f"q must be a CUDA tensor (no CPU path), got {q.device}")
    try:
        return getattr(native.block_ops(q), op)(q, k, positions, inv_freq, axis, interleaved,
                                                scale, False)
    except ValueError as exc:
        raise SvdqB200Error(f"{op}: {exc}") from None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
           inv_freq: torch.Tensor, *, axis: Optional[torch.Tensor] = None,
           interleaved: bool = False, scale: float = 1.0
           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [B, S, H, D], k [B, S, Hk, D] or None (or both without B), any
    strides with a dense last dimension (views of a fused projection are read
    as they lie) -> the rotated q and k, contiguous.

    ``positions`` int64, int32 or float32: [S] or [B, S]; with ``axis`` (int32
    [rotary_dim / 2], the position axis of each pair) [S, A] or [B, S, A].
    ``inv_freq`` float64 [rotary_dim / 2]. Rotated features are multiplied by
    ``scale``. Differentiable in q and k, to any order; positions and
    frequencies that need a gradient are refused."""
    qo, ko = _call("rotary", q, k, positions, inv_freq, axis, interleaved, scale)
    return qo, None if k is None else ko


def rotary_(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
            inv_freq: torch.Tensor, *, axis: Optional[torch.Tensor] = None,
            interleaved: bool = False, scale: float = 1.0) -> None:
    """:func:`rotary` in place, for serving: the features that pass through
    are not touched, and no gradient is kept (tensors that need one are
    refused)."""
    _call("rotary_", q, k, positions, inv_freq, axis, interleaved, scale)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, axes: Sequence[int] = (),
                       scaling: str = "none", factor: float = 1.0, trained_length: int = 0,
                       slow_turns: float = 1.0, fast_turns: float = 32.0
                       ) -> Tuple[torch.Tensor, Optional[torch.Tensor], float]:
    """(inv_freq float64 [rotary_dim / 2], axis int32 or None, attention scale).

    ``axes``: features of each position axis, summing to ``rotary_dim``; each
    axis has frequencies base ** (-2 i / features). ``scaling`` for contexts
    ``factor`` times the trained length:

    * ``linear``: every frequency divided by ``factor``;
    * ``ntk``: base multiplied by factor ** (d / (d - 2)), so the lowest
      frequency is divided by ``factor`` and the highest kept;
    * ``by_parts``: pairs that turn more than ``fast_turns`` times over
      ``trained_length`` are kept, pairs under ``slow_turns`` divided by
      ``factor``, a linear ramp between over the number of turns; attention
      scale 0.1 ln(factor) + 1. (Some code ramps over the pair's index between
      rounded bounds instead: frequencies of such a checkpoint are other ones.)
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise SvdqB200Error(f"rotary_dim {rotary_dim} is not a positive even number")
    if scaling not in SCALINGS:
        raise SvdqB200Error(f"scaling {scaling!r} is not one of {SCALINGS}")
    if not factor >= 1.0:
        raise SvdqB200Error(f"scaling factor {factor} is under 1")
    widths = list(axes) if axes else [rotary_dim]
    if sum(widths) != rotary_dim or any(w < 2 or w % 2 for w in widths):
        raise SvdqB200Error(f"axes {tuple(widths)} are not even and positive or do not sum to "
                            f"rotary_dim {rotary_dim}")
    parts, axis = [], []
    for a, width in enumerate(widths):
        b = base * factor ** (width / (width - 2)) if scaling == "ntk" and width > 2 else base
        i = torch.arange(width // 2, dtype=torch.float64)
        parts.append(torch.pow(torch.tensor(float(b), dtype=torch.float64), -2.0 * i / width))
        axis += [a] * (width // 2)
    inv = torch.cat(parts)
    scale = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "by_parts":
        if trained_length < 1 or not fast_turns > slow_turns:
            raise SvdqB200Error("by_parts scaling needs trained_length >= 1 and "
                                "fast_turns > slow_turns")
        turns = trained_length * inv / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        inv = inv * keep + inv / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    return inv, torch.tensor(axis, dtype=torch.int32) if len(widths) > 1 else None, scale


class RotaryEmbedding(nn.Module):
    """The frequencies of one model's rotary positions (buffers ``inv_freq``
    float64 and, with several axes, ``axis`` int32) and the calls that apply
    them: ``rope(q, k, positions)`` and ``rope.rotate_(q, k, positions)``."""

    def __init__(self, rotary_dim: int, *, interleaved: bool = False, base: float = 10000.0,
                 axes: Sequence[int] = (), scaling: str = "none", factor: float = 1.0,
                 trained_length: int = 0, slow_turns: float = 1.0, fast_turns: float = 32.0,
                 attention_scale: Optional[float] = None, device: Any = None) -> None:
        super().__init__()
        inv, axis, scale = rotary_frequencies(
            rotary_dim, base=base, axes=axes, scaling=scaling, factor=factor,
            trained_length=trained_length, slow_turns=slow_turns, fast_turns=fast_turns)
        self.rotary_dim = int(rotary_dim)
        self.interleaved = bool(interleaved)
        self.scaling = scaling
        self.attention_scale = float(scale if attention_scale is None else attention_scale)
        self.register_buffer("inv_freq", inv.to(device), persistent=False)
        if axis is None:
            self.axis = None
        else:
            self.register_buffer("axis", axis.to(device), persistent=False)

    def _apply(self, fn, recurse=True):
        # a cast of the module (.half(), .to(dtype)) moves the frequencies and
        # leaves their 64 bits
        inv = self.inv_freq
        super()._apply(fn, recurse)
        if self.inv_freq.dtype != torch.float64:
            self.inv_freq = inv.to(self.inv_freq.device)
        return self

    def forward(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        return rotary(q, k, positions, self.inv_freq, axis=self.axis,
                      interleaved=self.interleaved, scale=self.attention_scale)

    def rotate_(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor) -> None:
        rotary_(q, k, positions, self.inv_freq, axis=self.axis, interleaved=self.interleaved,
                scale=self.attention_scale)

    def extra_repr(self) -> str:
        return (f"rotary_dim={self.rotary_dim}, interleaved={self.interleaved}, "
                f"scaling={self.scaling}, axes={1 if self.axis is None else int(self.axis[-1]) + 1}")


__all__ = ["RotaryEmbedding", "SCALINGS", "rotary", "rotary_", "rotary_frequencies"]
