"""Layer norm with an optional affine and an optional modulation, the operator
a transformer block runs before its quantised projections.

    y = ((x - mean) * rstd * weight + bias) * (1 + scale) + shift

``scale`` and ``shift`` are rows per sample: the chunks of a modulation
layer's output (``awq.AwqPackedLinear`` serves those), read as they lie. One
kernel forward; backward, one pass over x and dy for dx and the column sums
and a small one that joins them, in a fixed order (two runs give the same
bits). Statistics and sums are f32 whatever the type.
"""

from __future__ import annotations

from typing import Any, Optional

import torch
import torch.nn as nn

from . import native
from .ops import SvdqB200Error


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, scale: Optional[torch.Tensor] = None,
               shift: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """x [..., D] (float32, bfloat16 or float16) -> y of x's shape and type,
    contiguous. ``weight`` / ``bias`` [D]; ``scale`` / ``shift`` [D], [B, D] or
    [B, 1, ..., 1, D] with B = 1 or x's first size. Each may be absent; each
    pair is float32 or of x's type. Differentiable once in all of them, in
    reverse mode (``create_graph=True`` is refused).

    Rows of x may lie at any one stride (a slice of a wider tensor); an x
    whose rows do not is copied first. Work is enqueued on the current stream
    of x's device."""
    if not x.is_cuda:
        raise SvdqB200Error(f"x must be a CUDA tensor (no CPU path), got {x.device}")
    try:
        return native.block_ops(x).layer_norm(x, weight, bias, scale, shift, eps)
    except ValueError as exc:
        raise SvdqB200Error(f"layer_norm: {exc}") from None


class ModulatedLayerNorm(nn.Module):
    """Drop-in for ``nn.LayerNorm`` over the last dimension (parameters
    ``weight`` and ``bias``) that also takes a modulation: ``norm(x, scale,
    shift)``."""

    def __init__(self, dim: int, *, eps: float = 1e-6, affine: bool = True, bias: bool = True,
                 dtype: Any = torch.bfloat16, device: Any = None) -> None:
        super().__init__()
        if dim < 1:
            raise SvdqB200Error(f"ModulatedLayerNorm dim {dim} is not positive")
        self.dim = int(dim)
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(dim, dtype=dtype, device=device)) if affine else None
        self.bias = (nn.Parameter(torch.zeros(dim, dtype=dtype, device=device))
                     if affine and bias else None)

    def forward(self, x: torch.Tensor, scale: Optional[torch.Tensor] = None,
                shift: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.shape[-1] != self.dim:
            raise SvdqB200Error(f"x has {x.shape[-1]} features, the norm {self.dim}")
        return layer_norm(x, self.weight, self.bias, scale=scale, shift=shift, eps=self.eps)

    def extra_repr(self) -> str:
        return (f"dim={self.dim}, eps={self.eps}, affine={self.weight is not None}, "
                f"bias={self.bias is not None}")


def norm_from_layer_norm(mod: nn.LayerNorm) -> ModulatedLayerNorm:
    """A :class:`ModulatedLayerNorm` that shares ``mod``'s parameters."""
    if len(mod.normalized_shape) != 1:
        raise SvdqB200Error(f"layer norm over {len(mod.normalized_shape)} dimensions: the kernel "
                            f"normalises the last one")
    out = ModulatedLayerNorm(mod.normalized_shape[0], eps=mod.eps, affine=False)
    out.weight = mod.weight
    out.bias = mod.bias
    return out


__all__ = ["ModulatedLayerNorm", "layer_norm", "norm_from_layer_norm"]
