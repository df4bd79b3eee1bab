"""Gated feed-forward projections: both projections, the activation and the
product in one kernel, with their gradients.

    h = act(x · w_gateᵀ + b_gate) * (x · w_upᵀ + b_up)

for the blocks whose feed-forward is gated and kept in bf16 / f16; the down
projection that follows may be any module, a quantised linear of this package
included (:class:`GatedFeedForward`).
"""

from __future__ import annotations

from typing import Any, Optional

import torch
import torch.nn as nn

from . import native
from .ops import SvdqB200Error

# activation name -> GWB_ACT_* code; "gelu" is the erf form
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                 b_gate: Optional[torch.Tensor] = None, b_up: Optional[torch.Tensor] = None, *,
                 activation: str = "silu", recompute: bool = False) -> torch.Tensor:
    """x [..., D], w_gate / w_up [F, D], biases [F] or None, all bfloat16 or
    all float16 -> h [..., F], contiguous. D and F are multiples of 8; weights
    and biases contiguous and 16-byte aligned (halves of a fused weight are).
    x may be a slice of wider rows; rows that 16-byte loads cannot step
    through are copied first. f32 accumulation; h is rounded once.

    Differentiable once in all of them. The gradients of g and u are rounded to
    x's type, as operands of the products that give the gradients of x and the
    weights (a float16 one over 65504 is infinite there: scale the loss); the
    bias gradients add them in f32. Where a gradient is wanted, 4 bytes per
    element of h (bfloat16: act(g) and u act'(g) as scaled float16; 8 for
    float16, as float32) are kept for the backward pass, or, with
    ``recompute``, nothing, and it computes the projections again."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise SvdqB200Error(f"activation {activation!r} is not one of {sorted(ACTIVATIONS)}")
    if not x.is_cuda:
        raise SvdqB200Error(f"x must be a CUDA tensor (no CPU path), got {x.device}")
    try:
        return native.block_ops(x).gated_linear(x, w_gate, w_up, b_gate, b_up, code,
                                                recompute)
    except ValueError as exc:
        raise SvdqB200Error(f"gated_linear: {exc}") from None


class GatedFeedForward(nn.Module):
    """``down(gated_linear(x))`` with parameters ``w_gate`` / ``w_up``
    [hidden, dim] and, with ``bias``, ``b_gate`` / ``b_up`` [hidden]; ``down``
    is any module from hidden features (None: h itself is returned);
    ``recompute`` as in :func:`gated_linear`."""

    def __init__(self, dim: int, hidden: int, *, activation: str = "silu", bias: bool = False,
                 down: Optional[nn.Module] = None, recompute: bool = False,
                 dtype: Any = torch.bfloat16, device: Any = None) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise SvdqB200Error(f"activation {activation!r} is not one of {sorted(ACTIVATIONS)}")
        if dim < 8 or hidden < 8 or dim % 8 or hidden % 8:
            raise SvdqB200Error(f"GatedFeedForward sizes {dim} -> {hidden}: positive multiples of "
                                f"8 are needed")
        if dtype not in (torch.bfloat16, torch.float16):
            raise SvdqB200Error(f"GatedFeedForward type {dtype} is not bfloat16 or float16")
        self.dim, self.hidden, self.activation = int(dim), int(hidden), activation

        def param(*shape):
            p = torch.empty(*shape, dtype=dtype, device=device)
            bound = self.dim ** -0.5
            return nn.Parameter(p.uniform_(-bound, bound))

        self.w_gate, self.w_up = param(hidden, dim), param(hidden, dim)
        self.b_gate = param(hidden) if bias else None
        self.b_up = param(hidden) if bias else None
        self.down = down
        self.recompute = bool(recompute)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = gated_linear(x, self.w_gate, self.w_up, self.b_gate, self.b_up,
                         activation=self.activation, recompute=self.recompute)
        return h if self.down is None else self.down(h)

    def extra_repr(self) -> str:
        return (f"dim={self.dim}, hidden={self.hidden}, activation={self.activation}, "
                f"bias={self.b_gate is not None or self.b_up is not None}")


def _assemble(w_gate, w_up, b_gate, b_up, activation, down) -> GatedFeedForward:
    hidden, dim = w_gate.shape
    mod = GatedFeedForward(dim, hidden, activation=activation, down=down, dtype=w_gate.dtype,
                           device="meta")
    mod.w_gate, mod.w_up, mod.b_gate, mod.b_up = w_gate, w_up, b_gate, b_up
    return mod


def gated_from_linears(gate: nn.Linear, up: nn.Linear, *, down: Optional[nn.Module] = None,
                       activation: str = "silu") -> GatedFeedForward:
    """From separate gate and up linears, sharing their parameters."""
    if gate.weight.shape != up.weight.shape:
        raise SvdqB200Error(f"gate {tuple(gate.weight.shape)} and up {tuple(up.weight.shape)} "
                            f"do not match")
    return _assemble(gate.weight, up.weight, gate.bias, up.bias, activation, down)


def gated_from_fused(proj: nn.Linear, *, gate_first: bool = True,
                     down: Optional[nn.Module] = None, activation: str = "silu"
                     ) -> GatedFeedForward:
    """From one linear that holds both projections stacked (the gate's rows
    first, or last), for serving: the halves are views of its weight and keep
    no gradient."""
    if proj.out_features % 2:
        raise SvdqB200Error(f"fused projection of {proj.out_features} rows has no two halves")

    def halves(t):
        if t is None:
            return None, None
        a, b = (nn.Parameter(h, requires_grad=False) for h in t.detach().chunk(2, 0))
        return (a, b) if gate_first else (b, a)

    (w_gate, w_up), (b_gate, b_up) = halves(proj.weight), halves(proj.bias)
    return _assemble(w_gate, w_up, b_gate, b_up, activation, down)


__all__ = ["ACTIVATIONS", "GatedFeedForward", "gated_from_fused", "gated_from_linears",
           "gated_linear"]
