"""Fake (meta) implementations of the block operators that
``libgwb200_torch.so`` defines, so ``torch.compile`` and shape inference can
trace through them. Imported once the library is loaded."""

from __future__ import annotations

import torch


@torch.library.register_fake("gwb200::layer_norm")
def _(x, weight, bias, scale, shift, eps):
    return x.new_empty(x.shape)


@torch.library.register_fake("gwb200::layer_norm_stats")
def _(x, weight, bias, scale, shift, eps):
    rows = x.numel() // x.shape[-1]
    return (x.new_empty(x.shape), x.new_empty(rows, dtype=torch.float32),
            x.new_empty(rows, dtype=torch.float32))


@torch.library.register_fake("gwb200::layer_norm_backward")
def _(dy, x, mean, rstd, weight, bias, scale, shift, mask):
    given = (x, weight, bias, scale, shift)
    return tuple(t.new_empty(t.shape) if on else x.new_empty(0) for t, on in zip(given, mask))


@torch.library.register_fake("gwb200::rotary")
def _(q, k, positions, inv_freq, axis, interleaved, scale, inverse):
    return q.new_empty(q.shape), q.new_empty(0) if k is None else k.new_empty(k.shape)


@torch.library.register_fake("gwb200::rotary_")
def _(q, k, positions, inv_freq, axis, interleaved, scale, inverse):
    return None


@torch.library.register_fake("gwb200::gated_linear")
def _(x, w_gate, w_up, b_gate, b_up, activation, recompute):
    return x.new_empty((*x.shape[:-1], w_gate.shape[0]))


@torch.library.register_fake("gwb200::gated_linear_keep")
def _(x, w_gate, w_up, b_gate, b_up, activation):
    f = w_gate.shape[0]
    rows = x.numel() // x.shape[-1]
    kept = rows * f * 4 + rows * ((f + 63) // 64) * 8 if x.dtype == torch.bfloat16 else rows * f * 8
    return x.new_empty((*x.shape[:-1], f)), x.new_empty(kept, dtype=torch.uint8)


@torch.library.register_fake("gwb200::gated_linear_backward")
def _(dh, x, w_gate, w_up, b_gate, b_up, kept, activation, mask):
    given = (x, w_gate, w_up, b_gate, b_up)
    return tuple(t.new_empty(t.shape) if on else x.new_empty(0) for t, on in zip(given, mask))
