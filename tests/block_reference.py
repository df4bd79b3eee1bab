"""64-bit definitions of the block operators, and the error bounds of their
kernels, for the tests.

Bounds: an output of type t is one rounding, at most ``finfo(t).eps / 2`` of
its value (below the normal range, half the smallest subnormal), after f32
arithmetic whose error is a count of f32 roundings (u = 2^-24) times the
magnitudes that were added up. The counts are worst cases of the kernels'
summation order: at most 32 terms a thread in turn, five shuffle steps, five
across warps and the operator's own few operations, so 80 of the largest
partial magnitude covers a row sum and what is computed from it.
"""

import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, magnitude, count, what=""):
    """|got - want| <= one rounding to got's type + count f32 roundings of
    ``magnitude`` (elementwise, f64); NaN and infinities must agree."""
    g = got.detach().double().cpu()
    want, magnitude = want.detach().double().cpu(), torch.as_tensor(magnitude).double().cpu()
    assert g.shape == want.shape, f"{what}: shape {tuple(g.shape)} != {tuple(want.shape)}"
    assert torch.equal(torch.isnan(g), torch.isnan(want)), f"{what}: NaN places differ"
    fine = torch.isfinite(want)
    assert torch.equal(g[~fine].nan_to_num(), want[~fine].nan_to_num()), f"{what}: infinities"
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    slack = count * U * magnitude.expand_as(want)
    bound = half_step(got.dtype) * (want.abs() + slack) + slack + tiny / 2
    off = (g - want).abs()
    bad = fine & (off > bound)
    if bad.any():
        i = int((off / bound).nan_to_num().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got "
                             f"{g.flatten()[i]:.9g}, want {want.flatten()[i]:.9g}, bound "
                             f"{bound.flatten()[i]:.3g}")


# ---------------------------------------------------------------- layer norm
def norm64(x, w=None, b=None, s=None, t=None, eps=1e-6):
    """Layer norm in 64 bits; s / t already shaped to broadcast against x."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    z = (x - mean) / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    y = z if w is None else z * w.double()
    y = y if b is None else y + b.double()
    y = y if s is None else y * (1 + s.double())
    return y if t is None else y + t.double()


def norm_magnitudes(x, dy, w, b, s, t, eps):
    """Elementwise magnitudes of what each result is added up from."""
    x, dy = x.double(), dy.double()
    d = x.shape[-1]
    var = x.var(-1, correction=0, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    zmag = rstd * x.abs().amax(-1, keepdim=True) + rstd * (x - x.mean(-1, keepdim=True)).abs()
    w = torch.ones(d, dtype=torch.float64) if w is None else w.double().abs()
    b = torch.zeros(d, dtype=torch.float64) if b is None else b.double().abs()
    s1 = 1.0 if s is None else (1 + s.double().abs())
    t = 0.0 if t is None else t.double().abs()
    i = dy.abs() * w * s1
    rows = tuple(range(x.dim() - 1))
    out = {"y": (zmag * w + b) * s1 + t,
           "x": rstd * (i + i.mean(-1, keepdim=True) + zmag * (i * zmag).mean(-1, keepdim=True)),
           "weight": (dy.abs() * s1 * zmag).sum(rows), "bias": (dy.abs() * s1).sum(rows)}
    out["scale"] = dy.abs() * (zmag * w + b)
    out["shift"] = dy.abs()
    return out


# ---------------------------------------------------------------- rotary
def rotary64(x, positions, inv_freq, axis, interleaved, scale, sign=1.0):
    """x [B, S, H, D], positions [B or 1, S(, A)]."""
    pos = positions.double()
    pos = pos.unsqueeze(-1) if axis is None else pos[..., axis.long()]
    ang = (pos * inv_freq.double()).unsqueeze(2) * sign
    c, s = ang.cos() * scale, ang.sin() * scale
    v, n = x.double().clone(), inv_freq.numel()
    ia = torch.arange(n) * 2 if interleaved else torch.arange(n)
    ib = ia + 1 if interleaved else ia + n
    a, b = v[..., ia], v[..., ib]
    mag = v.abs()
    out, m = v.clone(), torch.zeros_like(mag)
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia] = m[..., ib] = (a.abs() + b.abs()) * abs(scale)
    return out, m


# Roundings in a rotated value, in units of (|a| + |b|) * scale: the angle
# (fraction of a turn to f32: pi), sincospi and the scale on each (3), two
# products and a sum (3).
ROTARY_COUNT = math.ceil(math.pi + 3 + 3)


# ---------------------------------------------------------------- gated projections
def gated64(x, wg, wu, bg, bu, activation):
    """(h, g, u) in 64 bits."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    g = g if bg is None else g + bg.double()
    u = u if bu is None else u + bu.double()
    if activation == "silu":
        a = g * torch.special.expit(g)
    elif activation == "gelu":
        a = g * torch.special.ndtr(g)
    else:
        a = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return a * u, g, u


def gated_magnitudes(x, wg, wu, bg, bu, dh, h64):
    """f64 bounds of the errors that come before each output's own rounding.

    A product's f32 accumulation over K terms is off by at most K * u times
    the terms' magnitudes (any order). In units of u: e = K + 2 for g and u;
    act and act' (slopes at most 1.13 and 1.7, act <= |g|) are off by 2 e
    |g|'s magnitude + 16 (|g| + 1) of their own arithmetic (exp to 2 ulp of an
    argument off by 3 roundings, at |t| <= 40 before it vanishes)."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    d = x.shape[1]
    zero = torch.zeros(wg.shape[0], dtype=torch.float64)
    bg, bu = (zero if b is None else b.double().abs() for b in (bg, bu))
    gm, um = x.abs() @ wg.abs().t() + bg, x.abs() @ wu.abs().t() + bu
    e = d + 2
    g, u = h64[1].abs(), h64[2].abs()
    act_err = (1.2 * e * gm + 48 * (g + 1)) * U
    slope_err = (1.0 * e * gm + 96 * (g + 1)) * U
    out = {"h": act_err * u + g * e * U * um + 4 * U * g * u}
    if dh is not None:
        dh = dh.double().abs()
        out["dg"] = dh * (1.2 * e * U * um + u * slope_err + 4 * U * 1.2 * u)
        out["du"] = dh * (act_err + 4 * U * g)
    return out
