"""Measured cases of the transformer-block operators that run beside the quantised linears: layer
norm with modulation, rotary positions, and the gated feed-forward projections, forward and
backward.

``own`` False computes each operator in its plain form (elementary torch operations in 32 bits,
angles in 64, one rounding at the end); ``own`` True makes the calls a user makes of
``gen_worker_b200``. ``exact`` is the operator's definition in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6


def listed():
    return [
        # a short batch of conditioning tokens through an affine norm: latency counts
        {"name": "norm_tokens", "op": "norm", "dtype": "float16", "batch": 1, "tokens": 7,
         "dim": 1280, "affine": True, "modulated": False, "grad": False},
        # the norm before every projection of one dual-stream block: 4096 image + 512 text tokens,
        # hidden 3072, scale and shift chunks of the modulation layer's output
        {"name": "norm_block", "op": "norm", "dtype": "bfloat16", "batch": 1, "tokens": 4608,
         "dim": 3072, "affine": False, "modulated": True, "grad": False},
        # the same norm in a training step of four samples, with the modulation's gradients
        {"name": "norm_train", "op": "norm", "dtype": "bfloat16", "batch": 4, "tokens": 4608,
         "dim": 3072, "affine": False, "modulated": True, "grad": True},
        # an fp32 affine norm of a width that divides by nothing, with weight and bias gradients
        {"name": "norm_train_odd", "op": "norm", "dtype": "float32", "batch": 3, "tokens": 1037,
         "dim": 1153, "affine": True, "modulated": False, "grad": True},
        # one new token for each of 48 sequences, far into a context extended by parts
        {"name": "rotary_step", "op": "rotary", "dtype": "float16", "batch": 48, "tokens": 1,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary_dim": 128, "interleaved": False,
         "axes": "", "scaling": "by_parts", "reach": 131072, "grad": False},
        # queries and keys of one dual-stream block: 24 heads, positions on three axes
        {"name": "rotary_block", "op": "rotary", "dtype": "bfloat16", "batch": 1, "tokens": 4608,
         "heads": 24, "kv_heads": 24, "head_dim": 128, "rotary_dim": 128, "interleaved": True,
         "axes": "16,56,56", "scaling": "none", "reach": 128, "grad": False},
        # a training step of long odd sequences, part of the head rotated, few key heads
        {"name": "rotary_train", "op": "rotary", "dtype": "bfloat16", "batch": 2, "tokens": 8191,
         "heads": 32, "kv_heads": 4, "head_dim": 96, "rotary_dim": 64, "interleaved": False,
         "axes": "", "scaling": "linear", "reach": 16384, "grad": True},
        # one token: every weight is read for one row
        {"name": "gated_token", "op": "gated", "dtype": "bfloat16", "rows": 1, "dim": 3072,
         "hidden": 12288, "activation": "silu", "bias": False, "grad": False},
        # a small ragged batch of single tokens
        {"name": "gated_batch", "op": "gated", "dtype": "float16", "rows": 27, "dim": 2560,
         "hidden": 6912, "activation": "gelu_tanh", "bias": True, "grad": False},
        # the feed-forward of one dual-stream block
        {"name": "gated_block", "op": "gated", "dtype": "bfloat16", "rows": 4608, "dim": 3072,
         "hidden": 12288, "activation": "gelu_tanh", "bias": True, "grad": False},
        # its training step
        {"name": "gated_train", "op": "gated", "dtype": "bfloat16", "rows": 4608, "dim": 3072,
         "hidden": 12288, "activation": "silu", "bias": False, "grad": True},
        # a training step of sizes that end inside every tile
        {"name": "gated_train_ragged", "op": "gated", "dtype": "float16", "rows": 1531,
         "dim": 1416, "hidden": 3880, "activation": "gelu", "bias": True, "grad": True},
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of low..high."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "gated"])
    half = rng.choice(["bfloat16", "float16"])
    grad = rng.random() < 0.5
    if op == "norm":
        dim = _spread(rng, 40, 8192)
        if rng.random() < 0.5:
            dim = dim // 8 * 8
        batch = rng.randint(1, 4)
        modulated = rng.random() < 0.5
        return {"op": op, "dtype": rng.choice([half, half, "float32"]), "batch": batch,
                "tokens": _spread(rng, 1, max(1, 28_000_000 // (batch * dim))), "dim": dim,
                "affine": (not modulated) or rng.random() < 0.3, "modulated": modulated,
                "grad": grad}
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 192, 256])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 3, 4, 8])
        batch = _spread(rng, 1, 64)
        axes = ""
        if rng.random() < 0.3:
            first = rotary_dim // 4
            axes = "%d,%d" % (first, rotary_dim - first)
        most = 40_000_000 // (batch * (heads + kv_heads) * head_dim)
        return {"op": op, "dtype": rng.choice([half, half, "float32"]), "batch": batch,
                "tokens": _spread(rng, 1, max(1, min(16384, most))), "heads": heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "rotary_dim": rotary_dim,
                "interleaved": rng.random() < 0.5, "axes": axes,
                "scaling": rng.choice(["none", "linear", "by_parts"]),
                "reach": _spread(rng, 128, 1 << 20), "grad": grad}
    dim = _spread(rng, 32, 512) * 8
    hidden = _spread(rng, 32, 1536) * 8
    most = 4608 * 3072 * 12288 // (dim * hidden)
    return {"op": op, "dtype": half, "rows": _spread(rng, 1, max(1, min(8192, most))), "dim": dim,
            "hidden": hidden, "activation": rng.choice(["silu", "gelu", "gelu_tanh"]),
            "bias": rng.random() < 0.5, "grad": grad}


# ---------------------------------------------------------------- inputs
def _frequencies(case, device):
    """(inv_freq f64 [rotary_dim / 2], axis i32 or None, attention scale)."""
    parts = [int(v) for v in case["axes"].split(",")] if case["axes"] else [case["rotary_dim"]]
    freq, axis = [], []
    for a, width in enumerate(parts):
        n = width // 2
        freq.append(10000.0 ** (-torch.arange(n, dtype=torch.float64) * 2 / width))
        axis += [a] * n
    inv = torch.cat(freq)
    scale, factor, trained = 1.0, 8.0, 4096
    if case["scaling"] == "linear":
        inv = inv / factor
    elif case["scaling"] == "by_parts":
        turns = trained * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        inv = inv * keep + inv / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    where = torch.tensor(axis, dtype=torch.int32, device=device) if len(parts) > 1 else None
    return inv.to(device), where, scale, len(parts)


def prepare(case, seed):
    device = "cuda"
    dtype = getattr(torch, case["dtype"])
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device=device) * std + mean).to(dtype)

    state = {"case": case}
    if case["op"] == "norm":
        b, s, d = case["batch"], case["tokens"], case["dim"]
        x = torch.randn(b, s, d, generator=g, device=device)
        # hidden states carry a few channels far larger than the rest, and a mean
        outliers = torch.randint(0, d, (max(1, d // 100),), generator=g, device=device)
        x[:, :, outliers] *= 20.0
        state["x"] = (x + 0.25).to(dtype)
        if case["affine"]:
            state["weight"] = normal(d, std=0.2, mean=1.0)
            state["bias"] = normal(d, std=0.2)
        if case["modulated"]:
            # chunks of the modulation layer's [batch, 6 * dim] output
            mod = normal(b, 6, d, std=0.3)
            state["shift"], state["scale"] = mod[:, 0], mod[:, 1]
        if case["grad"]:
            state["dy"] = normal(b, s, d)
        leaves = ("x", "weight", "bias", "scale", "shift")
    elif case["op"] == "rotary":
        b, s = case["batch"], case["tokens"]
        inv, axis, scale, n_axes = _frequencies(case, device)
        # the fused projection's output: queries, keys and values side by side per token
        heads, kv = case["heads"], case["kv_heads"]
        fused = normal(b, s, heads + 2 * kv, case["head_dim"])
        state["q"], state["k"] = fused[:, :, :heads], fused[:, :, heads:heads + kv]
        if n_axes > 1:
            state["positions"] = torch.randint(0, case["reach"], (b, s, n_axes), generator=g,
                                               device=device)
        else:
            first = torch.randint(0, max(1, case["reach"] - s), (b, 1), generator=g, device=device)
            state["positions"] = first + torch.arange(s, device=device)
        state["inv_freq"], state["axis"], state["attention_scale"] = inv, axis, scale
        if case["grad"]:
            state["dq"] = normal(b, s, heads, case["head_dim"])
            state["dk"] = normal(b, s, kv, case["head_dim"])
        leaves = ("q", "k")
    else:
        m, d, f = case["rows"], case["dim"], case["hidden"]
        state["x"] = normal(m, d)
        state["w_gate"] = normal(f, d, std=d ** -0.5)
        state["w_up"] = normal(f, d, std=d ** -0.5)
        if case["bias"]:
            state["b_gate"], state["b_up"] = normal(f, std=0.1), normal(f, std=0.1)
        if case["grad"]:
            state["dh"] = normal(m, f, std=0.1)
        leaves = ("x", "w_gate", "w_up", "b_gate", "b_up")
    if case["grad"]:
        for name in leaves:
            if name in state:
                state[name].requires_grad_(True)
        state["leaves"] = [name for name in leaves if name in state]
    return state


# ---------------------------------------------------------------- plain forms
def _plain_norm(st):
    x = st["x"].float()
    d = x.shape[-1]
    centred = x - x.sum(-1, keepdim=True) / d
    rstd = (centred.square().sum(-1, keepdim=True) / d + EPS).rsqrt()
    xhat = centred * rstd
    weight, bias = st.get("weight"), st.get("bias")
    a = xhat if weight is None else xhat * weight.float() + bias.float()
    gain = 1.0 if st.get("scale") is None else 1.0 + st["scale"].float().unsqueeze(1)
    y = a if st.get("scale") is None else a * gain + st["shift"].float().unsqueeze(1)
    out = {"y": y.to(st["x"].dtype)}
    if not st["case"]["grad"]:
        return out
    dy = st["dy"].float()
    da = dy * gain
    dxhat = da if weight is None else da * weight.float()
    dx = rstd * (dxhat - dxhat.sum(-1, keepdim=True) / d
                 - xhat * ((dxhat * xhat).sum(-1, keepdim=True) / d))
    out["x"] = dx.to(st["x"].dtype)
    if weight is not None:
        out["weight"] = (da * xhat).sum((0, 1)).to(weight.dtype)
        out["bias"] = da.sum((0, 1)).to(bias.dtype)
    if st.get("scale") is not None:
        out["scale"] = (dy * a).sum(1).to(st["scale"].dtype)
        out["shift"] = dy.sum(1).to(st["shift"].dtype)
    return out


def _plain_turn(x, cos, sin, interleaved):
    """Pairs (a, b) of the rotated part of each head -> (a cos - b sin, b cos + a sin)."""
    v, n = x.float(), cos.shape[-1]
    if interleaved:
        a, b = v[..., 0:2 * n:2], v[..., 1:2 * n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = v[..., :n], v[..., n:2 * n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, v[..., 2 * n:]), -1).to(x.dtype)


def _plain_rotary(st):
    pos, axis = st["positions"].double(), st["axis"]
    pos = pos.unsqueeze(-1) if axis is None else pos[..., axis.long()]
    angle = (pos * st["inv_freq"]).unsqueeze(2)
    cos = (angle.cos() * st["attention_scale"]).float()
    sin = (angle.sin() * st["attention_scale"]).float()
    inter = st["case"]["interleaved"]
    out = {"q_out": _plain_turn(st["q"], cos, sin, inter),
           "k_out": _plain_turn(st["k"], cos, sin, inter)}
    if st["case"]["grad"]:
        out["q"] = _plain_turn(st["dq"], cos, -sin, inter)
        out["k"] = _plain_turn(st["dk"], cos, -sin, inter)
    return out


def _plain_activation(g, kind):
    """(act(g), act'(g))"""
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return (0.5 * g * (1.0 + t),
            0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g))


def _plain_gated(st):
    kind = st["x"].dtype
    x, wg, wu = st["x"].float(), st["w_gate"].float(), st["w_up"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if st["case"]["bias"]:
        g, u = g + st["b_gate"].float(), u + st["b_up"].float()
    act, slope = _plain_activation(g, st["case"]["activation"])
    out = {"h": (act * u).to(kind)}
    if not st["case"]["grad"]:
        return out
    dh = st["dh"].float()
    dg, du = dh * u * slope, dh * act
    out["x"] = (dg @ wg + du @ wu).to(kind)
    out["w_gate"], out["w_up"] = (dg.t() @ x).to(kind), (du.t() @ x).to(kind)
    if st["case"]["bias"]:
        out["b_gate"], out["b_up"] = dg.sum(0).to(kind), du.sum(0).to(kind)
    return out


# ---------------------------------------------------------------- the framework's calls
def _package():
    root = str(Path(__file__).resolve().parent.parent / "python-gen-worker_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gen_worker_b200
    return gen_worker_b200


def _own_run(st):
    lib, case = _package(), st["case"]
    if case["op"] == "norm":
        names, into = ["y"], [st.get("dy")]
        out = [lib.layer_norm(st["x"], st.get("weight"), st.get("bias"), scale=st.get("scale"),
                              shift=st.get("shift"), eps=EPS)]
    elif case["op"] == "rotary":
        names, into = ["q_out", "k_out"], [st.get("dq"), st.get("dk")]
        out = list(lib.rotary(st["q"], st["k"], st["positions"], st["inv_freq"], axis=st["axis"],
                              interleaved=case["interleaved"], scale=st["attention_scale"]))
    else:
        names, into = ["h"], [st.get("dh")]
        out = [lib.gated_linear(st["x"], st["w_gate"], st["w_up"], st.get("b_gate"),
                                st.get("b_up"), activation=case["activation"])]
    answer = {n: v.detach() for n, v in zip(names, out)}
    if case["grad"]:
        grads = torch.autograd.grad(out, [st[n] for n in st["leaves"]], into)
        answer.update(zip(st["leaves"], grads))
    return answer


_PLAIN = {"norm": _plain_norm, "rotary": _plain_rotary, "gated": _plain_gated}


def run(state):
    if own:
        return _own_run(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    passes = 2 if case["grad"] else 1
    if case["op"] == "norm":
        n = case["batch"] * case["tokens"] * case["dim"]
        params = 2 * case["dim"] * (int(case["affine"]) + case["batch"] * int(case["modulated"]))
        return {"bytes": size * (2 * n * passes + params * passes),
                "flops": n * (8 if not case["grad"] else 22)}
    if case["op"] == "rotary":
        tokens = case["batch"] * case["tokens"]
        n = tokens * (case["heads"] + case["kv_heads"])
        axes = len(case["axes"].split(",")) if case["axes"] else 1
        return {"bytes": size * 2 * n * case["head_dim"] * passes + 8 * tokens * axes
                + 4 * case["rotary_dim"], "flops": 3 * n * case["rotary_dim"] * passes}
    m, d, f = case["rows"], case["dim"], case["hidden"]
    params = 2 * d * f + (2 * f if case["bias"] else 0)
    return {"bytes": size * (m * (d + f) + params) * passes,
            "flops": 4 * m * d * f * (3 if case["grad"] else 1)}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_norm(st, grad):
    def wide(name):
        return None if st.get(name) is None else st[name].detach().double()

    x, w, b, scale, shift = (wide(n) for n in ("x", "weight", "bias", "scale", "shift"))
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS)
    z = (x - mean) / sd
    affine = z if w is None else torch.addcmul(b, z, w)
    y = affine
    if scale is not None:
        y = affine + affine * scale[:, None, :] + shift[:, None, :]
    out = {"y": y}
    if grad:
        dy = wide("dy")
        up = dy if scale is None else dy + dy * scale[:, None, :]
        inner = up if w is None else up * w
        out["x"] = (inner - inner.mean(-1, keepdim=True)
                    - z * (inner * z).mean(-1, keepdim=True)) / sd
        if w is not None:
            out["weight"] = torch.einsum("bsd,bsd->d", up, z)
            out["bias"] = up.sum(dim=(0, 1))
        if scale is not None:
            out["scale"] = torch.einsum("bsd,bsd->bd", dy, affine)
            out["shift"] = dy.sum(dim=1)
    return out


def _exact_rotary(st, case, grad):
    place, where = st["positions"].to(torch.float64), st["axis"]
    place = place[..., None] if where is None else place.index_select(-1, where.long())
    n = case["rotary_dim"] // 2
    turn = torch.polar(torch.full_like(place * st["inv_freq"], st["attention_scale"]),
                       place * st["inv_freq"])[:, :, None, :]

    def apply(t, by):
        v = t.detach().double()
        r, rest = v[..., :2 * n], v[..., 2 * n:]
        pairs = r.unflatten(-1, (n, 2)) if case["interleaved"] else \
            r.unflatten(-1, (2, n)).transpose(-1, -2)
        c = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        r = c.flatten(-2) if case["interleaved"] else c.transpose(-1, -2).flatten(-2)
        return torch.cat([r, rest], dim=-1)

    out = {"q_out": apply(st["q"], turn), "k_out": apply(st["k"], turn)}
    if grad:
        out["q"], out["k"] = apply(st["dq"], turn.conj()), apply(st["dk"], turn.conj())
    return out


def _exact_gated(st, case, grad):
    x, wg, wu = (st[n].detach().double() for n in ("x", "w_gate", "w_up"))
    g, u = torch.einsum("md,fd->mf", x, wg), torch.einsum("md,fd->mf", x, wu)
    if case["bias"]:
        g += st["b_gate"].detach().double()
        u += st["b_up"].detach().double()
    # act(g) = g P(g); act'(g) = P + g P'
    if case["activation"] == "silu":
        p = torch.special.expit(g)
        dp = p * torch.special.expit(-g)
    elif case["activation"] == "gelu":
        p = torch.special.ndtr(g)
        dp = torch.exp(-g ** 2 / 2) / math.sqrt(2 * math.pi)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        p = torch.special.expit(c * (g + 0.044715 * g ** 3))
        dp = p * (1 - p) * c * (1 + 3 * 0.044715 * g ** 2)
    out = {"h": g * p * u}
    if grad:
        dh = st["dh"].double()
        dg, du = dh * u * (p + g * dp), dh * (g * p)
        out["x"] = torch.einsum("mf,fd->md", dg, wg) + torch.einsum("mf,fd->md", du, wu)
        out["w_gate"] = torch.einsum("mf,md->fd", dg, x)
        out["w_up"] = torch.einsum("mf,md->fd", du, x)
        if case["bias"]:
            out["b_gate"], out["b_up"] = dg.sum(0), du.sum(0)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(state, case["grad"])
        if case["op"] == "rotary":
            return _exact_rotary(state, case, case["grad"])
        return _exact_gated(state, case, case["grad"])
