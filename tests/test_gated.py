"""Gated feed-forward projections: forward and gradients against the 64-bit
definition, at sizes that end inside tiles, and what is refused."""

import pytest
import torch

from block_reference import U, check, gated64, gated_magnitudes, half_step

TYPES = [torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "gelu_tanh"]


def make(m, d, f, dtype, seed=0, bias=False):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s, std=1.0):
        return (torch.randn(*s, generator=g) * std).to(dtype)

    p = {"x": rnd(m, d), "w_gate": rnd(f, d, std=2 * d ** -0.5), "w_up": rnd(f, d, std=d ** -0.5)}
    if bias:
        p["b_gate"], p["b_up"] = rnd(f, std=0.5), rnd(f, std=0.5)
    p["dh"] = rnd(m, f, std=0.25)
    return p


def verify(p, act, h, grads):
    """h and the given gradients against the definition.

    dg and du are rounded to the operand type before the gradients' products:
    each is off by one half step of its value there, so the products' bounds
    add up half_step * |dg| and the f32 errors over the other operand."""
    dtype = p["x"].dtype
    names = [n for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if n in p]
    r = {n: p[n].double().requires_grad_(True) for n in names}
    h64, g64, u64 = gated64(r["x"], r["w_gate"], r["w_up"], r.get("b_gate"), r.get("b_up"), act)
    m = gated_magnitudes(p["x"], p["w_gate"], p["w_up"], p.get("b_gate"), p.get("b_up"), p["dh"],
                         (h64.detach(), g64.detach(), u64.detach()))
    check(h, h64, m["h"], 1 / U, "h")
    if not grads:
        return
    dg, du = torch.autograd.grad(h64, [g64, u64], p["dh"].double(), retain_graph=True)
    want = dict(zip(names, torch.autograd.grad(h64, [r[n] for n in names], p["dh"].double())))
    x, wg, wu = (p[n].double().abs() for n in ("x", "w_gate", "w_up"))
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    # bf16: a and b are kept as f16 times a power of two per 64 columns, off by
    # half a step of f16 or, far below the largest of the 64, 2^-39 of that
    kept = half_step(torch.float16) if dtype == torch.bfloat16 else 0.0
    dh = p["dh"].double().abs()
    low = 2.0 ** -38 if dtype == torch.bfloat16 else 0.0
    far_a, far_b = (dh * (t.abs() / dh.clamp(min=1e-30)).amax(1, keepdim=True) for t in (dg, du))
    eg = m["dg"] + (half_step(dtype) + kept) * (dg.abs() + m["dg"]) + low * far_a + tiny
    eu = m["du"] + (half_step(dtype) + kept) * (du.abs() + m["du"]) + low * far_b + tiny
    rows, f = dg.shape
    err = {"x": eg @ wg + eu @ wu + (2 * f + 2) * U * ((dg.abs() + eg) @ wg + (du.abs() + eu) @ wu),
           "w_gate": eg.t() @ x + (rows + 2) * U * ((dg.abs() + eg).t() @ x),
           "w_up": eu.t() @ x + (rows + 2) * U * ((du.abs() + eu).t() @ x),
           "b_gate": (eg + (rows + 2) * U * (dg.abs() + eg)).sum(0),
           "b_up": (eu + (rows + 2) * U * (du.abs() + eu)).sum(0)}
    for n, got in grads.items():
        check(got, want[n], err[n], 1 / U, n)
        assert got.dtype == dtype


def run(p, act="silu", names=None, recompute=False):
    from gen_worker_b200 import gated_linear

    names = names or [n for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if n in p]
    dev = {n: v.cuda() for n, v in p.items()}
    for n in names:
        dev[n].requires_grad_(True)
    h = gated_linear(dev["x"], dev["w_gate"], dev["w_up"], dev.get("b_gate"), dev.get("b_up"),
                     activation=act, recompute=recompute)
    return h, dict(zip(names, torch.autograd.grad(h, [dev[n] for n in names], dev["dh"])))


SIZES = [(1, 8, 8), (1, 64, 128), (2, 72, 136), (7, 200, 72), (8, 1024, 256), (16, 256, 1000),
         (17, 640, 512), (33, 136, 264), (64, 512, 384), (65, 320, 120), (127, 64, 64),
         (128, 128, 128), (129, 264, 392), (300, 1000, 520), (257, 512, 1032), (700, 256, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d,f", SIZES)
def test_sizes(cuda_ready, m, d, f, dtype):
    p = make(m, d, f, dtype, seed=m + d, bias=(m + f) % 3 == 0)
    verify(p, "silu", *run(p))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("recompute", [False, True])
def test_activations_and_biases(cuda_ready, recompute, m, act, dtype):
    p = make(m, 320, 264, dtype, bias=True)
    p["x"][0] *= 12                                # far into both tails
    p["x"][1] *= 2.0 ** -9                         # far below the kept planes' usual scale
    verify(p, act, *run(p, act, recompute=recompute))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d,f", [(40, 72, 4104), (1000, 256, 2600), (3000, 96, 136), (2100, 8, 264)])
def test_split_products(cuda_ready, m, d, f, dtype):
    """Gradients of few tiles and a long sum, which is split and joined: both
    weights', one weight's, and x's."""
    p = make(m, d, f, dtype, bias=m == 1000)
    verify(p, "silu", *run(p))
    for names in (["w_up"], ["w_gate"], ["x"]):
        verify(p, "silu", *run(p, names=names))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("f", [12288, 148 * 40, 13096])
@pytest.mark.parametrize("m", [33, 100, 128])
def test_few_rows_whose_tiles_end_inside_a_warp(cuda_ready, m, f, dtype):
    """Two chunks of rows or more for each half of the epilogue, and tiles of 88
    and 40 features, so a warp's lanes part at the stores of every chunk, or of
    96, the last of which ends inside a warp."""
    p = make(m, 72, f, dtype, bias=m == 100)
    from gen_worker_b200 import gated_linear

    h = gated_linear(*(p[n].cuda() for n in ("x", "w_gate", "w_up")),
                     *(p[n].cuda() for n in ("b_gate", "b_up") if n in p))
    verify(p, "silu", h, None)


@pytest.mark.gpu
def test_many_tiles(cuda_ready):
    """More tiles than multiprocessors, so the persistent walk wraps."""
    p = make(1100, 520, 2600, torch.bfloat16, bias=True)
    for recompute in (False, True):
        verify(p, "gelu_tanh", *run(p, "gelu_tanh", recompute=recompute))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("names", [["x"], ["w_gate"], ["w_up"], ["b_gate"], ["b_up"],
                                   ["w_up", "b_gate"], ["x", "w_gate", "w_up"]])
def test_each_gradient_alone(cuda_ready, names, m):
    p = make(m, 136, 200, torch.bfloat16, bias=True)
    h, grads = run(p, "gelu", names)
    verify(p, "gelu", h, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("one", ["b_gate", "b_up"])
def test_one_bias(cuda_ready, one):
    for m in (4, 140):
        p = make(m, 64, 72, torch.float16, bias=True)
        p.pop("b_up" if one == "b_gate" else "b_gate")
        verify(p, "silu", *run(p))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40, 150])
def test_strides_shapes_and_fused_weights(cuda_ready, m):
    """Slices of wider rows, rows that need a copy, leading dimensions, the
    halves of a fused weight, and an expanded gradient."""
    from gen_worker_b200 import gated_linear

    p = make(m, 128, 72, torch.bfloat16)
    w = torch.cat([p["w_gate"], p["w_up"]]).cuda()
    wg, wu = w[:72], w[72:]
    for lo, width in ((0, 128), (8, 160), (3, 131), (4, 140)):
        big = torch.zeros(m, width, dtype=torch.bfloat16)
        lo = min(lo, width - 128)
        big[:, lo:lo + 128] = p["x"]
        h = gated_linear(big.cuda()[:, lo:lo + 128], wg, wu)
        verify(p, "silu", h, None)
    h3 = gated_linear(p["x"].cuda().view(1, m, 1, 128), wg, wu)
    assert h3.shape == (1, m, 1, 72) and torch.equal(h3.view(m, 72), h)
    cols = p["x"].t().contiguous().t().cuda()      # column-major
    assert torch.equal(gated_linear(cols, wg, wu), h)
    x = p["x"].cuda().requires_grad_(True)
    grad, = torch.autograd.grad(gated_linear(x, wg, wu).sum(), x)
    q = dict(p, dh=torch.ones_like(p["dh"]))
    verify(q, "silu", h, {"x": grad})


@pytest.mark.gpu
@pytest.mark.parametrize("m", [6, 133])
def test_gradient_against_differences(cuda_ready, m):
    """<grad, v> against central differences of the 64-bit definition: the
    gradient's error is that of the operands' and its own rounding, at most
    1.5 steps of the type on every term; the difference's own error is under
    1e-6 of the same sum at h = 1e-4."""
    p = make(m, 64, 48, torch.float16, bias=True)
    _, grads = run(p, "gelu_tanh")
    h = 1e-4
    order = ("x", "w_gate", "w_up", "b_gate", "b_up")
    for n in order:
        v = torch.randn(p[n].shape, generator=torch.Generator().manual_seed(3)).double()

        def loss(sign):
            q = {k: t.double() for k, t in p.items()}
            q[n] = q[n] + sign * h * v
            return float((gated64(*(q[k] for k in order), "gelu_tanh")[0] * q["dh"]).sum())

        diff = (loss(1) - loss(-1)) / (2 * h)
        got = float((grads[n].double().cpu() * v).sum())
        a = {k: t.double().abs() for k, t in p.items()}
        _, g, u = gated64(*(p[k] for k in order), "gelu_tanh")
        dg, du = a["dh"] * u.abs() * 1.2, a["dh"] * g.abs()
        size = {"x": lambda: dg @ a["w_gate"] + du @ a["w_up"], "w_gate": lambda: dg.t() @ a["x"],
                "w_up": lambda: du.t() @ a["x"], "b_gate": lambda: dg.sum(0),
                "b_up": lambda: du.sum(0)}[n]()
        assert abs(got - diff) <= 1.5 * torch.finfo(torch.float16).eps * float((size * v.abs()).sum())


@pytest.mark.gpu
def test_non_finite_rows_stay_alone(cuda_ready):
    from gen_worker_b200 import gated_linear

    for m in (5, 140):
        p = make(m, 72, 88, torch.bfloat16)
        clean = gated_linear(*(p[n].cuda() for n in ("x", "w_gate", "w_up")))
        p["x"][1, 3] = float("nan")
        p["x"][3, 5] = float("inf")
        h = gated_linear(*(p[n].cuda() for n in ("x", "w_gate", "w_up")))
        others = [i for i in range(m) if i not in (1, 3)]
        assert torch.equal(h[others], clean[others])
        assert torch.isnan(h[1]).all() and not torch.isfinite(h[3]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [2, 150])
def test_negative_tail_is_relative(cuda_ready, m, act, dtype):
    """Gates in [-5.5, -3], where act(g) falls to 1e-7: h and the gradients keep
    their accuracy relative to act(g) and act'(g). Row 0 of x is a unit vector
    and the others are zero, so g and u are single exact products and the bias
    gradients are row 0's dg and du alone.

    f32 roundings (U) of act and act': the argument of exp or erfc is off by up
    to 4 U of at most 21, which the function turns into 84 U of its value; exp's
    own error is 2 + 1.16 * 21 ulp, 54 U, erfc's 8 U; products and the sum of
    two terms of which neither is over 8 times the result, 20 U: 160 U. Each
    output adds its rounding, and dg and du for bf16 that of a kept f16."""
    f = 64 * 5
    g = -torch.linspace(3.0, 5.5, f).to(dtype)
    up = 1024.0                                   # keeps f16's h out of its subnormals
    p = {"x": torch.zeros(m, 8, dtype=dtype), "w_gate": torch.zeros(f, 8, dtype=dtype),
         "w_up": torch.zeros(f, 8, dtype=dtype), "b_gate": torch.zeros(f, dtype=dtype),
         "b_up": torch.zeros(f, dtype=dtype), "dh": torch.zeros(m, f, dtype=dtype)}
    p["x"][0, 0], p["dh"][0] = 1.0, 1.0
    p["w_gate"][:, 0], p["w_up"][:, 0] = g, up
    g64 = g.double().requires_grad_(True)
    a64 = gated64(torch.ones(1, 1), g64[:, None], torch.ones(f, 1), None, None, act)[0][0]
    slope, = torch.autograd.grad(a64.sum(), g64)
    a64 = a64.detach()
    step, kept = half_step(dtype), half_step(torch.float16) if dtype == torch.bfloat16 else 0.0
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2

    def near(got, want, extra, what):
        off = (got.detach().double().cpu() - want).abs()
        bound = want.abs() * (160 * U + extra) * (1 + 2 * step) + step * want.abs() + tiny
        assert (off <= bound).all(), (what, float((off / want.abs()).max()), float(g[off.argmax()]))

    for recompute in (False, True):
        h, grads = run(p, act, recompute=recompute)
        near(h[0], a64 * up, 0.0, "h")
        assert not h[1:].any()
        near(grads["b_gate"], slope * up, 0.0 if recompute else kept, "dg")
        near(grads["b_up"][a64.abs() > 2 * torch.finfo(dtype).smallest_normal],
             a64[a64.abs() > 2 * torch.finfo(dtype).smallest_normal], 0.0 if recompute else kept, "du")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 150])
def test_erf_gelu_over_its_whole_range(cuda_ready, m):
    """Gates in [-12, 12]: act(g) = g times the normal distribution function,
    down to 1e-32 in bfloat16. The argument of exp, at most 72, is off by 2 U
    and exp itself by 2 + 1.16 * 72 ulp: 144 + 172 U; what exp multiplies and
    the products add under 30 U: 350 U of the value."""
    f = 1536
    g = torch.linspace(-12.0, 12.0, f).bfloat16()
    p = make(m, 8, f, torch.bfloat16)
    p = {"x": torch.zeros_like(p["x"]), "w_gate": torch.zeros_like(p["w_gate"]),
         "w_up": torch.zeros_like(p["w_up"])}
    p["x"][0, 0], p["w_gate"][:, 0], p["w_up"][:, 0] = 1.0, g, 1.0
    from gen_worker_b200 import gated_linear

    h = gated_linear(*(t.cuda() for t in p.values()), activation="gelu")[0].double().cpu()
    # erfc: torch's ndtr cancels in its own tail (0 at -12, where it is 1.8e-33)
    want = g.double() * 0.5 * torch.special.erfc(g.double() * -0.5 ** 0.5)
    assert ((h - want).abs() <= want.abs() * (half_step(torch.bfloat16) + 350 * U)).all()
    bad = torch.tensor([float("inf"), float("-inf"), float("nan"), 3e38, -3e38]).bfloat16()
    w = torch.zeros(8, 8, dtype=torch.bfloat16)
    w[:5, 0] = bad
    one = torch.zeros(1, 8, dtype=torch.bfloat16)
    one[0, 0] = 1.0
    up = torch.zeros(8, 8, dtype=torch.bfloat16)
    up[:, 0] = 1.0
    h = gated_linear(one.cuda(), w.cuda(), up.cuda(), activation="gelu")[0].float().cpu()
    assert torch.isinf(h[0]) and torch.isnan(h[1]) and torch.isnan(h[2])
    assert h[3] == bad[3].float() and h[4] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("recompute", [False, True])
def test_infinite_neighbour_of_finite_gradients(cuda_ready, recompute):
    """One infinite column of a group of 64: the other columns' gradients stay
    what they are, large and small (bf16 keeps 64 columns under one scale)."""
    f = 128
    p = {"x": torch.zeros(1, 8), "w_gate": torch.zeros(f, 8), "w_up": torch.zeros(f, 8),
         "b_gate": torch.zeros(f), "b_up": torch.zeros(f), "dh": torch.ones(1, f)}
    p["x"][0, 0] = 1.0
    p["w_gate"][:, 0] = 3.0
    p["w_up"][:, 0] = 2.0 ** 18
    p["w_up"][1::2, 0] = 2.0 ** -3
    p["w_up"][5, 0] = float("inf")
    p = {n: v.bfloat16() for n, v in p.items()}
    h, grads = run(p, recompute=recompute)
    s = torch.sigmoid(torch.tensor(3.0, dtype=torch.float64))
    dg = p["w_up"][:, 0].double() * s * (1 + 3 * (1 - s))
    # the largest finite value of the group is 2^18, so 2^-3 is 21 powers of two
    # below it and still a normal f16: half a step of f16, then of bf16
    for name, want in (("b_gate", dg), ("w_gate", dg), ("b_up", torch.full((f,), float(3 * s)).double())):
        got = grads[name].double().cpu()
        got = got[:, 0] if got.dim() == 2 else got
        others = [i for i in range(f) if i != 5]
        off = (got - want).abs()[others]
        assert (off <= want[others].abs() * (2 * 2.0 ** -8 + 2.0 ** -11 + 200 * U)).all(), name
    assert torch.isinf(grads["b_gate"][5]) and torch.isinf(h[0, 5])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("m", [2, 34, 300])
def test_bias_gradients_add_unrounded_terms(cuda_ready, m, recompute, dtype):
    """Bias gradients are f32 sums of f32 dg and du, rounded once: rows in pairs
    of opposite dh, so that a rounding of each term to the operand type would
    show beside sums that nearly cancel. Only what bf16 keeps (f16 values) is
    rounded before."""
    p = make(m, 64, 392, dtype, seed=m, bias=True)
    p["x"][1::2] = p["x"][0::2] + (torch.randn(m // 2, 64, generator=torch.Generator().manual_seed(1))
                                   * 0.02).to(dtype)
    p["dh"][1::2] = -p["dh"][0::2]
    h, grads = run(p, "silu", ["b_gate", "b_up"], recompute=recompute)
    r = {n: p[n].double().requires_grad_(True) for n in ("b_gate", "b_up")}
    h64, g64, u64 = gated64(p["x"], p["w_gate"], p["w_up"], r["b_gate"], r["b_up"], "silu")
    terms = dict(zip(r, torch.autograd.grad(h64, [g64, u64], p["dh"].double(), retain_graph=True)))
    want = dict(zip(r, torch.autograd.grad(h64, list(r.values()), p["dh"].double())))
    mag = gated_magnitudes(p["x"], p["w_gate"], p["w_up"], p["b_gate"], p["b_up"], p["dh"],
                           (h64.detach(), g64.detach(), u64.detach()))
    kept = half_step(torch.float16) if dtype == torch.bfloat16 and not recompute else 0.0
    for n, e in (("b_gate", mag["dg"]), ("b_up", mag["du"])):
        term = terms[n].abs() + e
        check(grads[n], want[n], (e + (kept + (m + 2) * U) * term).sum(0), 1 / U, n)


@pytest.mark.gpu
def test_f16_products_of_large_gradients_stay_in_their_rows(cuda_ready):
    """dg and du are float16 operands of the next products: a dg over 65504 is
    infinite there, in its own row of dx and its own row of dw_gate."""
    p = make(140, 64, 72, torch.float16)
    p["x"][7] *= 4
    h64, g64, _ = gated64(*(p[n].double().requires_grad_(n == "x") for n in ("x", "w_gate", "w_up")),
                          None, None, "silu")
    slope, = torch.autograd.grad(h64.sum(), g64)       # dg of a unit dh
    f = int(slope[7].abs().argmax())
    p["dh"][7, f] = 60000.0
    assert float(slope[7, f].abs()) * 60000 > 1e5
    h, grads = run(p)
    bad = torch.isfinite(grads["x"]).logical_not()
    assert bad[7].any() and not bad[torch.arange(140) != 7].any()
    bad = torch.isfinite(grads["w_gate"]).logical_not()
    assert bad[f].any() and not bad[torch.arange(72) != f].any()


@pytest.mark.gpu
def test_no_rows(cuda_ready):
    p = make(0, 64, 128, torch.bfloat16, bias=True)
    h, g = run(p)
    assert h.shape == (0, 128) and g["x"].shape == (0, 64)
    for n in ("w_gate", "w_up", "b_gate", "b_up"):
        assert g[n].shape == p[n].shape and not g[n].any()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [9, 260])
def test_same_bits_streams_and_graphs(cuda_ready, m):
    from gen_worker_b200 import gated_linear, native

    sets = [make(m, 256, 392, torch.bfloat16, seed=k, bias=True) for k in range(2)]
    want = [run(p, "silu") for p in sets]
    again = run(sets[0], "silu")
    assert torch.equal(again[0], want[0][0])
    assert all(torch.equal(again[1][n], want[0][1][n]) for n in again[1])
    names = ["x", "w_gate", "w_up", "b_gate", "b_up"]
    graphs = []
    for k in range(2):
        st = {n: torch.zeros_like(v, device="cuda") for n, v in sets[k].items()}
        for n in names:
            st[n].requires_grad_(True)

        def step():
            h = gated_linear(*(st[n] for n in names))
            return [h.detach(), *torch.autograd.grad(h, [st[n] for n in names], st["dh"])]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, st, out))
    for turn in range(2):
        for k, (g, st, out) in enumerate(graphs):
            with torch.no_grad():
                for n, v in sets[(k + turn) % 2].items():
                    st[n].copy_(v)
            g.replay()
        torch.cuda.synchronize()
        for k, (g, st, out) in enumerate(graphs):
            h, grads = want[(k + turn) % 2]
            assert torch.equal(out[0], h)
            assert all(torch.equal(o, grads[n]) for o, n in zip(out[1:], names))
    assert native.device_error() == 0


@pytest.mark.gpu
def test_modules(cuda_ready):
    import gen_worker_b200 as gw

    gate, up = (torch.nn.Linear(64, 136, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    down = torch.nn.Linear(136, 64, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(2, 9, 64, device="cuda", dtype=torch.bfloat16)
    ff = gw.gated_from_linears(gate, up, down=down, activation="gelu")
    h = gw.gated_linear(x, gate.weight, up.weight, gate.bias, up.bias, activation="gelu")
    assert torch.equal(ff(x), down(h))
    ff(x).sum().backward()
    assert gate.weight.grad is not None and up.bias.grad is not None
    fused = torch.nn.Linear(64, 272, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        fused.weight.copy_(torch.cat([up.weight, gate.weight]))
        fused.bias.copy_(torch.cat([up.bias, gate.bias]))
    both = gw.gated_from_fused(fused, gate_first=False, activation="gelu")
    assert torch.equal(both(x), h)
    assert both.w_gate.data_ptr() == fused.weight.data_ptr() + 136 * 64 * 2
    own = gw.GatedFeedForward(64, 136, bias=True, device="cuda")
    assert own(x).shape == (2, 9, 136)


@pytest.mark.gpu
def test_refusals(cuda_ready):
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    p = {n: v.cuda() for n, v in make(4, 64, 72, torch.bfloat16, bias=True).items()}
    x, wg, wu, bg = p["x"], p["w_gate"], p["w_up"], p["b_gate"]
    bad = [
        lambda: gw.gated_linear(x.float(), wg.float(), wu.float()),
        lambda: gw.gated_linear(x, wg.half(), wu), lambda: gw.gated_linear(x, wg, wu[:64]),
        lambda: gw.gated_linear(x[:, :60], wg[:, :60].contiguous(), wu[:, :60].contiguous()),
        lambda: gw.gated_linear(x, wg[:70].contiguous(), wu[:70].contiguous()),
        lambda: gw.gated_linear(x, wg.t().contiguous().t(), wu),
        lambda: gw.gated_linear(x, wg, wu, bg[:64]), lambda: gw.gated_linear(x, wg, wu, bg.float()),
        lambda: gw.gated_linear(x, wg.cpu(), wu), lambda: gw.gated_linear(x, wg, wu, activation="relu"),
        lambda: gw.gated_linear(x[:, :0], wg, wu),
        lambda: gw.gated_linear(x, torch.zeros(72 * 64 + 1, device="cuda",
                                               dtype=torch.bfloat16)[1:].view(72, 64), wu),
    ]
    for call in bad:
        with pytest.raises(SvdqB200Error):
            call()
    xr = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(gw.gated_linear(xr, wg, wu).sum(), xr, create_graph=True)


def test_refusals_on_the_cpu():
    import gen_worker_b200 as gw
    from gen_worker_b200 import native
    from gen_worker_b200.ops import SvdqB200Error

    z = torch.zeros(8, 8, dtype=torch.bfloat16)
    with pytest.raises(SvdqB200Error, match="no CPU path"):
        gw.gated_linear(z, z, z)
    for kw in ({"dim": 12, "hidden": 8}, {"dim": 8, "hidden": 0}, {"dim": 8, "hidden": 8, "activation": "x"},
               {"dim": 8, "hidden": 8, "dtype": torch.float32}):
        with pytest.raises(SvdqB200Error):
            gw.GatedFeedForward(**kw)
    with pytest.raises(SvdqB200Error):
        gw.gated_from_linears(torch.nn.Linear(8, 8), torch.nn.Linear(8, 16))
    with pytest.raises(SvdqB200Error):
        gw.gated_from_fused(torch.nn.Linear(8, 9))

    lib = native.lib()

    def call(m=4, d=8, f=8, act=0, dtype=1):
        return lib.gwb_gated_linear(None, d, None, None, None, None, m, d, f, act, dtype, None, None)

    assert call(m=0) == 0
    for kw in ({"d": 0}, {"f": 0}, {"d": 12}, {"f": 9}, {"m": -1}, {"act": 3}, {"act": -1}, {"dtype": 0},
               {}):
        assert call(**kw) == 1, kw
    assert lib.gwb_gated_linear_backward_work(0, 8, 8) == 0
    assert lib.gwb_gated_linear_backward_work(3, 8, 8) == 2 * 256 + 256
    assert lib.gwb_gated_linear_kept(3, 40, 1) == 3 * 40 * 4 + 3 * 8
    assert lib.gwb_gated_linear_kept(3, 40, 2) == 3 * 40 * 8 and lib.gwb_gated_linear_kept(3, 40, 0) == 0
