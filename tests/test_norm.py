"""Layer norm with affine and modulation: forward and gradients against the
64-bit definition, and what the entry point refuses."""

import pytest
import torch

from block_reference import check, norm64, norm_magnitudes

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ROW, COLUMN = 80, 200   # f32 roundings of a row result, of a column sum (see block_reference)


def make(shape, dtype, seed=0, affine=False, mod=None, param=None):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s, std=1.0, mean=0.0, d=dtype):
        return (torch.randn(*s, generator=g) * std + mean).to(d)

    d = shape[-1]
    p = {"x": rnd(*shape, mean=0.5)}
    p["x"][..., :: max(1, d // 3)] *= 8
    if affine:
        p["weight"], p["bias"] = rnd(d, std=0.3, mean=1.0, d=param or dtype), rnd(d, d=param or dtype)
    if mod is not None:
        p["scale"], p["shift"] = (rnd(*mod, std=0.4, d=param or dtype) for _ in range(2))
    p["dy"] = rnd(*shape)
    return p


def wide(p, name, x):
    """scale / shift shaped to broadcast against x."""
    v = p.get(name)
    if v is None or v.dim() == 1:
        return v
    return v.reshape(v.shape[0], *([1] * (x.dim() - 2)), x.shape[-1])


def run_and_check(p, eps=1e-6, device="cuda", names=None):
    from gen_worker_b200 import layer_norm

    names = names or [n for n in ("x", "weight", "bias", "scale", "shift") if n in p]
    dev = {n: v.to(device) for n, v in p.items()}
    for n in names:
        dev[n] = dev[n].detach().requires_grad_(True)
    y = layer_norm(dev["x"], dev.get("weight"), dev.get("bias"), scale=dev.get("scale"),
                   shift=dev.get("shift"), eps=eps)
    grads = dict(zip(names, torch.autograd.grad(y, [dev[n] for n in names], dev["dy"])))
    ref = {n: p[n].double().requires_grad_(True) for n in names}
    full = {n: ref.get(n, p.get(n)) for n in ("x", "weight", "bias", "scale", "shift")}
    want = norm64(full["x"], full["weight"], full["bias"], wide(full, "scale", p["x"]),
                  wide(full, "shift", p["x"]), eps)
    wg = dict(zip(names, torch.autograd.grad(want, [ref[n] for n in names], p["dy"].double())))
    mag = norm_magnitudes(p["x"], p["dy"], p.get("weight"), p.get("bias"),
                          wide(p, "scale", p["x"]), wide(p, "shift", p["x"]), eps)
    check(y, want, mag["y"], ROW, "y")
    for n in names:
        m = mag[n]
        if n in ("scale", "shift"):
            m = m.sum_to_size(*wide(p, n, p["x"]).shape).reshape(p[n].shape)
        check(grads[n], wg[n], m, ROW if n == "x" else COLUMN, n)
        assert grads[n].dtype == p[n].dtype
    return y, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 3), (5, 64), (1, 256), (7, 257), (33, 512),
                                   (9, 1000), (130, 1280), (17, 1153), (6, 2304), (5, 4095),
                                   (4, 8192), (3, 8200), (2, 9001), (2, 40000)])
def test_affine_shapes(cuda_ready, dtype, shape):
    run_and_check(make(shape, dtype, seed=shape[1], affine=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,mod", [((3, 37, 640), (3, 640)), ((3, 37, 640), (640,)),
                                       ((2, 5, 7, 129), (2, 129)), ((1, 700, 2304), (1, 2304)),
                                       ((4, 1, 96), (4, 96)), ((300, 64), (300, 64)),
                                       ((2, 3, 9001), (2, 9001))])
@pytest.mark.parametrize("affine", [False, True])
def test_modulated(cuda_ready, dtype, shape, mod, affine):
    run_and_check(make(shape, dtype, seed=5, affine=affine, mod=mod))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_f32_parameters(cuda_ready, dtype):
    run_and_check(make((3, 50, 1024), dtype, affine=True, mod=(3, 1024), param=torch.float32))
    run_and_check(make((3, 50, 333), dtype, affine=True, mod=(3, 333), param=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("names", [["x"], ["weight"], ["bias"], ["shift"], ["scale"],
                                   ["x", "scale"], ["weight", "shift"]])
def test_each_gradient_alone(cuda_ready, names):
    run_and_check(make((2, 41, 384), torch.bfloat16, affine=True, mod=(2, 384)), names=names)


@pytest.mark.gpu
@pytest.mark.parametrize("only", ["weight", "bias", "scale", "shift"])
def test_each_parameter_alone(cuda_ready, only):
    p = make((2, 41, 384), torch.bfloat16, affine=True, mod=(2, 384))
    run_and_check({n: p[n] for n in ("x", "dy", only)})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_row_strides_and_chunks(cuda_ready, dtype):
    """Rows of a wider tensor, odd offsets, the chunks of a modulation."""
    from gen_worker_b200 import layer_norm

    g = torch.Generator().manual_seed(1)
    big = torch.randn(4, 33, 3 * 264 + 1, generator=g).to(dtype)
    mod = (torch.randn(4, 6 * 264, generator=g) * 0.3).to(dtype)
    dev, dmod = big.cuda(), mod.cuda()
    for lo in (0, 264, 265):
        x, dx = big[..., lo:lo + 264], dev[..., lo:lo + 264]
        s, t = mod.chunk(6, -1)[1], mod.chunk(6, -1)[0]
        ds, dt = dmod.chunk(6, -1)[1], dmod.chunk(6, -1)[0]
        y = layer_norm(dx, scale=ds, shift=dt)
        m = norm_magnitudes(x, x, None, None, s.unsqueeze(1), t.unsqueeze(1), 1e-6)
        check(y, norm64(x, s=s.unsqueeze(1), t=t.unsqueeze(1)), m["y"], ROW, f"slice {lo}")
    # rows at no single stride, and a last dimension that is not dense
    x = dev.transpose(0, 1)[..., :264]
    check(layer_norm(x), norm64(x.cpu()), norm_magnitudes(x.cpu(), x.cpu(), *[None] * 4, 1e-6)["y"],
          ROW, "transposed")
    x = dev[0, :, :33].t()
    check(layer_norm(x), norm64(x.cpu()), norm_magnitudes(x.cpu(), x.cpu(), *[None] * 4, 1e-6)["y"],
          ROW, "column-major")


@pytest.mark.gpu
@pytest.mark.parametrize("d", [96, 101, 700, 1153])
def test_rows_on_top_of_each_other(cuda_ready, d):
    """One row seen as many (stride 0), as x and as the gradient."""
    from gen_worker_b200 import layer_norm

    row = torch.randn(d, generator=torch.Generator().manual_seed(d)).to(torch.bfloat16)
    x = row.cuda().expand(37, d).detach().requires_grad_(True)
    y = layer_norm(x)
    g, = torch.autograd.grad(y, x, row.cuda().expand(37, d))
    xc, dy = row.expand(37, d), row.expand(37, d)
    r = xc.double().requires_grad_(True)
    want = norm64(r)
    wg, = torch.autograd.grad(want, r, dy.double())
    m = norm_magnitudes(xc, dy, None, None, None, None, 1e-6)
    check(y, want, m["y"], ROW, "y")
    check(g, wg, m["x"], ROW, "x")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_constant_rows_far_means_and_bad_values(cuda_ready, dtype):
    from gen_worker_b200 import layer_norm

    x = torch.randn(6, 320, generator=torch.Generator().manual_seed(2)).to(dtype)
    x[0] = 3.0                       # no variance: z = 0
    x[1] = 0.0
    x[2] += 200.0                    # a mean far from the spread
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    y = layer_norm(x.cuda())
    ok = [0, 1, 2, 5]
    m = norm_magnitudes(x[ok], x[ok], *[None] * 4, 1e-6)["y"]
    check(y[ok], norm64(x[ok]), m, ROW, "finite rows")
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()


# widths whose rounded reciprocal times the row sum misses the mean of a row of 200
INEXACT = [56, 61, 112, 190, 240, 504, 760, 1000, 1427, 1520, 1784, 2040, 2741, 3040, 3584, 3119,
           5480, 5507, 5792, 10952]


@pytest.mark.gpu
@pytest.mark.parametrize("d", INEXACT)
def test_rows_of_one_value_are_their_own_mean(cuda_ready, d):
    """The sum of d values of 200 is exact in f32 (200 d < 2^24), so its quotient
    by d is 200 and z is zero: few rows and many, aligned and not."""
    from gen_worker_b200 import layer_norm

    for dtype in TYPES:
        for rows in (3, 8400 if d < 4000 else 9):
            y = layer_norm(torch.full((rows, d), 200.0, device="cuda", dtype=dtype))
            assert not y.any(), (dtype, rows)
        wide = torch.full((5, d + 1), 200.0, device="cuda", dtype=dtype)
        assert not layer_norm(wide[:, 1:]).any(), (dtype, "unaligned")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [96, 320, 1280, 1153])
def test_gradients_of_rows_far_from_zero(cuda_ready, d, dtype):
    p = make((70, d), dtype, seed=d, affine=True)
    p["x"] = (p["x"].float() + 200.0 * torch.linspace(-1, 1, 70)[:, None]).to(dtype)
    run_and_check(p)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 40, 264])
def test_column_sums_over_many_samples(cuda_ready, d):
    """A modulation row for each of 40000 rows: weight and bias gradients add
    40000 samples. dy = 1 + 2^-10 loses its last bit in every step of one long
    f32 sum; chains of at most 64 terms, joined in turn, keep it. The bound is
    the column sums' usual count, 200 roundings of the magnitudes."""
    rows = 40000
    g = torch.Generator().manual_seed(d)
    p = {"x": torch.randn(rows, d, generator=g), "weight": torch.ones(d), "bias": torch.zeros(d),
         "scale": torch.zeros(rows, d), "shift": torch.zeros(rows, d),
         "dy": torch.full((rows, d), 1 + 2.0 ** -10)}
    run_and_check(p)
    p["scale"] = torch.randn(rows, d, generator=g) * 0.3
    p["dy"] = torch.randn(rows, d, generator=g)
    run_and_check(p, names=["weight", "scale"])


@pytest.mark.gpu
def test_expanded_gradient_and_broadcast_modulation(cuda_ready):
    """A gradient of stride 0, and one modulation row expanded over the batch."""
    from gen_worker_b200 import layer_norm

    p = make((3, 20, 200), torch.float32, affine=True, mod=(1, 200))
    x, w, b = (p[n].cuda().requires_grad_(True) for n in ("x", "weight", "bias"))
    s = p["scale"].cuda().requires_grad_(True)
    y = layer_norm(x, w, b, scale=s.expand(3, 200), shift=p["shift"].cuda().expand(3, 200))
    gx, gw, gb, gs = torch.autograd.grad(y.sum(), [x, w, b, s])
    r = {n: p[n].double().requires_grad_(True) for n in ("x", "weight", "bias", "scale")}
    want = norm64(r["x"], r["weight"], r["bias"], r["scale"], p["shift"])
    wx, ww, wb, wsc = torch.autograd.grad(want.sum(), list(r.values()))
    m = norm_magnitudes(p["x"], torch.ones_like(p["x"]), p["weight"], p["bias"], p["scale"],
                        p["shift"], 1e-6)
    check(gx, wx, m["x"], ROW, "x")
    check(gw, ww, m["weight"], COLUMN, "weight")
    check(gb, wb, m["bias"], COLUMN, "bias")
    # three f32 gradients, summed once more over the batch
    check(gs, wsc, m["scale"].sum((0, 1), keepdim=True)[0], COLUMN + 4, "scale")


@pytest.mark.gpu
def test_gradient_against_differences(cuda_ready):
    """<grad, v> against central differences of the 64-bit definition. The
    difference itself is off by h^2 of a third derivative that the rows'
    unit spread keeps under 1e3, and by 2^-52 / h: 1e-5 with h = 1e-4."""
    p = make((2, 9, 48), torch.float32, affine=True, mod=(2, 48))
    _, grads = run_and_check(p)
    h = 1e-4
    for n in ("x", "weight", "bias", "scale", "shift"):
        v = torch.randn(p[n].shape, generator=torch.Generator().manual_seed(7)).double()

        def loss(sign):
            q = {**{k: t.double() for k, t in p.items()}}
            q[n] = q[n] + sign * h * v
            y = norm64(q["x"], q["weight"], q["bias"], wide(q, "scale", q["x"]),
                       wide(q, "shift", q["x"]))
            return float((y * q["dy"]).sum())

        diff = (loss(1) - loss(-1)) / (2 * h)
        got = float((grads[n].double().cpu() * v).sum())
        size = float((grads[n].double().cpu() * v).abs().sum())
        assert abs(got - diff) <= 1e-5 * (1 + size), (n, got, diff)


@pytest.mark.gpu
def test_no_rows(cuda_ready):
    from gen_worker_b200 import layer_norm

    x = torch.empty(0, 5, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    s = torch.zeros(1, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = layer_norm(x, w, scale=s)
    assert y.shape == x.shape
    gx, gw, gs = torch.autograd.grad(y, [x, w, s], torch.empty_like(y))
    assert gx.shape == x.shape and not gw.any() and gw.shape == w.shape and not gs.any()


@pytest.mark.gpu
def test_same_bits_every_run_and_batch_invariant_rows(cuda_ready):
    p = make((2, 1500, 1024), torch.bfloat16, affine=True, mod=(2, 1024))
    y0, g0 = run_and_check(p)
    for _ in range(2):
        y, g = run_and_check(p)
        assert torch.equal(y, y0) and all(torch.equal(g[n], g0[n]) for n in g0)
    from gen_worker_b200 import layer_norm
    x = p["x"].cuda()
    assert torch.equal(layer_norm(x[1:, 7:9]), layer_norm(x)[1:, 7:9])


@pytest.mark.gpu
def test_streams_and_graphs(cuda_ready):
    """On a side stream, and captured with its backward pass and replayed on
    new inputs; two graphs that share nothing replay in turn."""
    from gen_worker_b200 import layer_norm, native

    p = [make((2, 65, 768), torch.bfloat16, seed=k, affine=True, mod=(2, 768)) for k in range(2)]
    want = [run_and_check(q) for q in p]
    names = ["x", "weight", "bias", "scale", "shift"]
    graphs = []
    for k in range(2):
        st = {n: torch.zeros_like(v, device="cuda") for n, v in p[k].items()}
        for n in names:
            st[n].requires_grad_(True)

        def step():
            y = layer_norm(st["x"], st["weight"], st["bias"], scale=st["scale"], shift=st["shift"])
            return [y.detach(), *torch.autograd.grad(y, [st[n] for n in names], st["dy"])]

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
            q = p[(k + turn) % 2]
            with torch.no_grad():
                for n, v in q.items():
                    st[n].copy_(v)
            g.replay()
        torch.cuda.synchronize()
        for k, (g, st, out) in enumerate(graphs):
            y, grads = want[(k + turn) % 2]
            assert torch.equal(out[0], y)
            assert all(torch.equal(o, grads[n]) for o, n in zip(out[1:], names))
    assert native.device_error() == 0


@pytest.mark.gpu
def test_module_and_refusals(cuda_ready):
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    ln = torch.nn.LayerNorm(96, eps=1e-5, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        ln.weight.uniform_(0.5, 1.5)
        ln.bias.uniform_(-1, 1)
    holder = torch.nn.Sequential(ln)
    gw.swap_linears(holder, {"0": gw.norm_from_layer_norm(ln)})
    x = torch.randn(4, 7, 96, device="cuda", dtype=torch.bfloat16)
    m = norm_magnitudes(x.cpu(), x.cpu(), ln.weight.cpu(), ln.bias.cpu(), None, None, 1e-5)["y"]
    check(holder(x), norm64(x.cpu(), ln.weight.cpu(), ln.bias.cpu(), eps=1e-5), m, ROW, "module")

    w = torch.ones(96, device="cuda", dtype=torch.bfloat16)
    bad = [
        lambda: gw.layer_norm(x.double()),
        lambda: gw.layer_norm(x, w.half()),
        lambda: gw.layer_norm(x, w[:95]),
        lambda: gw.layer_norm(x, w, w.float()),
        lambda: gw.layer_norm(x, scale=w.expand(3, 96)),
        lambda: gw.layer_norm(x, scale=w.expand(4, 96), shift=w),
        lambda: gw.layer_norm(x, scale=w.expand(4, 7, 96)),
        lambda: gw.layer_norm(x, w.cpu()),
        lambda: gw.layer_norm(x, eps=-1.0),
        lambda: gw.layer_norm(x[..., :0]),
        lambda: gw.layer_norm(torch.tensor(1.0, device="cuda")),
    ]
    for call in bad:
        with pytest.raises(SvdqB200Error):
            call()
    xr = x.float().requires_grad_(True)
    y = gw.layer_norm(xr)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), xr, create_graph=True)


def test_refusals_on_the_cpu():
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    with pytest.raises(SvdqB200Error, match="no CPU path"):
        gw.layer_norm(torch.zeros(2, 8))
    with pytest.raises(SvdqB200Error, match="not positive"):
        gw.ModulatedLayerNorm(0)
    with pytest.raises(SvdqB200Error, match="features"):
        gw.ModulatedLayerNorm(8)(torch.zeros(2, 9))
    with pytest.raises(SvdqB200Error, match="dimensions"):
        gw.norm_from_layer_norm(torch.nn.LayerNorm((4, 4)))


def test_entry_points_refuse_sizes():
    """Status codes of the C entries for sizes they cannot take, on null
    pointers: nothing is launched."""
    from gen_worker_b200 import native

    lib = native.lib()

    def fwd(m, d, rows, dtype=1):
        return lib.gwb_layer_norm(None, d, None, None, 0, None, 0, None, 0, 0, m, d, rows, 1e-6,
                                  dtype, None, None, None, None)

    assert fwd(0, 8, 1) == 0
    assert fwd(4, 0, 1) == 1 and fwd(4, 8, 0) == 1 and fwd(4, 8, 3) == 1 and fwd(-1, 8, 1) == 1
    assert fwd(4, 8, 4, dtype=3) == 1 and fwd(4, 8, 4) == 1
    assert lib.gwb_layer_norm_backward_work(0, 8, 1) == 0
    assert lib.gwb_layer_norm_backward_work(64, 8, 64) == 8 * 2 * 8
    assert lib.gwb_layer_norm_backward(None, 8, None, 8, None, None, None, None, 0, None, 0, 0, 4, 8,
                                       4, 1, None, None, None, None, None, None, None) == 1
