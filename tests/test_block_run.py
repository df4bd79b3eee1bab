"""The block operators as a transformer block runs them, beside the quantised
linears: modulation -> norm -> quantised qkv -> rotary -> attention -> quantised
out, norm -> gated projections -> quantised down; eager, captured and as a
training step."""

import pytest
import torch

from block_reference import ROTARY_COUNT, U, check, gated64, gated_magnitudes, norm64, norm_magnitudes, rotary64

DIM, HEADS, HEAD, HIDDEN, TOKENS, BATCH = 512, 4, 128, 1024, 97, 2


def build():
    """One block's modules on the GPU, from seeded dense weights."""
    import gen_worker_b200 as gw
    from gen_worker_b200.awq import AwqPackedLinear

    torch.manual_seed(5)

    def linear(i, o):
        lin = torch.nn.Linear(i, o, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            lin.weight.normal_(0, i ** -0.5)
            lin.bias.normal_(0, 0.1)
        return lin

    mod = AwqPackedLinear(DIM, 6 * DIM, bias=True, device="cuda")
    mod.weight.random_(0, 256)
    mod.wscales.fill_(2e-4)
    mod.wzeros.fill_(-15e-4)
    with torch.no_grad():
        mod.bias.normal_(0, 0.1)
    block = torch.nn.ModuleDict({
        "mod": mod, "norm1": gw.ModulatedLayerNorm(DIM, affine=False, device="cuda"),
        "norm2": gw.ModulatedLayerNorm(DIM, affine=False, device="cuda"),
        "qkv": gw.svdq_int4_from_linear(linear(DIM, 3 * DIM)),
        "out": gw.fp8_rowwise_from_linear(linear(DIM, DIM)),
        "ff": gw.gated_from_linears(linear(DIM, HIDDEN), linear(DIM, HIDDEN), activation="gelu_tanh",
                                    down=gw.svdq_int4_from_linear(linear(HIDDEN, DIM))),
        "rope": gw.RotaryEmbedding(HEAD, interleaved=True, axes=(16, 56, 56), device="cuda"),
    })
    return block.requires_grad_(False)


def forward(m, x, cond, pos, seen=None):
    def note(name, *tensors):
        if seen is not None:
            seen[name] = [t.clone() for t in tensors]

    shift1, scale1, gate1, shift2, scale2, gate2 = m["mod"](cond).chunk(6, -1)
    a = m["norm1"](x, scale1, shift1)
    note("norm1", x, scale1, shift1, a)
    qkv = m["qkv"](a).view(BATCH, TOKENS, 3 * HEADS, HEAD)
    q, k = qkv[:, :, :HEADS], qkv[:, :, HEADS:2 * HEADS]
    qr, kr = m["rope"](q, k, pos)
    note("rope", q, k, qr, kr)
    s = torch.einsum("bihd,bjhd->bhij", qr, kr).float() * HEAD ** -0.5
    att = torch.einsum("bhij,bjhd->bihd", s.softmax(-1).to(x.dtype), qkv[:, :, 2 * HEADS:])
    x = x + gate1.unsqueeze(1) * m["out"](att.reshape(BATCH, TOKENS, DIM))
    b = m["norm2"](x, scale2, shift2)
    note("norm2", x, scale2, shift2, b)
    ff = m["ff"]
    if seen is not None:
        import gen_worker_b200 as gw
        note("gated", b, gw.gated_linear(b, ff.w_gate, ff.w_up, ff.b_gate, ff.b_up,
                                         activation=ff.activation))
    return x + gate2.unsqueeze(1) * ff(b)


def inputs(seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(BATCH, TOKENS, DIM, generator=g)
    x[..., ::100] *= 20                                   # activation outliers
    cond = torch.randn(BATCH, DIM, generator=g)
    pos = torch.randint(0, 128, (BATCH, TOKENS, 3), generator=g)
    return x.bfloat16().cuda(), cond.bfloat16().cuda(), pos.cuda()


@pytest.mark.gpu
def test_block_stages(cuda_ready):
    """Each new operator against its definition on what the stage before gave it."""
    m, seen = build(), {}
    x, cond, pos = inputs(0)
    with torch.no_grad():
        y = forward(m, x, cond, pos, seen)
    assert torch.isfinite(y).all()
    for name in ("norm1", "norm2"):
        xin, s, t, out = (v.cpu() for v in seen[name])
        s, t = s.unsqueeze(1), t.unsqueeze(1)
        check(out, norm64(xin, s=s, t=t), norm_magnitudes(xin, xin, None, None, s, t, 1e-6)["y"], 80, name)
    q, k, qr, kr = seen["rope"]
    rope = m["rope"]
    for a, b in ((q, qr), (k, kr)):
        want, mag = rotary64(a.cpu(), pos.cpu(), rope.inv_freq.cpu(), rope.axis.cpu(), True, 1.0)
        check(b, want, mag, ROTARY_COUNT, "rope")
    b, h = (v.cpu().flatten(0, 1) for v in seen["gated"])
    w = [t.detach().cpu() for t in (m["ff"].w_gate, m["ff"].w_up, m["ff"].b_gate, m["ff"].b_up)]
    h64 = gated64(b, *w, "gelu_tanh")
    check(h, h64[0], gated_magnitudes(b, *w, None, h64)["h"], 1 / U, "gated")


@pytest.mark.gpu
def test_block_captured(cuda_ready):
    """The whole block in one graph, replayed on new contents, gives the bits
    of the eager calls."""
    from gen_worker_b200 import native

    m = build()
    with torch.no_grad():
        want = [forward(m, *inputs(k)) for k in range(3)]
        x, cond, pos = inputs(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            forward(m, x, cond, pos)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = forward(m, x, cond, pos)
        for k in (2, 1, 0):
            for dst, src in zip((x, cond, pos), inputs(k)):
                dst.copy_(src)
            graph.replay()
            assert torch.equal(y, want[k])
    assert native.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("recompute", [False, True])
def test_training_step(cuda_ready, recompute):
    """Gradients of norm -> gated -> down -> rotary through a whole step, against
    64-bit autograd of the same bf16 values. Between x and a gradient lie at most
    12 tensors rounded to bf16, each off by at most 2^-8 of its own norm (half a
    step, relative), and none of the maps between them (rotations, a norm of unit
    rows, products with weights of unit gain) stretches a relative error more
    than twofold: 12 * 2 * 2^-8 bounds the relative L2 error."""
    import gen_worker_b200 as gw

    torch.manual_seed(0)
    dim, hidden = 256, 344
    ff = gw.GatedFeedForward(dim, hidden, bias=True, recompute=recompute, device="cuda",
                             down=torch.nn.Linear(hidden, dim, device="cuda", dtype=torch.bfloat16))
    norm = gw.ModulatedLayerNorm(dim, device="cuda")
    rope = gw.RotaryEmbedding(64, device="cuda")
    x, s, t = (torch.randn(*n, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
               for n in ((2, 150, dim), (2, dim), (2, dim)))
    goal = torch.randn(2, 150, 4, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(150, device="cuda")
    leaves = {"x": x, "scale": s, "shift": t, **dict(norm.named_parameters()),
              **{n: p for n, p in ff.named_parameters()}}
    y, _ = rope((x + ff(norm(x, s, t))).view(2, 150, 4, 64), None, pos)
    (y * goal).sum().backward()

    r = {n: p.detach().cpu().double().requires_grad_(True) for n, p in leaves.items()}
    b = norm64(r["x"], r["weight"], r["bias"], r["scale"].unsqueeze(1), r["shift"].unsqueeze(1))
    h = gated64(b.flatten(0, 1), r["w_gate"], r["w_up"], r["b_gate"], r["b_up"], "silu")[0]
    z = r["x"] + (h @ r["down.weight"].t() + r["down.bias"]).view(2, 150, dim)
    z = z.view(2, 150, 4, 64)
    ang = pos.cpu().double()[:, None] * rope.inv_freq.cpu()
    c, sn = ang.cos()[:, None], ang.sin()[:, None]
    p, q = z[..., :32], z[..., 32:]
    out = torch.cat([p * c - q * sn, q * c + p * sn], -1)
    (out * goal.cpu().double()).sum().backward()
    for n, leaf in leaves.items():
        got, want = leaf.grad.double().cpu(), r[n].grad
        rel = float((got - want).norm() / want.norm())
        assert rel <= 12 * 2 * 2.0 ** -8, (n, rel)


@pytest.mark.gpu
def test_captured_backward_beside_an_eager_graph(cuda_ready):
    """Capturing a pass with gradients while an eager graph of the same leaves
    lives is refused where it begins; leaves of its own, or no such graph, and
    it gives the eager bits."""
    import gen_worker_b200 as gw

    x = torch.randn(40, 64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    w = torch.randn(72, 64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    rope = gw.RotaryEmbedding(16, device="cuda")
    pos = torch.arange(40, device="cuda")
    calls = [lambda x, w: gw.layer_norm(x), lambda x, w: gw.gated_linear(x, w, w),
             lambda x, w: rope(x.view(40, 4, 16), None, pos)[0]]

    def capture(call, x, w):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(x, w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(x, w)
            out = torch.autograd.grad(y, x, torch.ones_like(y))
        return graph, out

    for i, call in enumerate(calls):
        y = call(x, w)                                   # the eager graph lives
        if i < 2:                                        # rotary's q is a view: no leaf of its own
            with pytest.raises(RuntimeError, match="leaves of its own"):
                capture(call, x, w)
        mine = [t.detach().requires_grad_(True) for t in (x, w)]
        graph, inside = capture(call, *mine)
        graph.replay()
        outside, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(inside[0], outside)
        del y, inside, graph
        graph, inside = capture(call, x, w)              # and with it gone
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(inside[0], outside)


@pytest.mark.gpu
def test_two_streams_at_once(cuda_ready):
    """The same calls from two streams at the same time share nothing."""
    import gen_worker_b200 as gw

    g = torch.Generator().manual_seed(4)
    sets = [[torch.randn(*n, generator=g).bfloat16().cuda() for n in ((600, 512), (776, 512), (776, 512),
                                                                     (600, 776))] for _ in range(2)]
    pos = torch.arange(600, device="cuda")
    rope = gw.RotaryEmbedding(64, device="cuda")

    def step(x, wg, wu, dh):
        x = x.detach().requires_grad_(True)
        a = gw.layer_norm(x)
        b, _ = rope(a.view(600, 8, 64), None, pos)
        h = gw.gated_linear(b.reshape(600, 512), wg, wu)
        small = gw.gated_linear(b.reshape(600, 512)[:9], wg, wu)
        return [h.detach(), small.detach(), *torch.autograd.grad(h, x, dh)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(step(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for run in got[k] for a, b in zip(run, want[k]))


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_ready):
    """Tensors of over 2^31 elements: the last rows come out as the definition
    has them, and sums over all rows count every one."""
    import gen_worker_b200 as gw

    def near(got, want, count):
        """Within one rounding and `count` f32 roundings of unit values."""
        tol = 2.0 ** -8 * want.abs() + count * U * 8
        assert ((got.double() - want).abs() <= tol).all()

    # norm: 2.2e9 elements; ones in dy make the column sums row counts
    rows, dim = 270_000, 8192
    x = torch.empty(rows, dim, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_(True)
    w = torch.ones(dim, device="cuda").requires_grad_(True)
    b = torch.zeros(dim, device="cuda").requires_grad_(True)
    y = gw.layer_norm(x, w, b)
    tail = x.detach()[-3:].double()
    near(y.detach()[-3:], (tail - tail.mean(1, keepdim=True)) / tail.var(1, correction=0, keepdim=True)
         .add(1e-6).sqrt(), 80)
    dy = torch.ones_like(x)
    gx, gb = torch.autograd.grad(y, [x, b], dy)
    assert torch.equal(gb, torch.full_like(gb, float(rows)))
    near(gx[-3:], torch.zeros(3, dim, device="cuda", dtype=torch.float64), 400)
    del x, y, dy, gx, tail
    # rotary: one head's last tokens
    q = torch.empty(1, 4_200_000, 4, 128, device="cuda", dtype=torch.bfloat16).normal_()
    pos = torch.arange(4_200_000, device="cuda") % 5000
    rope = gw.RotaryEmbedding(128, device="cuda")
    qo, _ = rope(q, None, pos)
    again, _ = rope(q[:, -50:].clone(), None, pos[-50:])
    assert torch.equal(qo[:, -50:], again)
    del q, qo
    # gated: h of 2.2e9 elements, with its backward pass
    rows, dim, hidden = 180_000, 64, 12288
    x = torch.randn(rows, dim, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    wg, wu = (torch.randn(hidden, dim, device="cuda", dtype=torch.bfloat16) * 0.1 for _ in range(2))
    h = gw.gated_linear(x, wg, wu)
    few = x.detach()[-200:].clone().requires_grad_(True)
    part = gw.gated_linear(few, wg, wu)
    assert torch.equal(h.detach()[-200:], part)
    dh = torch.ones_like(h)
    gx, = torch.autograd.grad(h, x, dh)
    gp, = torch.autograd.grad(part, few, dh[:200])
    assert float((gx[-200:].double() - gp.double()).norm() / gp.double().norm()) <= 2.0 ** -8


def test_package_lists_the_operators():
    """The entry points are exported, and the library has the C functions."""
    import gen_worker_b200 as gw
    from gen_worker_b200 import native

    for name in ("layer_norm", "ModulatedLayerNorm", "rotary", "rotary_", "RotaryEmbedding",
                 "gated_linear", "GatedFeedForward"):
        assert name in gw.__all__ and callable(getattr(gw, name))
    lib = native.lib()
    for name in native.EXPORTED:
        assert hasattr(lib, name)


def test_fake_tensors_trace_through():
    """Shapes and types for torch.compile, without a GPU."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import gen_worker_b200 as gw

    with FakeTensorMode():
        x = torch.empty(2, 5, 64, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(72, 64, device="cuda", dtype=torch.bfloat16)
        assert gw.layer_norm(x).shape == x.shape
        assert gw.gated_linear(x, w, w).shape == (2, 5, 72)
        q, k = gw.rotary(x.view(2, 5, 2, 32), None, torch.empty(5, device="cuda", dtype=torch.int64),
                         torch.empty(8, device="cuda", dtype=torch.float64))
        assert q.shape == (2, 5, 2, 32) and k is None


def _fake_calls():
    """Each operator on fake tensors: (call of its tensors, the tensors)."""
    import gen_worker_b200 as gw

    def new(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    pos, inv = new(5, dtype=torch.int64), new(8, dtype=torch.float64)
    return [
        (lambda x, w, b, s, t: gw.layer_norm(x, w, b, scale=s, shift=t),
         [new(2, 5, 64), new(64), new(64), new(2, 64), new(2, 64)]),
        (lambda q, k: gw.rotary(q, k, pos, inv), [new(2, 5, 2, 32), new(2, 5, 1, 32)]),
        (lambda x, a, b, c, d: gw.gated_linear(x, a, b, c, d),
         [new(2, 5, 64), new(72, 64), new(72, 64), new(72), new(72)]),
        (lambda x, a, b: gw.gated_linear(x, a, b, recompute=True),
         [new(2, 5, 64), new(72, 64), new(72, 64)]),
    ]


def test_fake_tensors_trace_what_needs_gradients():
    """The calls of a training step trace on a machine without a GPU, and the
    backward ops' fakes give each gradient its parameter's shape and type. (The
    autograd engine itself asks for the device: the whole pass runs below.)"""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        for call, tensors in _fake_calls():
            out = call(*(t.detach().requires_grad_(True) for t in tensors))
            for o in out if isinstance(out, tuple) else [out]:
                assert o.requires_grad
        ops = torch.ops.gwb200
        (_, norm), (_, qk), (_, gated), _ = _fake_calls()
        y, mean, rstd = ops.layer_norm_stats(*norm, 1e-6)
        h, kept = ops.gated_linear_keep(*gated, 0)
        assert mean.shape == rstd.shape == (10,) and mean.dtype == torch.float32
        for mask in ([True] * 5, [True, False, True, False, True]):
            for given, grads in ((norm, ops.layer_norm_backward(y, norm[0], mean, rstd, *norm[1:], mask)),
                                 (gated, ops.gated_linear_backward(h, *gated, kept, 0, mask)),
                                 (gated, ops.gated_linear_backward(h, *gated, None, 0, mask))):
                for t, g, on in zip(given, grads, mask):
                    assert g.shape == (t.shape if on else (0,)) and g.dtype == t.dtype


@pytest.mark.gpu
def test_fake_tensors_trace_gradients(cuda_ready):
    """Forward and backward shapes of every operator through autograd."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        for call, tensors in _fake_calls():
            for some in (tensors, tensors[:1]):
                leaves = [t.detach().requires_grad_(any(t is s for s in some)) for t in tensors]
                out = call(*leaves)
                out = list(out) if isinstance(out, tuple) else [out]
                wanted = [t for t in leaves if t.requires_grad]
                grads = torch.autograd.grad(out, wanted, [torch.ones_like(o) for o in out],
                                            allow_unused=True)
                assert grads[0] is not None
                for t, g in zip(wanted, grads):
                    assert g is None or (g.shape == t.shape and g.dtype == t.dtype)


def _dual_calls(calls):
    """Calls with a tangent on one of their tensors, by forward_ad and by jvp."""
    from torch.autograd import forward_ad

    for call, tensors in calls:
        for i in range(len(tensors)):
            def dual(call=call, tensors=tensors, i=i):
                with forward_ad.dual_level():
                    mixed = list(tensors)
                    mixed[i] = forward_ad.make_dual(tensors[i], torch.ones_like(tensors[i]))
                    return call(*mixed)

            yield dual


def test_forward_mode_is_refused():
    """A tangent on any input is refused, never dropped."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    with FakeTensorMode():
        calls = _fake_calls()
        pos = torch.empty(5, device="cuda", dtype=torch.float32)
        inv = torch.empty(8, device="cuda", dtype=torch.float64)
        q = [torch.empty(2, 5, 2, 32, device="cuda") for _ in range(2)]
        calls.append((lambda q, k, p, f: gw.rotary(q, k, p, f), [*q, pos, inv]))
        calls.append((lambda q, k, p, f: gw.rotary_(q, k, p, f), [*q, pos, inv]))
        for dual in _dual_calls(calls):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(SvdqB200Error, match="forward-mode"):
                    dual()


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_gpu(cuda_ready):
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    x = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(72, 64, device="cuda", dtype=torch.bfloat16)
    rope = gw.RotaryEmbedding(16, device="cuda")
    pos = torch.arange(4, device="cuda")
    calls = [(lambda x: gw.layer_norm(x), [x]), (lambda x, w: gw.gated_linear(x, w, w), [x, w]),
             (lambda x: rope(x.view(4, 4, 16), None, pos), [x]),
             (lambda x: rope.rotate_(x.view(4, 4, 16), None, pos), [x.clone()])]
    for dual in _dual_calls(calls):
        with pytest.raises(SvdqB200Error, match="forward-mode"):
            dual()


@pytest.mark.gpu
def test_compiled_training_step(cuda_ready):
    """A step through torch.compile gives the eager bits, forward and backward."""
    import gen_worker_b200 as gw

    torch.manual_seed(1)
    ff = gw.GatedFeedForward(64, 72, bias=True, device="cuda")
    norm = gw.ModulatedLayerNorm(64, device="cuda")
    rope = gw.RotaryEmbedding(16, device="cuda")
    pos = torch.arange(40, device="cuda")

    def step(x, s, t):
        a, _ = rope(norm(x, s, t).view(2, 40, 4, 16), None, pos)
        return ff(a.reshape(2, 40, 64))

    leaves = [torch.randn(*n, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
              for n in ((2, 40, 64), (2, 64), (2, 64))]
    want = step(*leaves)
    dh = torch.randn_like(want)
    params = [*leaves, *ff.parameters(), *norm.parameters()]
    grads = torch.autograd.grad(want, params, dh)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, params, dh), grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_saved_tensor_hooks(cuda_ready):
    """Kept tensors pass through saved-tensor hooks (offload to the host)."""
    import gen_worker_b200 as gw

    x = torch.randn(40, 64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    w = torch.randn(72, 64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)

    def step():
        h = gw.gated_linear(gw.layer_norm(x), w, w)
        return torch.autograd.grad(h, [x, w], torch.ones_like(h))

    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_sizes_past_32_bit_steps_are_refused():
    """Sizes near 2^31, whose rounding up would wrap, and more columns than a
    grid takes: status codes of the C entries on null pointers, nothing is
    launched."""
    from gen_worker_b200 import native

    lib, full, capacity = native.lib(), (1 << 31) - 8, 8

    def norm(m, d):
        return lib.gwb_layer_norm(None, d, None, None, 0, None, 0, None, 0, 0, m, d, m, 1e-6, 1,
                                  None, None, None, None)

    def norm_backward(m, d, dw=None):
        return lib.gwb_layer_norm_backward(None, d, None, d, None, None, None, None, 0, None, 0, 0, m,
                                           d, m, 1, None, dw, None, None, None, None, None)

    def gated(m, d, f):
        a = lib.gwb_gated_linear(None, d, None, None, None, None, m, d, f, 0, 1, None, None)
        b = lib.gwb_gated_linear_backward(None, f, None, d, *[None] * 5, m, d, f, 0, 1, *[None] * 7)
        assert a == b
        return a

    for m, d in ((1, full), (full, 8), (1, (1 << 30) + 1)):
        assert norm(m, d) == capacity and norm_backward(m, d) == capacity
    assert norm(1, 1 << 30) == 1 and norm_backward(1, 1 << 30) == 1        # null pointers
    assert norm_backward(1, 2097121, dw=16) == capacity and norm_backward(1, 2097120, dw=16) == 1
    for sizes in ((1, 8, full), (1, full, 8), (full, 8, 8)):
        assert gated(*sizes) == capacity
    assert gated(1, 8, 1 << 27) == 1
    assert lib.gwb_rotary(None, None, None, None, 1 << 62, None, None, None, None, 1 << 62, None, 0, None,
                          None, None, 1, 1, 1, 2, 8, 1.0, 0, 0, 1, None) == 1
