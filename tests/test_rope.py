"""Rotary positions: layouts, partial heads, axes, far positions, strides,
gradients, in-place form, and what the entry points refuse."""

import math

import pytest
import torch

from block_reference import ROTARY_COUNT, check, rotary64

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(b, s, h, hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    fused = torch.randn(b, s, h + 2 * hk, d, generator=g).to(dtype)
    return fused, g


def verify(q, k, pos, rope, qo, ko, sign=1.0, what=""):
    ax = None if rope.axis is None else rope.axis.cpu()
    for name, x, y in (("q", q, qo), ("k", k, ko)):
        if x is None:
            continue
        want, mag = rotary64(x.cpu(), pos.cpu(), rope.inv_freq.cpu(), ax, rope.interleaved,
                             rope.attention_scale, sign)
        check(y, want, mag, ROTARY_COUNT, what + name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (96, 64), (80, 40), (256, 256), (6, 2),
                                   (7, 6), (36, 20), (192, 96)])
def test_layouts(cuda_ready, dtype, interleaved, d, rot):
    from gen_worker_b200 import RotaryEmbedding

    fused, g = inputs(2, 19, 6, 2, d, dtype, seed=d)
    dev = fused.cuda()
    q, k = dev[:, :, :6], dev[:, :, 6:8]
    pos = torch.randint(0, 5000, (2, 19), generator=g)
    rope = RotaryEmbedding(rot, interleaved=interleaved, device="cuda")
    qo, ko = rope(q, k, pos.cuda())
    verify(q, k, pos, rope, qo, ko)
    rest = slice(rot, d)
    assert torch.equal(qo[..., rest], q[..., rest]) and torch.equal(ko[..., rest], k[..., rest])
    # in place on the fused projection's own memory; values beside them stay
    rope.rotate_(q, k, pos.cuda())
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(dev[:, :, 8:].cpu(), fused[:, :, 8:])


@pytest.mark.gpu
@pytest.mark.parametrize("b,s,h,hk", [(1, 1, 1, 1), (1, 1, 64, 8), (48, 1, 32, 8), (3, 1, 5, 5),
                                      (1, 333, 24, 24), (2, 700, 3, 1), (1, 5000, 2, 2)])
def test_sizes(cuda_ready, b, s, h, hk):
    from gen_worker_b200 import RotaryEmbedding

    fused, g = inputs(b, s, h, hk, 128, torch.bfloat16)
    q, k = fused.cuda()[:, :, :h], fused.cuda()[:, :, h:h + hk]
    pos = torch.randint(0, 1 << 17, (b, s), generator=g)
    for inter in (False, True):
        rope = RotaryEmbedding(128, interleaved=inter, device="cuda")
        verify(q, k, pos, rope, *rope(q, k, pos.cuda()))
        qo, none = rope(q, None, pos.cuda())
        assert none is None
        verify(q, None, pos, rope, qo, None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes_and_position_types(cuda_ready, kind, interleaved):
    from gen_worker_b200 import RotaryEmbedding

    fused, g = inputs(2, 40, 4, 4, 128, torch.float32)
    q, k = fused.cuda()[:, :, :4], fused.cuda()[:, :, 4:8]
    pos = torch.randint(-30, 200, (2, 40, 3), generator=g).to(kind)
    if kind == torch.float32:
        pos = pos + 0.25
    rope = RotaryEmbedding(128, interleaved=interleaved, axes=(16, 56, 56), device="cuda")
    verify(q, k, pos, rope, *rope(q, k, pos.cuda()))
    # one sequence's positions for the whole batch, [S, A] and [1, S, A]; strided positions
    for form in (pos[0].cuda(), pos[:1].cuda(), pos.cuda().transpose(1, 2).contiguous().transpose(1, 2)[:1]):
        verify(q, k, pos[:1], rope, *rope(q, k, form))
    one = RotaryEmbedding(128, interleaved=interleaved, device="cuda")
    verify(q, k, pos[:1, :, 0], one, *one(q, k, pos[0, :, 0].cuda()))


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "by_parts"])
def test_far_positions(cuda_ready, scaling):
    """Positions whose angles an f32 product would lose; up to 2^26 the f64
    product is off by less than 2^-26 rad, an eighth of ROTARY_COUNT."""
    from gen_worker_b200 import RotaryEmbedding

    fused, _ = inputs(1, 8, 4, 2, 128, torch.float32)
    q, k = fused.cuda()[:, :, :4], fused.cuda()[:, :, 4:6]
    pos = torch.tensor([[0, 1, 4095, 131071, 1 << 20, (1 << 24) + 1, (1 << 26) - 1, 1 << 26]])
    rope = RotaryEmbedding(128, scaling=scaling, factor=8.0, trained_length=4096, device="cuda")
    verify(q, k, pos, rope, *rope(q, k, pos.cuda()))


@pytest.mark.gpu
def test_strides(cuda_ready):
    """[B, H, S, D] tensors seen as [B, S, H, D], odd element offsets, no
    batch dimension, and a last dimension that is not dense."""
    from gen_worker_b200 import RotaryEmbedding, rotary

    g = torch.Generator().manual_seed(3)
    base = torch.randn(2, 6, 50, 65, generator=g).to(torch.float16).cuda()
    pos = torch.arange(50)
    rope = RotaryEmbedding(64, device="cuda")
    for x in (base[..., :64].transpose(1, 2), base[..., 1:].transpose(1, 2),
              base.permute(0, 1, 3, 2)[:, :, :64, :].permute(0, 3, 1, 2)):
        qo, ko = rope(x, x[:, :, :2], pos.cuda())
        verify(x, x[:, :, :2], pos[None], rope, qo, ko)
    x = base[0, ..., :64].transpose(0, 1)
    qo, ko = rope(x, x, pos.cuda())
    verify(x[None], x[None], pos[None], rope, qo[None], ko[None])
    y = base[..., 1:].transpose(1, 2).clone()
    want, _ = rotary(y, None, pos.cuda(), rope.inv_freq)
    z = base[..., 1:].transpose(1, 2)
    rope.rotate_(z, None, pos.cuda())
    assert torch.equal(z, want)


@pytest.mark.gpu
@pytest.mark.parametrize("b,s,h,hk", [(1, 7, 4, 4), (2, 7, 4, 4), (3, 1, 4, 2), (2, 5, 2, 2),
                                      (2, 9, 6, 2)])
def test_in_place_in_common_layouts(cuda_ready, b, s, h, hk):
    """q and k of one fused tensor with its dimensions in any order: they share
    no element, so both are rotated where they lie."""
    from gen_worker_b200 import RotaryEmbedding

    rope = RotaryEmbedding(64, device="cuda")
    pos = torch.arange(s, device="cuda") + 5
    g = torch.Generator().manual_seed(b + s)
    fused = torch.randn(b, s, h + 2 * hk, 64, generator=g)
    for order in ((0, 1, 2, 3), (0, 2, 1, 3), (1, 0, 2, 3), (1, 2, 0, 3), (2, 0, 1, 3), (2, 1, 0, 3)):
        back = [order.index(i) for i in range(4)]
        base = fused.permute(order).contiguous().cuda()       # the layout in memory
        view = base.permute(back)                             # as [B, S, heads, D]
        q, k = view[:, :, :h], view[:, :, h:h + hk]
        qo, ko = rope(q, k, pos)
        rope.rotate_(q, k, pos)
        assert torch.equal(q, qo) and torch.equal(k, ko), order
        assert torch.equal(view[:, :, h + hk:].cpu(), fused[:, :, h + hk:])
    mesh = fused.reshape(b, s, -1, 2, 64).cuda() if h == hk else None     # heads of q and k in turn
    if mesh is not None:
        q, k = mesh[:, :, :, 0], mesh[:, :, :, 1]
        qo, ko = rope(q, k, pos)
        rope.rotate_(q, k, pos)
        assert torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.gpu
def test_in_place_still_refuses_shared_elements(cuda_ready):
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    inv = gw.rotary_frequencies(16)[0].cuda()
    pos = torch.arange(6, device="cuda")
    base = torch.randn(2, 8, 6, 16, device="cuda")           # [B, heads, S, D]
    flat = torch.randn(4000, device="cuda")
    pairs = [
        (base[:, :4].transpose(1, 2), base[:, 3:7].transpose(1, 2)),
        (base[:1, :4].transpose(1, 2), base[:1, 3:4].transpose(1, 2)),
        # k one feature behind q, and in steps that meet q's only now and then
        (flat[:768].view(1, 6, 8, 16), flat[1:769].view(1, 6, 8, 16)),
        (flat.as_strided((1, 6, 2, 16), (0, 100, 32, 1)),
         flat.as_strided((1, 6, 2, 16), (0, 70, 32, 1), 16)),
    ]
    for q, k in pairs:
        with pytest.raises(SvdqB200Error, match="share memory"):
            gw.rotary_(q, k, pos, inv)


@pytest.mark.gpu
def test_in_place_refuses_a_tensor_over_itself(cuda_ready):
    """Windows of one buffer that overlap are refused, those that only lie close
    are rotated."""
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    inv = gw.rotary_frequencies(16)[0].cuda()
    pos = torch.arange(6, device="cuda")
    flat = torch.randn(4000, device="cuda")
    over = [((1, 6, 2, 16), (0, 24, 16, 1)), ((2, 6, 2, 16), (100, 32, 16, 1)),
            ((1, 6, 2, 16), (0, 0, 16, 1)), ((1, 6, 3, 16), (0, 32, 16, 1)),
            ((1, 6, 2, 16), (0, 32, 15, 1)), ((2, 6, 2, 16), (176, 34, 17, 1))]
    for size, stride in over:
        with pytest.raises(SvdqB200Error, match="overlaps itself"):
            gw.rotary_(flat.as_strided(size, stride), None, pos, inv)
        with pytest.raises(SvdqB200Error, match="overlaps itself"):
            gw.rotary_(torch.randn(size, device="cuda"), flat.as_strided(size, stride), pos, inv)
    close = [((1, 6, 2, 16), (7, 32, 16, 1)), ((2, 6, 2, 16), (192, 32, 16, 1)),
             ((2, 6, 2, 16), (32, 64, 16, 1)), ((2, 6, 2, 16), (16, 64, 32, 1)),
             ((2, 6, 2, 16), (999, 17, 500, 1)), ((1, 1, 2, 16), (0, 3, 16, 1))]
    for size, stride in close:
        q = flat.as_strided(size, stride)
        want, _ = gw.rotary(q, None, pos[:size[1]], inv)
        gw.rotary_(q, None, pos[:size[1]], inv)
        assert torch.equal(q, want), (size, stride)


@pytest.mark.gpu
def test_in_place_counts_as_a_change(cuda_ready):
    """Autograd must see that a saved tensor was rotated, in inference mode too."""
    from gen_worker_b200 import RotaryEmbedding

    rope = RotaryEmbedding(16, device="cuda")
    pos = torch.arange(3, device="cuda")
    for mode in (torch.no_grad, torch.inference_mode):
        q, k = (torch.randn(1, 3, 2, 16, device="cuda") for _ in range(2))
        w = torch.randn(16, device="cuda", requires_grad=True)
        y = (w * q).sum() + (w * k).sum()
        with mode():
            before = q._version, k._version
            rope.rotate_(q, k, pos)
            assert (q._version, k._version) == (before[0] + 1, before[1] + 1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.gpu
def test_learned_angles_are_refused(cuda_ready):
    """No gradient reaches positions or frequencies: asking for one is an error,
    not a silent zero."""
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    q = torch.randn(1, 3, 2, 16, device="cuda")
    pos = torch.arange(3, device="cuda").float()
    inv = gw.rotary_frequencies(16)[0].cuda()
    for p, f in ((pos.clone().requires_grad_(True), inv), (pos, inv.clone().requires_grad_(True))):
        for x in (q, q.clone().requires_grad_(True)):
            with pytest.raises(SvdqB200Error, match="gradient"):
                gw.rotary(x, None, p, f)
        with pytest.raises(SvdqB200Error, match="gradient"):
            gw.rotary_(q, None, p, f)
        with torch.no_grad():
            assert gw.rotary(q, None, p, f)[0].shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(cuda_ready, dtype, interleaved):
    from gen_worker_b200 import RotaryEmbedding

    fused, g = inputs(2, 33, 4, 2, 96, dtype)
    dev = fused.cuda().requires_grad_(True)
    q, k = dev[:, :, :4], dev[:, :, 4:6]
    pos = torch.randint(0, 9000, (2, 33), generator=g)
    rope = RotaryEmbedding(64, interleaved=interleaved, scaling="by_parts", factor=4.0,
                           trained_length=2048, device="cuda")
    qo, ko = rope(q, k, pos.cuda())
    dq, dk = torch.randn_like(qo), torch.randn_like(ko)
    gq, gk = torch.autograd.grad([qo, ko], [q, k], [dq, dk], retain_graph=True)
    verify(dq, dk, pos, rope, gq, gk, sign=-1.0)
    # one of the two alone; into the fused tensor, whose values get nothing
    only, = torch.autograd.grad(ko, [k], [dk], retain_graph=True)
    assert torch.equal(only, gk)
    full, = torch.autograd.grad([qo, ko], [dev], [dq, dk])
    assert torch.equal(full[:, :, :4], gq) and torch.equal(full[:, :, 4:6], gk)
    assert not full[:, :, 6:].any()


@pytest.mark.gpu
def test_gradient_against_differences(cuda_ready):
    """The map is linear: <grad, v> = <dq, f(x + v) - f(x)> of the definition,
    up to the f32 roundings of the gradient."""
    from gen_worker_b200 import RotaryEmbedding

    fused, g = inputs(1, 12, 2, 1, 32, torch.float32)
    q = fused[:, :, :2].cuda().requires_grad_(True)
    pos = torch.randint(0, 999, (1, 12), generator=g)
    rope = RotaryEmbedding(32, device="cuda")
    dq, v = torch.randn(1, 12, 2, 32, generator=g), torch.randn(1, 12, 2, 32, generator=g)
    grad, = torch.autograd.grad(rope(q, None, pos.cuda())[0], q, dq.cuda())
    f0, _ = rotary64(q.detach().cpu(), pos, rope.inv_freq.cpu(), None, False, 1.0)
    f1, _ = rotary64(q.detach().cpu().double() + v.double(), pos, rope.inv_freq.cpu(), None, False, 1.0)
    diff = float(((f1 - f0) * dq.double()).sum())
    got = float((grad.double().cpu() * v.double()).sum())
    assert abs(got - diff) <= (ROTARY_COUNT + 1) * 2.0 ** -24 * 2 * float((dq.abs().sum() * v.abs().max()))


@pytest.mark.gpu
def test_second_order_streams_and_graphs(cuda_ready):
    from gen_worker_b200 import RotaryEmbedding

    fused, _ = inputs(1, 17, 3, 1, 64, torch.float32)
    rope = RotaryEmbedding(64, device="cuda")
    pos = torch.arange(17, device="cuda")
    q = fused[:, :, :3].cuda().requires_grad_(True)
    d = torch.randn_like(q).requires_grad_(True)
    gq, = torch.autograd.grad(rope(q, None, pos)[0], q, d, create_graph=True)
    back, = torch.autograd.grad(gq, d, fused[:, :, :3].cuda())
    assert torch.equal(back, rope(q, None, pos)[0])   # the transpose's transpose

    # captured in place for one token each, replayed on new contents
    x, at = torch.zeros(5, 1, 4, 64, device="cuda"), torch.zeros(5, 1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope.rotate_(x, None, at)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope.rotate_(x, None, at)
    for k in range(2):
        new = torch.randn(5, 1, 4, 64)
        x.copy_(new)
        at.fill_(1000 + k)
        graph.replay()
        verify(new, None, torch.full((5, 1), 1000 + k), rope, x, None)


@pytest.mark.gpu
def test_empty_and_non_finite(cuda_ready):
    from gen_worker_b200 import RotaryEmbedding

    rope = RotaryEmbedding(64, device="cuda")
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y, _ = rope(x, None, torch.zeros(shape[1], dtype=torch.int64, device="cuda"))
        g, = torch.autograd.grad(y, x, torch.empty_like(y))
        assert y.shape == x.shape == g.shape
    x = torch.randn(1, 3, 1, 64)
    x[0, 1, 0, 5] = float("nan")
    x[0, 2, 0, 6] = float("inf")
    y, _ = rope(x.cuda(), None, torch.tensor([3, 4, 5], device="cuda"))
    bad = torch.isfinite(y[0, :, 0]).logical_not().cpu()
    want = torch.zeros(3, 64, dtype=torch.bool)
    want[1, 5] = want[1, 37] = want[2, 6] = want[2, 38] = True
    assert torch.equal(bad, want)


@pytest.mark.gpu
def test_refusals(cuda_ready):
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    q = torch.randn(2, 5, 4, 64, device="cuda")
    pos = torch.arange(5, device="cuda")
    inv, _, _ = gw.rotary_frequencies(64)
    inv = inv.cuda()
    axis = torch.zeros(32, dtype=torch.int32, device="cuda")
    bad = [
        lambda f: f(q, q[:1], pos, inv), lambda f: f(q, q.half(), pos, inv),
        lambda f: f(q, q[..., :32], pos, inv), lambda f: f(q, None, pos[:4], inv),
        lambda f: f(q, None, pos.double(), inv), lambda f: f(q, None, pos, inv.float()),
        lambda f: f(q[..., :62], None, pos, inv), lambda f: f(q, None, pos.cpu(), inv),
        lambda f: f(q, None, pos, inv, axis=axis), lambda f: f(q, None, pos, inv, axis=axis[:5]),
        lambda f: f(q, None, pos.expand(3, 5), inv), lambda f: f(q[0, 0], None, pos, inv),
        lambda f: f(q.double(), None, pos, inv), lambda f: f(q, None, pos[None, None], inv),
    ]
    for call in bad:
        for f in (gw.rotary, gw.rotary_):
            with pytest.raises(SvdqB200Error):
                call(f)
    inplace = [
        (q.transpose(2, 3).contiguous().transpose(2, 3), None), (q[:, :, :1].expand(2, 5, 3, 64), None),
        (q, q), (q[:, :, :3], q[:, :, 2:]), (q.clone().requires_grad_(True), None),
        (q, q.view(2, 5, 2, 128)[..., :64]),
    ]
    for a, b in inplace:
        with pytest.raises(SvdqB200Error):
            gw.rotary_(a, b, pos, inv)


def test_frequencies():
    """The formulas of each scaling, and refusals, on the CPU."""
    import gen_worker_b200 as gw
    from gen_worker_b200.ops import SvdqB200Error

    inv, axis, scale = gw.rotary_frequencies(64)
    want = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert axis is None and scale == 1.0 and torch.allclose(inv, want, rtol=1e-14)
    lin, _, _ = gw.rotary_frequencies(64, scaling="linear", factor=4)
    assert torch.allclose(lin, want / 4, rtol=1e-14)
    ntk, _, _ = gw.rotary_frequencies(64, scaling="ntk", factor=4)
    assert math.isclose(ntk[0], 1.0) and math.isclose(ntk[-1], want[-1] / 4, rel_tol=1e-12)
    parts, _, scale = gw.rotary_frequencies(64, scaling="by_parts", factor=4, trained_length=2048)
    turns = 2048 * want / (2 * math.pi)
    assert math.isclose(scale, 0.1 * math.log(4) + 1)
    assert torch.equal(parts[turns >= 32], inv[turns >= 32])
    assert torch.allclose(parts[turns <= 1], want[turns <= 1] / 4, rtol=1e-14)
    assert ((parts <= inv) & (parts >= inv / 4)).all()
    inv, axis, _ = gw.rotary_frequencies(128, axes=(16, 56, 56))
    assert axis.tolist() == [0] * 8 + [1] * 28 + [2] * 28
    assert math.isclose(inv[8], 1.0) and math.isclose(inv[9], 10000.0 ** (-2 / 56))
    for kw in ({"scaling": "best"}, {"axes": (16, 16)}, {"axes": (63, 1)}, {"scaling": "by_parts"},
               {"scaling": "linear", "factor": 0.5},
               {"scaling": "by_parts", "trained_length": 9, "fast_turns": 1.0}):
        with pytest.raises(SvdqB200Error):
            gw.rotary_frequencies(64, **kw)
    for dim in (0, 7, -2):
        with pytest.raises(SvdqB200Error):
            gw.rotary_frequencies(dim)


def test_module_keeps_its_frequencies_in_64_bits():
    import gen_worker_b200 as gw

    rope = gw.RotaryEmbedding(64, axes=(32, 32))
    before = rope.inv_freq.clone()
    rope.half().to(torch.bfloat16)
    assert rope.inv_freq.dtype == torch.float64 and torch.equal(rope.inv_freq, before)
    assert rope.axis.dtype == torch.int32


def test_refusals_on_the_cpu():
    import gen_worker_b200 as gw
    from gen_worker_b200 import native
    from gen_worker_b200.ops import SvdqB200Error

    inv, _, _ = gw.rotary_frequencies(8)
    for f in (gw.rotary, gw.rotary_):
        with pytest.raises(SvdqB200Error, match="no CPU path"):
            f(torch.zeros(1, 2, 1, 8), None, torch.arange(2), inv)

    lib = native.lib()

    def call(B=1, S=1, qh=1, n=2, dh=8, axes=1, kind=0, dtype=1):
        return lib.gwb_rotary(None, None, None, None, qh, None, None, None, None, 0, None, kind, None,
                              None, None, axes, B, S, n, dh, 1.0, 0, 0, dtype, None)

    assert call(B=0) == 0 and call(S=0) == 0 and call(qh=0) == 0
    for kw in ({"B": -1}, {"n": 5}, {"dh": 5000}, {"axes": 0}, {"axes": 65}, {"kind": 3},
               {"dtype": 4}, {"B": 1 << 20, "S": 1 << 20}, {"qh": 1 << 21}, {}):
        assert call(**kw) == 1, kw
