"""The gated feed-forward block against its definition in 64 bits: types, channel and hidden widths around every
tile, chunk and padding edge, grids whose rows are odd or unaligned, resident and streamed weights.

Tolerances are in the 2-norm of each output, relative to its size: the same sums over the terms' magnitudes (`sizes`).
With u = finfo(T).eps / 2, a 16-bit type rounds h (backward: dg, du, h) once, by u of each term, and the result once
more, by u of a value no larger than its size: 2 u.  Its fp32 sums, and all of an fp32 call (operands exact to 2^-26,
the activation to 1.5e-7, sums in fp32 whose errors do not add up in one direction), are held to 2e-6.  For outputs of
64 values and more twice the value's own norm bounds the size: sums of random terms are smaller than their
magnitudes' sums, and so are the random errors."""

import math

import pytest
import torch
import torch.nn.functional as F

import neuraloperator_b200 as nb
from neuraloperator_b200 import _lib

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")


def tolerance(dtype):
    return 2e-6 + (0 if dtype == torch.float32 else 2 * torch.finfo(dtype).eps / 2)


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def operands(batch, c, h, o, grid, dtype, bias=True, seed=0):
    x = make((batch, c, *grid), dtype, seed)
    ws = [make((h, c), dtype, seed + 1, c ** -0.5), make((h, c), dtype, seed + 2, c ** -0.5),
          make((o, h), dtype, seed + 3, h ** -0.5)]
    bs = [make((n,), dtype, seed + 4 + i, 0.3) if bias else None for i, n in enumerate((h, h, o))]
    return [x, *ws, *bs]


def define(x, wg, wu, wd, bg, bu, bd, act):
    rows = x.movedim(1, -1)
    g, u = F.linear(rows, wg, bg), F.linear(rows, wu, bu)
    return F.linear((F.silu if act == "silu" else F.gelu)(g) * u, wd, bd).movedim(-1, 1)


def rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm()) if float(b.norm()) else float(a.norm())


def sizes(x, wg, wu, wd, bg, bu, bd, act, gy):
    """The sizes of y and of the gradients in float64: their sums with every term's magnitude."""
    c, o = x.shape[1], wd.shape[0]
    rows, e = x.movedim(1, -1).reshape(-1, c), gy.movedim(1, -1).reshape(-1, o)
    g, u = (F.linear(rows, wg, bg)).requires_grad_(), F.linear(rows, wu, bu)
    a = (F.silu if act == "silu" else F.gelu)(g)
    (slope,) = torch.autograd.grad(a.sum(), g)
    a, g = a.detach(), g.detach()
    f = e @ wd
    h, dg, du = (a * u).abs(), (f * u).abs() * (slope.abs() + 0.1), (f * a).abs()
    back = lambda t: t.reshape(x.shape[0], *x.shape[2:], -1).movedim(-1, 1)  # noqa: E731
    y = back(h @ wd.abs().t() + (0 if bd is None else bd.abs()))
    gx = back(dg @ wg.abs() + du @ wu.abs())
    return [y, gx, dg.t() @ rows.abs(), du.t() @ rows.abs(), e.abs().t() @ h, dg.sum(0), du.sum(0), e.abs().sum(0)]


def hold(name, got, want, size, dtype):
    err, scale = float((got.double() - want.detach()).norm()), float(size.norm())
    if want.numel() >= 64:
        scale = min(scale, 2 * float(want.norm()))
    assert err <= tolerance(dtype) * scale, (name, err / scale)


def check(ops, act, train=True):
    dtype = ops[1].dtype
    leaves = [None if t is None else t.clone().requires_grad_() for t in ops]
    y = nb.gated_mlp(*leaves, activation=act)
    gy = make(y.shape, dtype, 99)
    ref = [None if t is None else t.double().requires_grad_() for t in ops]
    want = define(*ref, act)
    y_size, *g_sizes = sizes(*[None if t is None else t.detach() for t in ref], act, gy.double())
    assert y.dtype == dtype and y.shape == want.shape
    hold("y", y, want, y_size, dtype)
    with torch.no_grad():
        assert torch.equal(nb.gated_mlp(*ops, activation=act), y)
    if not train:
        return
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], gy)
    exp = torch.autograd.grad(want, [t for t in ref if t is not None], gy.double())
    kept = [(n, z) for n, z, t in zip(NAMES, g_sizes, ops) if t is not None]
    for (name, size), a, b in zip(kept, got, exp):
        assert a.dtype == dtype and a.shape == b.shape
        hold(name, a, b, size, dtype)
    assert _lib.device_status() == 0


# batch, channels, hidden, out, grid
SHAPES = [
    (1, 1, 1, 1, (1,)), (1, 3, 5, 2, (7,)), (2, 16, 16, 16, (64,)), (1, 17, 33, 15, (13, 11)), (1, 32, 16, 32, (16, 16)),
    (3, 32, 64, 32, (9, 5)), (2, 64, 65, 64, (40, 8)), (1, 64, 128, 64, (33, 20)), (2, 33, 96, 48, (10, 13)),
    (1, 128, 200, 128, (50, 4)), (1, 129, 70, 130, (19, 8)), (1, 256, 300, 256, (12, 12)), (1, 96, 1030, 40, (77,)),
    (2, 250, 64, 3, (100,)), (5, 20, 24, 256, (3, 3, 3)), (2, 64, 128, 64, (4, 32, 32)),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_against_definition(shape, dtype, act):
    b, c, h, o, grid = shape
    check(operands(b, c, h, o, grid, dtype), act)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_biases(dtype):
    check(operands(2, 40, 72, 40, (21, 6), dtype, bias=False), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("points", [(60000,), (60001,)])
def test_many_tiles(dtype, points):
    """Several tiles a CTA and several slabs of the backward's scratch; aligned and odd rows."""
    check(operands(2, 32, 64, 32, points, dtype), "silu")
    check(operands(1, 64, 320, 64, points, dtype), "gelu")


def test_gradients_against_differences():
    ops = operands(2, 12, 20, 9, (6, 5), torch.float32, seed=30)
    leaves = [t.clone().requires_grad_() for t in ops]
    y = nb.gated_mlp(*leaves, activation="gelu")
    gy = make(y.shape, torch.float32, 50)
    grads = torch.autograd.grad(y, leaves, gy)
    point = [t.double() for t in ops]
    h = 1e-6
    for k in range(len(point)):
        d = [torch.zeros_like(t) for t in point]
        d[k] = make(point[k].shape, torch.float64, 60 + k)
        f = lambda s: float((define(*[p + s * e for p, e in zip(point, d)], "gelu") * gy.double()).sum())  # noqa: E731
        diff = (f(h) - f(-h)) / (2 * h)
        got = float((grads[k].double() * d[k]).sum())
        size = float((grads[k].double().norm() * d[k].norm()))
        assert abs(got - diff) <= 4e-6 * size, NAMES[k]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 3, 5, 2, (7,)), (2, 33, 96, 48, (10, 13)), (1, 64, 128, 64, (32, 32)),
                                   (1, 200, 300, 120, (50, 4)), (2, 96, 256, 96, (100, 61))])
def test_quantized_field(shape, dtype):
    """The norm's 8-bit output through the block: exact against the values that it stands for."""
    b, c, h, o, grid = shape
    x, *rest = operands(b, c, h, o, grid, dtype)
    w = make((c,), torch.float32, 70)
    with torch.no_grad():
        q, scale = nb.rms_norm_quantized(x, w)
        y = nb.gated_mlp(q, *rest, activation="silu", x_scale=scale)
        rest64 = [None if t is None else t.double() for t in rest]
        assert torch.equal(y, nb.gated_mlp(q, *rest, activation="silu", x_scale=scale))
    for times in (1.0, 4.0):  # the scales count, point by point
        scale2 = scale * times
        scale2[..., 0] *= 2
        x64 = q.double() * scale2.double()
        want = define(x64, *rest64, "silu")
        size = sizes(x64, *rest64, "silu", torch.zeros_like(want))[0]
        with torch.no_grad():
            y = nb.gated_mlp(q, *rest, activation="silu", x_scale=scale2)
        hold("y", y, want, size, dtype)


def test_range_of_values():
    """fp32 accuracy over the exponents: the parts of a split keep the value's range."""
    for scale in (1e-12, 1e-4, 1e4):
        ops = operands(1, 24, 40, 24, (300,), torch.float32, bias=False)
        ops[0] = ops[0] * scale
        ops[3] = ops[3] / scale
        check(ops, "silu")
    for big in (30.0, 200.0):  # saturated gates
        ops = operands(1, 24, 40, 24, (300,), torch.float32)
        ops[1] = ops[1] * big
        check(ops, "silu")
        check(ops, "gelu")


def test_points_do_not_mix():
    """A point that is not finite leaves the others as they are."""
    for dtype in TYPES:
        ops = operands(1, 40, 64, 40, (1000,), dtype)
        want = nb.gated_mlp(*ops)
        ops[0][0, 3, 200] = float("nan")
        ops[0][0, 5, 601] = float("inf")
        got = nb.gated_mlp(*ops)
        keep = torch.ones(1000, dtype=torch.bool, device="cuda")
        keep[[200, 601]] = False
        assert torch.equal(got[..., keep], want[..., keep])
        assert not torch.isfinite(got[..., [200, 601]]).any()


def test_parts_of_the_gradient():
    """Any subset of the operands; what is not asked for is not computed and nothing else changes."""
    ops = operands(2, 24, 40, 24, (11, 9), torch.float32)
    gy = make((2, 24, 11, 9), torch.float32, 9)
    full = [t.clone().requires_grad_() for t in ops]
    want = torch.autograd.grad(nb.gated_mlp(*full), full, gy)
    for picked in ([0], [3], [1, 5], [6], [0, 4]):
        some = [t.clone().requires_grad_(i in picked) for i, t in enumerate(ops)]
        got = torch.autograd.grad(nb.gated_mlp(*some), [some[i] for i in picked], gy)
        for i, g in zip(picked, got):
            assert torch.equal(g, want[i]), NAMES[i]


def test_repeats_are_equal():
    ops = [t.requires_grad_() for t in operands(2, 64, 128, 64, (70, 90), torch.float32)]
    gy = make((2, 64, 70, 90), torch.float32, 9)
    first = torch.autograd.grad(nb.gated_mlp(*ops), ops, gy)
    for _ in range(3):
        for a, b in zip(first, torch.autograd.grad(nb.gated_mlp(*ops), ops, gy)):
            assert torch.equal(a, b)


def test_empty_views_and_streams():
    ops = operands(2, 16, 24, 8, (10, 12), torch.float32)
    for shape in ((0, 16, 5), (2, 16, 0)):
        some = [torch.empty(shape, device="cuda"), *ops[1:]]
        some = [t.clone().requires_grad_() for t in some]
        y = nb.gated_mlp(*some)
        assert y.shape == (shape[0], 8, shape[2])
        for g in torch.autograd.grad(y, some[1:], torch.empty_like(y)):
            assert (g == 0).all()
    want = nb.gated_mlp(*ops)
    x, rest = ops[0], ops[1:]
    assert torch.equal(nb.gated_mlp(x.to(memory_format=torch.channels_last), *rest), want)
    assert torch.equal(nb.gated_mlp(x.transpose(2, 3), *rest), want.transpose(2, 3))
    buf = torch.empty(x.numel() + 1, device="cuda")
    odd = buf[1:].view(x.shape)
    odd.copy_(x)
    assert torch.equal(nb.gated_mlp(odd, *rest), want)
    wide = torch.empty(24, 40, device="cuda")
    wide[:, 5:21] = ops[1]
    assert torch.equal(nb.gated_mlp(x, wide[:, 5:21], *ops[2:]), want)
    assert torch.equal(nb.gated_mlp(x, ops[1][..., None], ops[2][..., None], ops[3][..., None], *ops[4:]), want)
    two = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in two:  # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(nb.gated_mlp(*ops))
    for s in two:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want) for o in outs)


def test_captured_and_replayed():
    ops = [t.requires_grad_() for t in operands(2, 32, 64, 32, (30, 31), torch.float32)]
    gy = make((2, 32, 30, 31), torch.float32, 9)

    def step():
        y = nb.gated_mlp(*ops)
        return [y, *torch.autograd.grad(y, ops, gy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (5, 6):
        with torch.no_grad():
            ops[0].copy_(make(ops[0].shape, torch.float32, seed))
        for g in graphs:
            g.replay()
        kept = [[t.clone() for t in o] for o in outs]
        for a, b, c in zip(kept[0], kept[1], step()):
            assert torch.equal(a, c) and torch.equal(b, c)


def test_norm_block_and_clipping_together():
    """A pre-norm feed-forward step as a model makes it: the norm of x + skip, the block, the sum, the clipped
    gradients of all parameters."""
    c, h = 24, 40
    x, skip = make((2, c, 17, 9), torch.float32, 1), make((2, c, 17, 9), torch.float32, 2)
    params = [make((c,), torch.float32, 3)] + operands(1, c, h, c, (1,), torch.float32, seed=4)[1:]
    ours = [torch.nn.Parameter(p.clone()) for p in params]
    y, r = nb.rms_norm(x, ours[0], residual=skip)
    out = r + nb.gated_mlp(y, *ours[1:])
    out.square().mean().backward()
    norm = nb.clip_grad_norm_(ours, 0.01)
    ref = [p.double().requires_grad_() for p in params]
    r64 = x.double() + skip.double()
    y64 = r64 / torch.sqrt((r64 * r64).mean(1, keepdim=True) + 1e-6) * ref[0].view(1, -1, 1, 1)
    grads = torch.autograd.grad((r64 + define(y64, *ref[1:], "silu")).square().mean(), ref)
    n = math.sqrt(sum(float(g.square().sum()) for g in grads))
    assert abs(float(norm) - n) <= 4e-6 * n
    for p, g in zip(ours, grads):
        assert rel(p.grad, g * 0.01 / n) <= 4e-6


def test_offsets_past_32_bits():
    """A field of 2.2e9 values: its last points, forward, backward and both kinds of rows, equal those of a small one."""
    c, h, o = 256, 20, 3
    rest = operands(1, c, h, o, (1,), torch.bfloat16, seed=3)[1:]
    for p in (4_300_000, 4_300_001):
        x = torch.zeros(2, c, p, device="cuda", dtype=torch.bfloat16)
        gy = torch.zeros(2, o, p, device="cuda", dtype=torch.bfloat16)
        n = 2 * p % 128 + 128   # the last tiles, whole: a small field of them has the same tiles
        x[1, :, p - n:], gy[1, :, p - n:] = make((c, n), torch.bfloat16, 1), make((o, n), torch.bfloat16, 2)
        x.requires_grad_()
        y = nb.gated_mlp(x, *rest)
        (gx,) = torch.autograd.grad(y, x, gy)
        xs = x.detach()[1:, :, p - n:].clone().requires_grad_()
        ys = nb.gated_mlp(xs, *rest)
        (gs,) = torch.autograd.grad(ys, xs, gy[1:, :, p - n:].contiguous())
        assert torch.equal(y[1:, :, p - n:], ys) and torch.equal(gx[1:, :, p - n:], gs)
        assert (gx[:, :, : p - n] == 0).all()
        assert _lib.device_status() == 0
        del x, y, gx


@pytest.mark.parametrize("dtype", TYPES)
def test_samples_of_whole_tiles(dtype):
    """Samples of whole tiles, more points than the fp32 scratch of 16-bit fields takes: the fields are contracted in
    place, over several samples; and the last size that takes that scratch, and the first that does not."""
    check(operands(3, 48, 72, 40, (160, 128), dtype), "gelu")
    check(operands(1, 20, 24, 20, (1 << 15,), dtype), "silu")
    check(operands(1, 20, 24, 20, ((1 << 15) + 1,), dtype), "silu")
