"""How exact the gated feed-forward block is, output by output, against float64.

A result v + d of a computation that is d off, rounded to the type, is at most |round(v) - v| + 2 |d| from v: the nearest
value of the type to v + d is no farther from it than the nearest one to v is.  So in the 2-norm

    |got - v| <= |round(v) - v| + 2 |d|.

d, relative to the size of v (the same sums over the terms' magnitudes, at most twice the value's own norm where there are
64 values and more): 4e-6 for fp32 sums; where h, dg and du go on in two 16-bit parts, two roundings of them, u^2 with
u = finfo(T).eps / 2.  Rounded once they would be off by u, as much as the result's own rounding."""

import pytest
import torch
import torch.nn.functional as F

import neuraloperator_b200 as nb

NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")
HALVES = [torch.bfloat16, torch.float16]


def make(shape, dtype, seed, scale=1.0, device="cuda"):
    g = torch.Generator(device).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * scale).to(dtype)


def operands(batch, c, h, o, grid, dtype, seed=0, device="cuda"):
    to = dict(device=device)
    return [make((batch, c, *grid), dtype, seed, **to), make((h, c), dtype, seed + 1, c ** -0.5, **to),
            make((h, c), dtype, seed + 2, c ** -0.5, **to), make((o, h), dtype, seed + 3, h ** -0.5, **to),
            *[make((n,), dtype, seed + 4 + i, 0.3, **to) for i, n in enumerate((h, h, o))]]


def define(ops, gy, act, keep=lambda t: t):
    """y and the gradients with their sizes, in float64, by the formulas; `keep`: what h, dg and du go through on their way
    into the products."""
    x, wg, wu, wd, bg, bu, bd = [t.double() for t in ops]
    rows, e = x.movedim(1, -1).reshape(-1, x.shape[1]), gy.double().movedim(1, -1).reshape(-1, wd.shape[0])
    g, u = F.linear(rows, wg, bg).requires_grad_(), F.linear(rows, wu, bu)
    a = (F.silu if act == "silu" else F.gelu)(g)
    (slope,) = torch.autograd.grad(a.sum(), g)
    a, f = a.detach(), e @ wd
    h, dg, du = keep(a * u), keep(f * u * slope), keep(f * a)
    back = lambda t: t.reshape(x.shape[0], *x.shape[2:], -1).movedim(-1, 1)  # noqa: E731
    values = [back(h @ wd.t() + bd), back(dg @ wg + du @ wu), dg.t() @ rows, du.t() @ rows, e.t() @ h, dg.sum(0), du.sum(0),
              e.sum(0)]
    m = [t.abs() for t in (rows, e, h, dg, du, wg, wu, wd, bd)]
    rows, e, h, dg, du, wg, wu, wd, bd = m
    sizes = [back(h @ wd.t() + bd), back(dg @ wg + du @ wu), dg.t() @ rows, du.t() @ rows, e.t() @ h, dg.sum(0), du.sum(0),
             e.sum(0)]
    return values, sizes


def allowed(want, size, dtype):
    scale = float(size.norm())
    if want.numel() >= 64:
        scale = min(scale, 2 * float(want.norm()))
    own = float((want.to(dtype).double() - want).norm())
    u = torch.finfo(dtype).eps / 2
    return own + 2 * scale * (4e-6 + (u * u if dtype != torch.float32 else 0.0))


def check(ops, act, seed=99):
    dtype = ops[1].dtype
    leaves = [t.clone().requires_grad_() for t in ops]
    y = nb.gated_mlp(*leaves, activation=act)
    gy = make(y.shape, dtype, seed)
    got = [y, *torch.autograd.grad(y, leaves, gy)]
    with torch.no_grad():
        for name, a, b, size in zip(("y",) + NAMES, got, *define_detached(ops, gy, act)):
            err = float((a.double() - b).norm())
            assert err <= allowed(b, size, dtype), (name, err / float(b.norm()), allowed(b, size, dtype) / float(b.norm()))
    assert nb._lib.device_status() == 0


def define_detached(ops, gy, act):
    with torch.enable_grad():
        values, sizes = define(ops, gy, act)
    return [t.detach() for t in values], [t.detach() for t in sizes]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("batch, c, h, o, grid", [
    (1, 32, 48, 32, (30, 40)),          # few points
    (2, 40, 72, 24, (128, 200)),        # samples of whole tiles, above 2^15 points
    (3, 33, 65, 17, (131, 97)),         # odd rows, above 2^15 points
    (1, 130, 150, 129, (50000,)),       # several tiles of rows and of columns, aligned rows
])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_results_are_rounded_once(batch, c, h, o, grid, dtype, act):
    check(operands(batch, c, h, o, grid, dtype, seed=7), act)


@pytest.mark.gpu
def test_small_gradients_of_half_precision():
    """dL/dy of 2^-20: dg and du have few bits in fp16, or none, and their sums over the points have all of theirs."""
    ops = operands(1, 24, 40, 24, (40000,), torch.float16, seed=3)
    leaves = [t.clone().requires_grad_() for t in ops]
    gy = make((1, 24, 40000), torch.float32, 9).sign().mul(2.0 ** -20).to(torch.float16)
    grads = torch.autograd.grad(nb.gated_mlp(*leaves), leaves[1:], gy)
    for name, a, b, size in zip(NAMES[1:], grads, *[v[2:] for v in define_detached(ops, gy, "silu")]):
        floor = 2.0 ** -25 * b.numel() ** 0.5  # half a step of the smallest values of the result
        assert float((a.double() - b).norm()) <= allowed(b, size, torch.float16) + floor, name


@pytest.mark.parametrize("dtype", HALVES)
def test_the_bound_notices_one_rounding(dtype):
    """In the formulas alone: h, dg and du rounded once are outside the bound, in two parts they are inside."""
    ops = operands(1, 24, 40, 24, (3000,), dtype, device="cpu")
    gy = make((1, 24, 3000), dtype, 5, device="cpu")
    once = lambda t: t.to(dtype).double()  # noqa: E731
    twice = lambda t: once(t) + once(t - once(t))  # noqa: E731
    want, sizes = define(ops, gy, "silu")
    for keep, inside in ((once, False), (twice, True)):
        got, _ = define(ops, gy, "silu", keep)
        # y, dL/dx and the matrices' gradients; the biases' have fewer than 64 values here, where the bound counts the terms'
        # magnitudes, and the last one takes none of the three
        for k in range(5):
            a, b = got[k].detach(), want[k].detach()
            err = float((a.to(dtype).double() - b).norm())
            assert (err <= allowed(b, sizes[k].detach(), dtype)) == inside, k


@pytest.mark.gpu
@pytest.mark.parametrize("h", [300, 513, 4096, 16384])
@pytest.mark.parametrize("c, o", [(32, 32), (20, 150), (150, 20)])
def test_wide_hidden_layers(h, c, o):
    """fp32 sums over the hidden layer do not drift with its width.  Every add to a tensor-core accumulator truncates it by
    at most 2^-25: 6 C / 16 adds of the first product in each of g, u and f, 32 of a part of the second one, and one fp32
    rounding for each part that joins them."""
    ops = operands(1, c, h, o, (300,), torch.float32, seed=11)
    leaves = [t.clone().requires_grad_() for t in ops]
    y = nb.gated_mlp(*leaves)
    gy = make(y.shape, torch.float32, 12)
    got = [y, *torch.autograd.grad(y, leaves, gy)]
    adds = 3 * 6 * max(c, o) / 16 + 32 + 2 * h / 256
    for name, a, b, size in zip(("y", "x"), got, *define_detached(ops, gy, "silu")):
        scale = min(float(size.norm()), 2 * float(b.norm()))
        # the activation's own error (1.5e-7 and its special functions, 2^-22) on the way
        assert float((a.detach().double() - b).norm()) <= scale * (adds * 2.0 ** -25 + 6e-7), name
    check(ops, "gelu")


def values_and_slopes(gates, act):
    """act(g) and act'(g) of every gate, each in a hidden channel of its own: x = 1, up = 1, the outputs one hidden channel
    each (256 a call), and the gradient of the gate's bias."""
    acts, slopes = [], []
    for part in gates.split(256):
        h = part.numel()
        bias = torch.zeros(h, device="cuda", requires_grad=True)
        ones = torch.ones(h, 1, device="cuda")
        y = nb.gated_mlp(torch.ones(1, 1, 1, device="cuda"), part[:, None], ones, torch.eye(h, device="cuda"), bias,
                         activation=act)
        slopes.append(torch.autograd.grad(y, bias, torch.ones_like(y))[0])
        acts.append(y.detach()[0, :, 0])
    return torch.cat(acts).double(), torch.cat(slopes).double()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("gate", [None, 50.0, 200.0, 1e3, 1e4, -50.0, -1e4])
def test_slope_of_every_gate(gate, act):
    """Elementwise; hidden channels go through the activation in pairs, so a saturated gate stands beside a small one."""
    g = (torch.rand(4096, generator=torch.Generator("cuda").manual_seed(2), device="cuda") - 0.5) * 24
    if gate is not None:
        g[0::2] = gate
    ref = g.double().requires_grad_()
    want = (F.silu if act == "silu" else F.gelu)(ref)
    (slope,) = torch.autograd.grad(want.sum(), ref)
    a, s = values_and_slopes(g, act)
    # exponential and reciprocal: some 2^-22 of a slope of at most 1.13; the normal distribution's approximation: 1.5e-7
    assert float((s - slope).abs().max()) <= 1.5e-6
    assert float(((a - want.detach()).abs() / (1 + g.abs())).max()) <= 1.5e-6


def check_huge(gate, act):
    """Hidden channels of a huge gate and of small ones in turn, each with an output of its own."""
    g = (torch.rand(256, generator=torch.Generator("cuda").manual_seed(3), device="cuda") - 0.5) * 12
    g[0::2] = gate
    ref = g.double().requires_grad_()
    want = (F.silu if act == "silu" else F.gelu)(ref)
    (slope,) = torch.autograd.grad(want.sum(), ref)
    a, s = values_and_slopes(g, act)
    assert float((a[1::2] - want[1::2].detach()).abs().max()) <= 1.5e-6 * 7
    assert float((s - slope).abs().max()) <= 1.5e-6
    if gate > 0:
        assert float((a[0::2] / gate - 1).abs().max()) <= 1e-6
    else:
        assert float(a[0::2].abs().max()) <= 1e-15


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [-1e4, -1e20, torch.finfo(torch.float32).min / 2])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_far_below_zero_are_shut(gate, act):
    """However far below zero, as a bias that switches hidden channels off would have it."""
    check_huge(gate, act)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [1e20, 3e38, -3e38])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_huge_gates_leave_their_neighbours(gate, act):
    """Gates whose products overflow fp32 share a reciprocal with small ones."""
    check_huge(gate, act)


# 148 tiles of a slab at a hidden width of 2400; 3996 tiles (fp32 scratch) and 4588 (two bf16 parts) at 64 with 64 channels
# in all: the last slab has fewer pieces than the points' splits
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", ["wide odd", "wide whole", "long odd", "long whole"])
def test_several_slabs(shape, dtype):
    """The backward's scratch is made and consumed slab by slab: sums that go on over two of them, the last one short, with
    the fields copied to the scratch (odd rows) and read in place (samples of whole tiles, one of them across the slabs)."""
    tiles = 4588 if dtype == torch.bfloat16 else 3996
    batch, c, h, o, grid = {"wide odd": (2, 20, 2400, 12, (12501,)), "wide whole": (2, 20, 2400, 12, (98, 128)),
                            "long odd": (1, 32, 64, 32, (tiles * 128 + 597,)),
                            "long whole": (2, 32, 64, 32, ((tiles + 6) // 2, 128))}[shape]
    check(operands(batch, c, h, o, grid, dtype, seed=21), "silu")
