"""The per-point norm against its definition in 64 bits: types, channel counts on both sides of every kernel
variant, grids whose rows are odd or unaligned, single points, empty batches, zero and non-finite points.

Tolerances count roundings: u = finfo(T).eps / 2 for the rounding to the output's type, v = 2^-24 for each fp32
operation.  A sum of C squares (all positive) is off by at most C v, its root by half of that."""

import pytest
import torch

import neuraloperator_b200 as nb

pytestmark = pytest.mark.gpu

V = 2.0 ** -24
EPS = 1e-6
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def define(x, w, res, eps=EPS):
    """(y, r, inv) in float64."""
    r = x.double() if res is None else (x.float() + res.float()).to(x.dtype).double()
    inv = 1 / torch.sqrt((r * r).mean(1, keepdim=True) + eps)
    shape = (1, -1) + (1,) * (x.ndim - 2)
    return r * inv * (1.0 if w is None else w.double().view(shape)), r, inv


def y_bound(y, c, dtype):
    return y.abs() * (torch.finfo(dtype).eps / 2 + (c / 2 + 8) * V) + torch.finfo(dtype).smallest_normal


SHAPES = [(1, 1, 1), (2, 3, 5), (1, 32, 16, 16), (3, 8, 7, 9), (2, 9, 64), (1, 64, 33, 8), (2, 65, 12, 4),
          (1, 128, 40), (1, 129, 3, 5, 7), (2, 256, 31), (1, 257, 64), (1, 700, 9), (5, 16), (1, 40, 61, 67)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward(shape, dtype, residual):
    x, w = make(shape, dtype, 1, 2.0), make((shape[1],), torch.float32, 2)
    res = make(shape, dtype, 3) if residual else None
    with torch.no_grad():
        out = nb.rms_norm(x, w, residual=res, eps=EPS)
    y, r = out if residual else (out, x)
    y64, r64, _ = define(x, w, res)
    assert y.dtype == r.dtype == dtype and y.shape == shape
    assert torch.equal(r.double(), r64)
    assert ((y.double() - y64).abs() <= y_bound(y64, shape[1], dtype)).all()


def test_forward_wide_grids():
    """Enough points for every vector width, in all three types."""
    for dtype in TYPES:
        for points in (1 << 16, (1 << 16) + 2, (1 << 16) + 4, (1 << 16) + 1):
            x, w = make((2, 24, points), dtype, 5), make((24,), torch.bfloat16, 6)
            y64, _, _ = define(x, w, None)
            assert ((nb.rms_norm(x, w, eps=EPS).double() - y64).abs() <= y_bound(y64, 24, dtype)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES + [(2, 20, 1 << 15), (1, 72, 1 << 15), (1, 300, 4100)])
@pytest.mark.parametrize("residual", [False, True])
def test_backward(shape, dtype, residual):
    x, w = make(shape, dtype, 1, 1.5).requires_grad_(), make((shape[1],), torch.float32, 2).requires_grad_()
    res = make(shape, dtype, 3).requires_grad_() if residual else None
    gy, gr = make(shape, dtype, 4), make(shape, dtype, 5)
    if residual:
        y, r = nb.rms_norm(x, w, residual=res, eps=EPS)
        gx, gres, gw = torch.autograd.grad([y, r], [x, res, w], [gy, gr])
        assert torch.equal(gx, gres)
    else:
        gx, gw = torch.autograd.grad(nb.rms_norm(x, w, eps=EPS), [x, w], gy)
    c = shape[1]
    dims = [0] + list(range(2, len(shape)))
    with torch.no_grad():
        _, r64, inv = define(x, w, res)
        g, wv = gy.double(), w.double().view((1, -1) + (1,) * (len(shape) - 2))
        hat = r64 * inv
        m, m_abs = (g * wv * hat).mean(1, keepdim=True), (g * wv * hat).abs().mean(1, keepdim=True)
        want = inv * (g * wv - hat * m)
        size = inv * ((g * wv).abs() + hat.abs() * m_abs)
        if residual:
            want, size = want + gr.double(), size + gr.double().abs()
        bound = want.abs() * torch.finfo(dtype).eps / 2 + size * (2 * c + 16) * V + torch.finfo(dtype).smallest_normal
        assert ((gx.double() - want).abs() <= bound).all()
        want, size = (g * hat).sum(dims), (g * hat).abs().sum(dims)
        # a thread adds its own points one by one; 32 lanes x tiles of the grid share them
        points = x.numel() // c
        assert ((gw.double() - want).abs() <= size * (points / 32 + c / 2 + 64) * V).all()


def test_gradients_against_differences():
    """A random direction: the loss's difference quotient in 64 bits equals the gradients' product with it."""
    x, w, res = make((2, 11, 6, 5), torch.float32, 1), make((11,), torch.float32, 2), make((2, 11, 6, 5), torch.float32, 3)
    gy, gr = make(x.shape, torch.float32, 4), make(x.shape, torch.float32, 5)
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    y, r = nb.rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=1e-2)
    grads = torch.autograd.grad([y, r], leaves, [gy, gr])

    def loss(x, w, res):
        r = x + res
        y = r / torch.sqrt((r * r).mean(1, keepdim=True) + 1e-2) * w.view(1, -1, 1, 1)
        return float((y * gy.double()).sum() + (r * gr.double()).sum())

    point = [t.double() for t in (x, w, res)]
    for k in range(3):
        d = [torch.zeros_like(t) for t in point]
        d[k] = make(point[k].shape, torch.float64, 10 + k)
        h = 1e-6
        diff = (loss(*[p + h * e for p, e in zip(point, d)]) - loss(*[p - h * e for p, e in zip(point, d)])) / (2 * h)
        got = float((grads[k].double() * d[k]).sum())
        size = float((grads[k].double() * d[k]).abs().sum())
        # fp32 gradients: some tens of roundings each; the quotient: h^2 and 2^-53 / h of the loss's terms
        assert abs(got - diff) <= size * 64 * V + 1e-6 * size


def test_parts_of_the_gradient():
    """Only the sum, only the norm, only the weight: the others get none."""
    x, res, w = (make(s, torch.float32, i) for i, s in enumerate([(2, 8, 9), (2, 8, 9), (8,)]))
    a, b = x.clone().requires_grad_(), res.clone().requires_grad_()
    y, r = nb.rms_norm(a, w, residual=b)
    g = make(x.shape, torch.float32, 7)
    for t in torch.autograd.grad(r, [a, b], g, retain_graph=True):
        assert torch.equal(t, g)
    full = torch.autograd.grad([y, r], [a], [g, torch.zeros_like(g)], retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, [a], g)[0], full)
    v = w.clone().requires_grad_()
    y = nb.rms_norm(x, v)
    (gw,) = torch.autograd.grad(y, [v], g)
    xx = x.clone().requires_grad_()
    gx, gw2 = torch.autograd.grad(nb.rms_norm(xx, v), [xx, v], g)
    assert torch.equal(gw, gw2)
    assert torch.autograd.grad(nb.rms_norm(xx), [xx], g)[0].shape == x.shape  # no weight at all


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 5, 7), (1, 32, 16, 16), (1, 96, 61, 9), (2, 130, 33), (1, 300, 8),
                                   (2, 24, 1 << 16)])
@pytest.mark.parametrize("residual", [False, True])
def test_quantized(shape, dtype, residual):
    x, w = make(shape, dtype, 1, 3.0), make((shape[1],), torch.float32, 2)
    res = make(shape, dtype, 3) if residual else None
    q, s, *r = nb.rms_norm_quantized(x, w, residual=res, eps=EPS)
    y64, r64, _ = define(x, w, res)
    if residual:
        assert torch.equal(r[0].double(), r64)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32 and s.shape == (shape[0], 1, *shape[2:])
    s64, err = s.double(), (shape[1] / 2 + 8) * V
    assert torch.equal(torch.frexp(s)[0], torch.full_like(s, 0.5))  # powers of two
    most = y64.abs().amax(1, keepdim=True)
    assert (most <= 448 * s64 * (1 + err)).all() and (most >= 224 * s64 * (1 - err)).all()
    # half a step of e4m3: 2^-4 of a normal value, 2^-10 below 2^-6
    bound = torch.maximum(y64.abs() * 2.0 ** -4, 2.0 ** -10 * s64) + 2 * err * y64.abs()
    assert ((q.double() * s64 - y64).abs() <= bound).all()


def test_zero_and_non_finite_points():
    x = make((1, 40, 8), torch.float32, 1)
    x[0, :, 2] = 0
    x[0, 3, 4] = float("nan")
    x[0, 5, 6] = float("inf")
    y = nb.rms_norm(x, eps=EPS)
    clean = [0, 1, 2, 3, 5, 7]
    y64, _, _ = define(x, None, None)
    assert (y[..., 2] == 0).all()
    assert ((y.double() - y64).abs() <= y_bound(y64, 40, torch.float32))[..., clean].all()
    assert torch.isnan(y[..., 4]).all()
    assert torch.isnan(y[0, 5, 6]) and (y[0, :5, 6] == 0).all()  # inf / inf, and finite / inf
    q, s = nb.rms_norm_quantized(x, eps=EPS)
    assert (q[..., 2].float() == 0).all() and s[0, 0, 2] == 1 and s[0, 0, 4] == 1
    assert torch.isnan(q[..., 4].float()).all() and torch.isfinite(q[..., clean].float()).all()
    xg = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(nb.rms_norm(xg, eps=EPS), xg, torch.ones_like(x))
    assert torch.isfinite(gx[..., clean]).all()


def test_empty_views_and_streams():
    w = make((6,), torch.float32)
    for shape in ((0, 6, 5), (2, 6, 0)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        v = w.clone().requires_grad_()
        gx, gw = torch.autograd.grad(nb.rms_norm(x, v), [x, v], torch.empty(shape, device="cuda"))
        assert gx.shape == shape and (gw == 0).all()
        with torch.no_grad():
            assert nb.rms_norm_quantized(x, w)[1].shape == (shape[0], 1, shape[2])
    x = make((2, 12, 10, 14), torch.float32, 1)
    want = nb.rms_norm(x)
    assert torch.equal(nb.rms_norm(x.to(memory_format=torch.channels_last)), want)
    assert torch.equal(nb.rms_norm(x.transpose(2, 3)), want.transpose(2, 3))
    # an offset that leaves no 16-byte alignment
    buf = torch.empty(x.numel() + 1, device="cuda")
    odd = buf[1:].view(x.shape)
    odd.copy_(x)
    assert torch.equal(nb.rms_norm(odd), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = nb.rms_norm(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)


def test_captured_and_replayed():
    """Forward and backward in one CUDA graph, replayed on new values in the same buffers."""
    x, res, w = make((2, 48, 900), torch.float32, 1), make((2, 48, 900), torch.float32, 2), make((48,), torch.float32, 3)
    g = make(x.shape, torch.float32, 4)
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]

    def step():
        y, r = nb.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        return [y, r, *torch.autograd.grad([y, r], leaves, [g, g])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6):
        with torch.no_grad():
            leaves[0].copy_(make(x.shape, torch.float32, seed))
        graph.replay()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """A field of 2.2e9 values: the last points of the last channel, forward and backward."""
    c, p = 32, 70_000_003
    x = torch.zeros(1, c, p, device="cuda", dtype=torch.bfloat16)
    tail = slice(p - 300, p)
    x[..., tail] = make((1, c, 300), torch.bfloat16, 1)
    w = make((c,), torch.float32, 2)
    with torch.no_grad():
        y = nb.rms_norm(x, w, eps=EPS)
    y64, _, inv = define(x[..., tail], w, None)
    assert ((y[..., tail].double() - y64).abs() <= y_bound(y64, c, torch.bfloat16)).all()
    assert (y[..., : p - 300] == 0).all()
    del y
    x.requires_grad_()
    g = torch.zeros_like(x, requires_grad=False)
    g[..., tail] = make((1, c, 300), torch.bfloat16, 3)
    (gx,) = torch.autograd.grad(nb.rms_norm(x, w, eps=EPS), x, g)
    xs = x.detach()[..., tail].clone().requires_grad_()
    (want,) = torch.autograd.grad(nb.rms_norm(xs, w, eps=EPS), xs, g[..., tail].contiguous())
    assert torch.equal(gx[..., tail], want)


def negated(t):
    """The same values as t, held with the other sign and a mark (as z.conj().imag is)."""
    n = torch._neg_view(-t)
    assert n.is_neg() and n.is_contiguous() and torch.equal(n, t)
    return n


@pytest.mark.parametrize("dtype", TYPES)
def test_lazily_negated_tensors(dtype):
    x, res, w = make((2, 12, 30), dtype, 1), make((2, 12, 30), dtype, 2), make((12,), torch.float32, 3)
    gy, gr = make(x.shape, dtype, 4), make(x.shape, dtype, 5)
    with torch.no_grad():
        for a, b in zip(nb.rms_norm(negated(x), negated(w), residual=negated(res)), nb.rms_norm(x, w, residual=res)):
            assert torch.equal(a, b)
        assert torch.equal(nb.rms_norm(x, negated(w.to(torch.bfloat16))), nb.rms_norm(x, w.to(torch.bfloat16)))
        for a, b in zip(nb.rms_norm_quantized(negated(x), negated(w)), nb.rms_norm_quantized(x, w)):
            assert torch.equal(a.float(), b.float())
    both = []
    for mark in (negated, lambda t: t.clone()):
        leaves = [mark(t).requires_grad_() for t in (x, w, res)]
        y, r = nb.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        both.append(torch.autograd.grad([y, r], leaves, [mark(gy), mark(gr)]))
    for a, b in zip(*both):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [24, 72, 128, 160, 256, 300])
@pytest.mark.parametrize("points", [76000, 76004, 76002])  # 8, 4 and 2 values a thread, forward; 4, 4 and 2 backward
def test_wide_rows_of_many_channels(channels, points, dtype):
    """Every channel class at every vector width: y, the sum, the 8-bit output and the gradients, with a residual."""
    shape = (1, channels, points)
    x, w, res = make(shape, dtype, 1, 1.5), make((channels,), torch.float32, 2), make(shape, dtype, 3)
    gy, gr = make(shape, dtype, 4), make(shape, dtype, 5)
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal
    leaves = [t.clone().requires_grad_() for t in (x, res, w)]
    y, r = nb.rms_norm(leaves[0], leaves[2], residual=leaves[1], eps=EPS)
    gx, gres, gw = torch.autograd.grad([y, r], leaves, [gy, gr])
    with torch.no_grad():
        y64, r64, inv = define(x, w, res)
        assert torch.equal(r.double(), r64) and torch.equal(gx, gres)
        assert ((y.double() - y64).abs() <= y_bound(y64, channels, dtype)).all()
        y0, _, _ = define(x, w, None)
        assert ((nb.rms_norm(x, w, eps=EPS).double() - y0).abs() <= y_bound(y0, channels, dtype)).all()
        q, s, r = nb.rms_norm_quantized(x, w, residual=res, eps=EPS)
        assert torch.equal(r.double(), r64)
        # e4m3: half a step of three bits after the first, 2^-10 of the scale below its smallest normal number
        off = (q.double() * s.double() - y64).abs()
        assert (off <= y64.abs() * (2.0 ** -4 + (channels / 2 + 8) * V) + s.double() * 2.0 ** -10).all()
        del q, s, off, y0
        g, wv = gy.double(), w.double().view(1, -1, 1)
        hat = r64 * inv
        m, m_abs = (g * wv * hat).mean(1, keepdim=True), (g * wv * hat).abs().mean(1, keepdim=True)
        want = inv * (g * wv - hat * m) + gr.double()
        size = inv * ((g * wv).abs() + hat.abs() * m_abs) + gr.double().abs()
        assert ((gx.double() - want).abs() <= want.abs() * u + size * (2 * channels + 16) * V + tiny).all()
        want, size = (g * hat).sum([0, 2]), (g * hat).abs().sum([0, 2])
        assert ((gw.double() - want).abs() <= size * (points / 32 + channels / 2 + 64) * V).all()
