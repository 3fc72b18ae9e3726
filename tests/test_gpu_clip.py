"""Global norm and clipping against 64 bits.  A thread adds at most 32 squares in fp32 (33 roundings of 2^-24, all
terms positive) before 64-bit sums; the factor adds a few, and each result is rounded once to its type."""

import math

import pytest
import torch

import neuraloperator_b200 as nb

pytestmark = pytest.mark.gpu

V = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.complex64]
SIZES = [(1,), (3,), (7, 5), (64, 1), (8192,), (8193,), (4, 4099), (300, 301), (0,), (2, 3, 5, 7)]


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    if dtype == torch.complex64:
        return torch.view_as_complex(torch.randn(*shape, 2, generator=g, device="cuda") * scale)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def tensors(dtype, seed=0):
    return [make(s, dtype, seed + i, 10.0 ** (i % 4 - 2)) for i, s in enumerate(SIZES)]


def norm64(ts):
    return math.sqrt(sum(float(t.abs().double().square().sum()) if not t.is_complex() else
                         float(torch.view_as_real(t).double().square().sum()) for t in ts))


def check_scaled(got, src, factor):
    for a, b in zip(got, src):
        assert a.dtype == b.dtype and a.shape == b.shape
        u = torch.finfo(b.dtype).eps / 2
        a, b = (torch.view_as_real(t).double() if t.is_complex() else t.double() for t in (a, b))
        bound = (b * factor).abs() * (u + 24 * V) + torch.finfo(got[0].dtype).smallest_normal
        assert ((a - b * factor).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_clip_by_global_norm(dtype, share):
    ts = tensors(dtype)
    kept = [t.clone() for t in ts]
    n = norm64(ts)
    out, norm = nb.clip_by_global_norm(ts, n * share)
    assert norm.dtype == torch.float32 and abs(float(norm) - n) <= n * 20 * V
    assert abs(float(nb.global_norm(ts)) - n) <= n * 20 * V
    if share > 1:
        assert all(torch.equal(a, b) for a, b in zip(out, ts))
    check_scaled(out, ts, min(1.0, share))
    assert all(torch.equal(a, b) for a, b in zip(ts, kept))


def test_mixed_types_and_largest_magnitude():
    ts = [t for dtype in TYPES for t in tensors(dtype, 50)]
    n = norm64(ts)
    out, norm = nb.clip_by_global_norm(ts, n / 3)
    assert abs(float(norm) - n) <= n * 20 * V
    for a, b in zip(out, ts):
        check_scaled([a], [b], 1 / 3)
    most = max(float((torch.view_as_real(t) if t.is_complex() else t).abs().max()) for t in ts if t.numel())
    out, norm = nb.clip_by_global_norm(ts, most / 2, norm_type=math.inf)
    assert float(norm) == most
    for a, b in zip(out, ts):
        check_scaled([a], [b], 0.5)


def test_many_tensors_and_large_ones():
    """More tensors than one launch's table takes, and chunks beyond one wave."""
    ts = [make((1 + i % 37,), torch.float32, i) for i in range(700)] + [make((3, 1 << 22), torch.float32, 9, 1e-3)]
    n = norm64(ts)
    out, norm = nb.clip_by_global_norm(ts, n / 2)
    assert abs(float(norm) - n) <= n * 20 * V
    check_scaled(out, ts, 0.5)


def test_sums_do_not_depend_on_scheduling():
    ts = [make((1 << 20,), torch.float32, i) for i in range(5)]
    first, norm = nb.clip_by_global_norm(ts, 1.0)
    for _ in range(3):
        again, n2 = nb.clip_by_global_norm(ts, 1.0)
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(first, again))


def test_unaligned_and_strided():
    buf = make((4097,), torch.float32, 1)
    ts = [buf[1:], make((40, 30), torch.float32, 2).t(), make((64, 64), torch.bfloat16, 3)[:, 1:33],
          make((65,), torch.bfloat16, 4)[1:], make((9, 4), torch.complex64, 5).conj()]
    n = norm64([t.resolve_conj() for t in ts])
    out, norm = nb.clip_by_global_norm(ts, n / 4)
    assert abs(float(norm) - n) <= n * 20 * V
    for a, b in zip(out, ts):
        check_scaled([a], [b.resolve_conj()], 0.25)


def test_clip_grad_norm_in_place():
    ps = [torch.nn.Parameter(make(s, torch.float32, i)) for i, s in enumerate(SIZES)]
    ps.append(torch.nn.Parameter(make((5, 4), torch.complex64, 20)))
    ps.append(torch.nn.Parameter(make((30, 20), torch.float32, 21).t()))
    ps.append(torch.nn.Parameter(make((3,), torch.float32, 22)))  # without a gradient
    for i, p in enumerate(ps[:-1]):
        p.grad = make(tuple(p.shape), p.dtype, 100 + i, 3.0)
    ps[-2].grad = make((20, 30), torch.float32, 40).t().contiguous().t()
    ps[2].grad = torch.as_strided(make((35 * 3,), torch.float32, 41), (7, 5), (15, 3))
    before = [p.grad.clone() for p in ps[:-1]]
    held = [p.grad for p in ps[:-1]]
    n = norm64(before)
    norm = nb.clip_grad_norm_(ps + [ps[3]], n / 2)  # a parameter listed twice counts once
    assert abs(float(norm) - n) <= n * 20 * V
    for h, p, b in zip(held, ps, before):
        assert h is p.grad
        check_scaled([p.grad], [b], 0.5)
    assert ps[-1].grad is None
    again = [p.grad.clone() for p in ps[:-1]]
    nb.clip_grad_norm_(ps, n)  # below the limit: nothing changes
    assert all(torch.equal(p.grad, a) for p, a in zip(ps, again))
    got = nb.clip_grad_norm_(ps[0], 1e9, norm_type=math.inf)
    assert float(got) == float(ps[0].grad.abs().max())


def test_non_finite():
    for bad, seen in ((float("nan"), math.isnan), (float("inf"), math.isinf)):
        p = torch.nn.Parameter(make((100,), torch.float32, 1))
        p.grad = make((100,), torch.float32, 2)
        p.grad[50] = bad
        kept = p.grad.clone()
        with pytest.raises(RuntimeError, match="cannot be clipped"):
            nb.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        assert torch.equal(torch.nan_to_num(p.grad), torch.nan_to_num(kept))
        for kind in (2.0, math.inf):
            out, norm = nb.clip_by_global_norm([p.grad], 1.0, norm_type=kind)
            assert seen(float(norm))
            assert torch.isnan(out[0]).all() if math.isnan(bad) else (torch.isnan(out[0][50]) and (out[0][:50] == 0).all())


def test_empty():
    assert float(nb.clip_grad_norm_([], 1.0)) == 0
    assert nb.clip_by_global_norm([], 1.0)[0] == []
    out, norm = nb.clip_by_global_norm([torch.empty(0, device="cuda")], 1.0)
    assert float(norm) == 0 and out[0].numel() == 0


def test_captured_and_replayed():
    ts = [make((5000,), torch.float32, 1), make((33, 9), torch.complex64, 2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        nb.clip_by_global_norm(ts, 1.0)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, norm = nb.clip_by_global_norm(ts, 1.0)
    for seed in (7, 8):
        ts[0].copy_(make((5000,), torch.float32, seed))
        graph.replay()
        want, n = nb.clip_by_global_norm(ts, 1.0)
        assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_training_step_of_a_model():
    """FNO: backward, clip, step; the clipped gradients are the unclipped ones scaled."""
    torch.manual_seed(0)
    model = nb.FNO(n_modes=(8, 8), in_channels=1, out_channels=1, hidden_channels=8, n_layers=2).cuda()
    x = torch.randn(2, 1, 16, 16, device="cuda")
    model(x).square().mean().backward()
    before = [p.grad.clone() for p in model.parameters()]
    n = norm64(before)
    norm = nb.clip_grad_norm_(model.parameters(), n / 10)
    assert abs(float(norm) - n) <= n * 20 * V
    for p, b in zip(model.parameters(), before):
        check_scaled([p.grad], [b], 0.1)


def test_lazy_views_and_inference_tensors():
    z = make((9, 4), torch.complex64, 5)
    neg = torch._neg_view(make((50,), torch.float32, 6))  # contiguous, its sign only noted
    n = norm64([z, neg])
    out, _ = nb.clip_by_global_norm([z.conj(), neg], n / 2)
    check_scaled([out[0]], [z.conj().resolve_conj()], 0.5)
    check_scaled([out[1]], [neg.resolve_neg()], 0.5)
    with torch.inference_mode():
        p = torch.nn.Parameter(make((100,), torch.float32, 1), requires_grad=False)
        p.grad = make((100,), torch.float32, 2)
        kept = p.grad.clone()
        nb.clip_grad_norm_(p, float(kept.norm()) / 2)
        check_scaled([p.grad], [kept], 0.5)
