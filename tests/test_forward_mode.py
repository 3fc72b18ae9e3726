"""Forward-mode derivatives: the kernels read pointers, so a tangent would be lost without a word; the calls refuse it."""

import pytest
import torch
from torch.autograd import forward_ad

import neuraloperator_b200 as nb
from neuraloperator_b200 import pointwise
from neuraloperator_b200.utils import refuse_tangents


def test_only_tangents_are_refused():
    t = torch.ones(3)
    refuse_tangents(t, None)
    with forward_ad.dual_level():
        refuse_tangents(t, None)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            refuse_tangents(None, t, forward_ad.make_dual(t, t))
    refuse_tangents(t)


@pytest.mark.gpu
def test_calls_refuse_tangents():
    def on(*shape):
        return torch.ones(shape, device="cuda")

    x, w, wg, wd, b = on(2, 4, 8), on(4), on(5, 4), on(3, 5), on(5)
    m1, m2 = on(8, 4), on(4, 8)
    calls = {
        "norm": (lambda x, w: nb.rms_norm(x, w), (x, w)),
        "residual": (lambda x, r: nb.rms_norm(x, residual=r)[0], (x, x.clone())),
        "quantized": (lambda x, w: nb.rms_norm_quantized(x, w)[1], (x, w)),
        "gated": (lambda x, wg, wd, b: nb.gated_mlp(x, wg, wg, wd, b), (x, wg, wd, b)),
        "clip": (lambda a, c: nb.clip_by_global_norm([a, c], 1.0)[1], (x, w)),
        "norm of all": (lambda a, c: nb.global_norm([a, c]), (x, w)),
        "chain": (lambda x, a, c: pointwise.chain(x, a, None, c, None), (x, m1, m2)),
    }
    for name, (call, args) in calls.items():
        call(*args)
        with forward_ad.dual_level():
            call(*args)
            for i, t in enumerate(args):
                some = list(args)
                some[i] = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="forward"):
                    call(*some)
                some = [s.detach().clone().requires_grad_() for s in args]
                some[i] = forward_ad.make_dual(some[i], torch.ones_like(t))
                with pytest.raises(Exception, match="forward|backward"):  # (an 8-bit result has no derivative at all)
                    call(*some)
    p = torch.nn.Parameter(on(3))
    with forward_ad.dual_level():
        p.grad = forward_ad.make_dual(on(3), on(3))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nb.clip_grad_norm_([p], 1.0)
