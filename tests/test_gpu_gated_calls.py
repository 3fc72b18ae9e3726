"""The gated block's operands as callers may have them."""

import pytest
import torch

import neuraloperator_b200 as nb

pytestmark = pytest.mark.gpu


def operands(dtype=torch.float32, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    shapes = ((2, 12, 30), (20, 12), (20, 12), (9, 20), (20,), (20,), (9,))
    return [torch.randn(s, generator=g, device="cuda").to(dtype) for s in shapes]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lazily_negated_tensors(dtype):
    """Held with the other sign and a mark, as z.conj().imag is: contiguous, and not the values that memory holds."""
    negated = lambda t: torch._neg_view(-t)  # noqa: E731
    ops = operands(dtype)
    assert negated(ops[0]).is_neg() and negated(ops[0]).is_contiguous()
    gy = torch.randn(2, 9, 30, device="cuda").to(dtype)
    both = []
    for mark in (negated, lambda t: t.clone()):
        leaves = [mark(t).requires_grad_() for t in ops]
        y = nb.gated_mlp(*leaves)
        both.append([y, *torch.autograd.grad(y, leaves, mark(gy))])
        with torch.no_grad():
            both[-1].append(nb.gated_mlp(*[mark(t) for t in ops], activation="gelu"))
    for a, b in zip(*both):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_frozen_weights_take_no_scratch(dtype):
    """dL/dx alone: the same values as with all gradients, in a workspace of the weights' size."""
    g = torch.Generator("cuda").manual_seed(0)
    ops = [torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((2, 12, 60000), (20, 12), (20, 12), (9, 20))]
    gy = torch.randn(2, 9, 60000, generator=g, device="cuda").to(dtype)
    leaves = [t.clone().requires_grad_() for t in ops]
    want = torch.autograd.grad(nb.gated_mlp(*leaves), leaves, gy)[0]
    x = ops[0].requires_grad_()
    y = nb.gated_mlp(x, *ops[1:])
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    (gx,) = torch.autograd.grad(y, x, gy)
    taken = torch.cuda.max_memory_allocated() - before
    assert torch.equal(gx, want)
    assert taken <= gx.numel() * gx.element_size() + (1 << 20)
