"""Global norm over all gradients of a model, and clipping by it (nop_clip_by_norm): the step between
``loss.backward()`` and ``optimizer.step()``.

Tensors are float32, bfloat16, float16 or complex64 (the spectral weights; a complex value counts as its real and
imaginary part), on one CUDA device.  No call synchronises with the host, and the sums do not depend on scheduling.  Squares
are float32: a value above 1.8e19 makes the 2-norm infinite, and values below 1e-22 do not count in it.
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable, List, Sequence, Tuple, Union

import torch

from . import _lib
from .utils import refuse_tangents

_DTYPES = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16,
           torch.complex64: _lib.DTYPE_FP32}
_NORMS = {2.0: _lib.NORM_L2, math.inf: _lib.NORM_INF}


def _norm_kind(norm_type: Union[float, str]) -> int:
    kind = _NORMS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return kind


def _limit(max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number >= 0, got {max_norm}")
    return max_norm


def _check(tensors: Sequence[torch.Tensor]) -> torch.device:
    devices = {t.device for t in tensors}
    if any(d.type != "cuda" for d in devices):
        raise RuntimeError("neuraloperator_b200 runs on CUDA devices only (there is no CPU path)")
    for dtype in {t.dtype for t in tensors}:
        if dtype not in _DTYPES:
            raise TypeError(f"expected float32, bfloat16, float16 or complex64 tensors, got {dtype}")
    if len(devices) > 1:
        raise ValueError("all tensors must be on one device")
    refuse_tangents(*tensors)
    return devices.pop()


def _run(src: List[torch.Tensor], dst, max_norm: float, kind: int, dev: torch.device) -> torch.Tensor:
    """The norm (a float32 scalar) of the contiguous tensors ``src``; their scaled values go to ``dst`` if given."""
    n = len(src)
    lib = _lib.library()
    size = ctypes.c_size_t()
    _lib.check(lib.nop_clip_workspace_size(n, size))
    norm = torch.empty((), device=dev, dtype=torch.float32)
    ws = torch.empty(size.value, device=dev, dtype=torch.uint8)
    pointers = ctypes.c_void_p * n
    a = pointers(*[t.data_ptr() for t in src])
    b = a if dst is src else None if dst is None else pointers(*[t.data_ptr() for t in dst])
    kinds = [t.dtype for t in src]
    numel = (ctypes.c_int64 * n)(*[2 * t.numel() if k is torch.complex64 else t.numel() for t, k in zip(src, kinds)])
    dtypes = (ctypes.c_int32 * n)(*[_DTYPES[k] for k in kinds])
    _lib.call(lib.nop_clip_by_norm, dev, n, a, b, numel, dtypes, kind, max_norm, norm.data_ptr(), ws.data_ptr(),
              size.value)
    return norm


@torch.no_grad()
def global_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all tensors' values together, a float32 scalar on their device.  norm_type: 2 or inf."""
    kind, tensors = _norm_kind(norm_type), list(tensors)
    if not tensors:
        return torch.zeros(())
    dev = _check(tensors)
    return _run([t.contiguous() for t in tensors], None, 0.0, kind, dev)


@torch.no_grad()
def clip_by_global_norm(tensors: Iterable[torch.Tensor], max_norm: float,
                        norm_type: float = 2.0) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """(clipped, norm): new tensors t * min(1, max_norm / (norm + 1e-6)), and the norm before clipping (a float32
    scalar on their device).  A norm that is not finite scales by 0 (infinite) or NaN."""
    kind, limit, tensors = _norm_kind(norm_type), _limit(max_norm), list(tensors)
    if not tensors:
        return [], torch.zeros(())
    dev = _check(tensors)
    src = [t if t.is_contiguous() and not t.is_conj() and not t.is_neg()
           else t.resolve_conj().resolve_neg().contiguous() for t in tensors]
    dst = [torch.empty_like(t) for t in src]
    return dst, _run(src, dst, limit, kind, dev)


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the gradients of ``parameters`` in place by their global norm and returns the norm before clipping
    (a float32 scalar on their device; torch.nn.utils.clip_grad_norm_'s arguments).  Parameters without a gradient
    are skipped, and one listed twice counts once.  ``error_if_nonfinite`` waits for the norm, and raises before any
    gradient is changed."""
    kind, limit = _norm_kind(norm_type), _limit(max_norm)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = list({id(p.grad): p.grad for p in list(parameters) if p.grad is not None}.values())
    if not grads:
        return torch.zeros(())
    dev = _check(grads)
    flat = [g.contiguous() for g in grads]
    if error_if_nonfinite:
        norm = _run(flat, None, 0.0, kind, dev)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the total norm of the gradients is {float(norm)}, so it cannot be clipped; pass "
                               "error_if_nonfinite=False to scale by it anyway")
    norm = _run(flat, flat, limit, kind, dev)
    torch.autograd.graph.increment_version([t for t in flat if not t.is_inference()])  # written behind autograd's back
    for g, f in zip(grads, flat):
        if f is not g:
            g.copy_(f)
    return norm
