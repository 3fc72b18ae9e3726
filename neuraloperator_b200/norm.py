"""Root-mean-square norm over the channels of every point of a field [batch, channels, *grid], with the
residual's addition and an 8-bit output (nop_rms_norm_forward / nop_rms_norm_backward).

    r = x + residual          (r = x without one)
    y = r / sqrt(mean over the channels of r^2 + eps) * weight

``rms_norm`` runs under autograd; ``RMSNorm`` is the layer, which FNOBlocks uses as ``norm="rms_norm"``.
``rms_norm_quantized`` leaves y in float8_e4m3fn with one power-of-two scale a point, the form in which
``gated_mlp`` reads it (inference).
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple, Union

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .utils import dense, refuse_tangents

_DTYPES = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}


def _check(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor], eps: float):
    if not x.is_cuda:
        raise RuntimeError("neuraloperator_b200 runs on CUDA devices only (there is no CPU path)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"expected a float32, bfloat16 or float16 field, got {x.dtype}")
    if x.ndim < 2 or x.shape[1] < 1:
        raise ValueError(f"expected a field [batch, channels, *grid], got shape {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must be a number >= 0, got {eps}")
    if weight is not None:
        if weight.ndim != 1 or weight.shape[0] != x.shape[1]:
            raise ValueError(f"weight must have shape ({x.shape[1]},), got {tuple(weight.shape)}")
        if weight.device != x.device or not weight.dtype.is_floating_point:
            raise ValueError("weight must be a floating-point tensor on x's device")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError("residual must have x's shape, dtype and device")
    refuse_tangents(x, weight, residual)


def _desc(x: torch.Tensor, eps: float) -> _lib.NopNormDesc:
    batch, channels = x.shape[0], x.shape[1]
    points = 1
    for n in x.shape[2:]:
        points *= n
    return _lib.NopNormDesc(_lib.ABI_VERSION, _DTYPES[x.dtype], batch, points, channels, eps)


@functools.lru_cache(maxsize=None)
def _workspace_bytes(channels: int) -> int:
    """Bytes of the backward's workspace: they depend on the channels alone."""
    size = ctypes.c_size_t()
    _lib.check(_lib.library().nop_rms_norm_backward_workspace_size(
        _lib.NopNormDesc(_lib.ABI_VERSION, _lib.DTYPE_FP32, 1, 1, channels, 0.0), size))
    return size.value


def _fp32(weight: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if weight is None or (weight.dtype is torch.float32 and weight.is_contiguous() and not weight.is_neg()):
        return weight
    return dense(weight.detach().to(torch.float32))


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _forward(x, weight, residual, eps):
    """(y, r): r is x itself without a residual."""
    x, residual = dense(x), dense(residual)
    y = torch.empty_like(x)
    r = x if residual is None else torch.empty_like(x)
    w = _fp32(weight)
    _lib.call(_lib.library().nop_rms_norm_forward, x.device, _desc(x, eps), x.data_ptr(), _ptr(residual), _ptr(w),
              y.data_ptr(), None if residual is None else r.data_ptr(), None, None)
    return y, r


class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, r = _forward(x, weight, residual, eps)
        ctx.set_materialize_grads(False)
        ctx.eps, ctx.with_residual = eps, residual is not None
        ctx.save_for_backward(r, weight)
        return (y, r) if residual is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gr=None):
        r, weight = ctx.saved_tensors
        need_x, need_w, need_res = ctx.needs_input_grad[:3]
        if gy is None:  # only the sum was used
            return gr if need_x else None, None, gr if need_res else None, None
        need_r = need_x or need_res
        gy = dense(gy)
        gr = dense(gr) if need_r else None
        gx = torch.empty_like(r) if need_r else None
        need_w = need_w and weight is not None
        gw = torch.empty(r.shape[1], device=r.device, dtype=torch.float32) if need_w else None
        size = _workspace_bytes(r.shape[1]) if need_w else 0
        ws = torch.empty(size, device=r.device, dtype=torch.uint8) if need_w else None
        w = _fp32(weight)
        _lib.call(_lib.library().nop_rms_norm_backward, r.device, _desc(r, ctx.eps), r.data_ptr(), _ptr(w), gy.data_ptr(),
                  _ptr(gr), _ptr(gx), _ptr(gw), _ptr(ws), size)
        return (gx if need_x else None, gw.to(weight.dtype) if need_w else None, gx if need_res else None, None)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """y, or (y, x + residual) with a residual (see the module docstring).  x: a float32, bfloat16 or float16 field
    [batch, channels, *grid] on a CUDA device; residual: the same shape and dtype; weight: [channels], any
    floating-point dtype (None: ones).  The sum is rounded to x's dtype before it is normed; the statistics are
    float32 (values above 1.8e19 have an infinite square).  Runs on x's device and its current stream."""
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        return _RMSNormFn.apply(x, weight, residual, eps)
    y, r = _forward(x, weight, residual, eps)
    return (y, r) if residual is not None else y


def rms_norm_quantized(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                       residual: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, ...]:
    """(q, scale), or (q, scale, x + residual): rms_norm with y in float8_e4m3fn, y ~ q * scale.  scale is float32
    [batch, 1, *grid], for every point the least power of two with max over the channels of |y| <= 448 * scale (1
    where every y is zero, or one is not finite: infinities and NaN become NaN).  Inference only."""
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_quantized has no backward; call it under torch.no_grad()")
    x, residual = dense(x), dense(residual)
    q = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scale = torch.empty((x.shape[0], 1, *x.shape[2:]), device=x.device, dtype=torch.float32)
    r = None if residual is None else torch.empty_like(x)
    w = _fp32(weight)
    _lib.call(_lib.library().nop_rms_norm_forward, x.device, _desc(x, eps), x.data_ptr(), _ptr(residual), _ptr(w), None,
              _ptr(r), q.data_ptr(), scale.data_ptr())
    return (q, scale) if r is None else (q, scale, r)


class RMSNorm(nn.Module):
    """rms_norm with a learned weight per channel (ones at the start)."""

    def __init__(self, channels: int, eps: float = 1e-6):
        super().__init__()
        self.channels, self.eps = channels, eps
        self.weight = nn.Parameter(torch.ones(channels))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, residual=residual, eps=self.eps)

    def extra_repr(self) -> str:
        return f"{self.channels}, eps={self.eps}"
