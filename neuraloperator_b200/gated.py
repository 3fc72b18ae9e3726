"""Gated feed-forward block at every point of a field [batch, channels, *grid] (nop_gated_forward /
nop_gated_backward):

    h = act(w_gate x + b_gate) * (w_up x + b_up),   y = w_down h + b_down

``gated_mlp`` runs under autograd (the backward computes the hidden values again from x, so none are kept);
``layers.GatedChannelMLP`` is the layer, which FNOBlocks uses as ``channel_mlp_type="gated"``.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .utils import dense, refuse_tangents

_DTYPES = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
MAX_CHANNELS = 256
MAX_HIDDEN = 16384


def _matrix(w: torch.Tensor) -> torch.Tensor:
    """[out, in] view of a matrix or of a Conv1d(k=1) weight [out, in, 1]."""
    return w[..., 0] if w.ndim == 3 and w.shape[-1] == 1 else w


def _check(x, w_gate, w_up, w_down, biases, activation, x_scale):
    """Refuses what the kernels do not take; returns (hidden, out_channels)."""
    if not x.is_cuda:
        raise RuntimeError("neuraloperator_b200 runs on CUDA devices only (there is no CPU path)")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if x.ndim < 2:
        raise ValueError(f"expected a field [batch, channels, *grid], got shape {tuple(x.shape)}")
    mats = [_matrix(w) for w in (w_gate, w_up, w_down)]
    if any(m.ndim != 2 for m in mats):
        raise ValueError("the weights must be matrices [out, in] (or Conv1d weights [out, in, 1])")
    hidden, channels, out = mats[0].shape[0], x.shape[1], mats[2].shape[0]
    if mats[0].shape != (hidden, channels) or mats[1].shape != (hidden, channels) or mats[2].shape != (out, hidden):
        raise ValueError(f"weight shapes {[tuple(m.shape) for m in mats]} do not fit {channels} channels: w_gate and "
                         "w_up are [hidden, channels], w_down [out, hidden]")
    if not (1 <= channels <= MAX_CHANNELS and 1 <= out <= MAX_CHANNELS):
        raise ValueError(f"channel counts must be in 1..{MAX_CHANNELS}, got {channels} and {out}")
    if not 1 <= hidden <= MAX_HIDDEN:
        raise ValueError(f"the hidden width must be in 1..{MAX_HIDDEN}, got {hidden}")
    dtype = w_gate.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"expected float32, bfloat16 or float16 weights, got {dtype}")
    for b, n in zip(biases, (hidden, hidden, out)):
        if b is not None and tuple(b.shape) != (n,):
            raise ValueError(f"a bias must have shape ({n},), got {tuple(b.shape)}")
    for t in (w_up, w_down, *biases):
        if t is not None and t.dtype != dtype:
            raise TypeError("weights and biases must have one dtype")
    for t in (w_gate, w_up, w_down, *biases, x_scale):
        if t is not None and t.device != x.device:
            raise ValueError("weights, biases and scales must be on x's device")
    if x_scale is None:
        if x.dtype != dtype:
            raise TypeError(f"x is {x.dtype} and the weights are {dtype}")
    else:
        if x.dtype != torch.float8_e4m3fn or dtype == torch.float32:
            raise TypeError("x_scale goes with a float8_e4m3fn field and bfloat16 or float16 weights")
        if x_scale.dtype != torch.float32 or tuple(x_scale.shape) != (x.shape[0], 1, *x.shape[2:]):
            raise ValueError("x_scale must be float32 [batch, 1, *grid]")
    refuse_tangents(x, w_gate, w_up, w_down, *biases, x_scale)
    return hidden, out


def _desc(x, dtype, hidden, out, activation) -> _lib.NopGatedDesc:
    points = 1
    for n in x.shape[2:]:
        points *= n
    return _lib.NopGatedDesc(_lib.ABI_VERSION, _DTYPES[dtype], _DTYPES.get(x.dtype, _lib.DTYPE_E4M3),
                             _ACTIVATIONS[activation], x.shape[0], points, x.shape[1], hidden, out, 0)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _workspace(lib, desc, backward: int, device) -> torch.Tensor:
    size = ctypes.c_size_t()
    _lib.check(lib.nop_gated_workspace_size(desc, backward, size))
    return torch.empty(size.value, device=device, dtype=torch.uint8)


def _forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, x_scale, hidden, out):
    tensors = [dense(t) for t in (x, x_scale, w_gate, w_up, w_down, b_gate, b_up, b_down)]
    y = torch.empty((x.shape[0], out, *x.shape[2:]), device=x.device, dtype=w_gate.dtype)
    lib, desc = _lib.library(), _desc(x, w_gate.dtype, hidden, out, activation)
    ws = _workspace(lib, desc, 0, x.device)
    ops = _lib.NopGatedOperands(*[_ptr(t) for t in tensors], y.data_ptr())
    _lib.call(lib.nop_gated_forward, x.device, desc, ops, ws.data_ptr(), ws.numel())
    return y


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, hidden, out):
        ctx.cfg = (activation, hidden, out)
        ctx.save_for_backward(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
        return _forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, None, hidden, out)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        activation, hidden, out = ctx.cfg
        saved = ctx.saved_tensors
        x, w_gate, w_up, w_down, b_gate, b_up, b_down = [dense(t) for t in saved]
        gy = dense(gy)
        grads = [torch.empty(t.shape, device=x.device, dtype=t.dtype) if t is not None and need else None
                 for t, need in zip(saved, ctx.needs_input_grad)]
        lib, desc = _lib.library(), _desc(x, w_gate.dtype, hidden, out, activation)
        ws = _workspace(lib, desc, 1 if any(t is not None for t in grads[1:]) else 2, x.device)
        ops = _lib.NopGatedOperands(_ptr(x), None, _ptr(w_gate), _ptr(w_up), _ptr(w_down), _ptr(b_gate), _ptr(b_up),
                                    _ptr(b_down), None)
        g = _lib.NopGatedGrads(gy.data_ptr(), *[_ptr(t) for t in grads])
        _lib.call(lib.nop_gated_backward, x.device, desc, ops, g, ws.data_ptr(), ws.numel())
        return (*grads, None, None, None)


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              b_gate: Optional[torch.Tensor] = None, b_up: Optional[torch.Tensor] = None,
              b_down: Optional[torch.Tensor] = None, *, activation: str = "silu",
              x_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [batch, out, *grid] (see the module docstring).  x: a field [batch, channels, *grid] on a CUDA device;
    w_gate, w_up: [hidden, channels], w_down: [out, hidden] (or Conv1d weights [., ., 1]); biases [hidden], [hidden],
    [out] or None; all of x's dtype: float32 (within about 1e-6 of the results' size at up to 64 channels, 4e-6 at 256),
    bfloat16 or float16 (fp32 sums, results rounded once).  activation: "silu" or "gelu" (exact).  channels and out <= 256,
    hidden <= 16384.  The hidden values, and their gradients on the way into dL/dx, have the dtype's range (float16: one
    above 65504 makes its point's output not finite, and 2^-24 is the smallest step).

    With ``x_scale`` (float32 [batch, 1, *grid]) x is float8_e4m3fn and stands for x * x_scale, as
    ``rms_norm_quantized`` leaves it; weights and output are bfloat16 or float16 (inference only).

    Runs on x's device and its current stream; its workspace is allocated by every call, so captured calls share
    none."""
    biases = (b_gate, b_up, b_down)
    hidden, out = _check(x, w_gate, w_up, w_down, biases, activation, x_scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, x_scale, w_gate, w_up, w_down, *biases)):
        if x_scale is not None:
            raise RuntimeError("an 8-bit field has no backward; call gated_mlp under torch.no_grad()")
        return _GatedFn.apply(x, w_gate, w_up, w_down, *biases, activation, hidden, out)
    return _forward(x, w_gate, w_up, w_down, *biases, activation, x_scale, hidden, out)
