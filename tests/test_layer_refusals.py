"""What the per-point layers and the clipping refuse, on the CPU: nothing of it reaches a device."""

import ctypes
import math

import pytest
import torch

import neuraloperator_b200 as nb
from neuraloperator_b200 import _lib

f32 = torch.float32


def fake(*shape, dtype=f32):
    return torch.empty(shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        nb.rms_norm(fake(1, 2, 3))
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        nb.rms_norm_quantized(fake(1, 2, 3))
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        nb.RMSNorm(2)(fake(1, 2, 3))
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        nb.clip_by_global_norm([fake(3)], 1.0)
    p = torch.nn.Parameter(fake(3))
    p.grad = fake(3)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        nb.clip_grad_norm_([p], 1.0)


@pytest.mark.parametrize("kw, msg", [(dict(max_norm=-1.0), "max_norm"), (dict(max_norm=math.nan), "max_norm"),
                                     (dict(max_norm=1.0, norm_type=1.0), "norm_type"),
                                     (dict(max_norm=1.0, norm_type=0), "norm_type")])
def test_clip_arguments(kw, msg):
    with pytest.raises(ValueError, match=msg):
        nb.clip_by_global_norm([], **kw)
    with pytest.raises(ValueError, match=msg):
        nb.clip_grad_norm_([], **kw)


def test_nothing_to_clip():
    assert float(nb.clip_grad_norm_([torch.nn.Parameter(fake(3))], 1.0)) == 0.0
    assert float(nb.global_norm([])) == 0.0


def norm_desc(**over):
    d = _lib.NopNormDesc(_lib.ABI_VERSION, 0, 2, 16, 8, 1e-6)
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over, code", [(dict(abi_version=7), -1), (dict(dtype=3), -1), (dict(dtype=-1), -1),
                                        (dict(batch=-1), -1), (dict(points=-1), -1), (dict(channels=0), -1),
                                        (dict(channels=8193), -2), (dict(eps=-1.0), -1), (dict(eps=math.nan), -1),
                                        (dict(batch=1 << 40, points=1 << 20), -2)])
def test_norm_descriptor(over, code):
    lib, size = _lib.library(), ctypes.c_size_t()
    d = norm_desc(**over)
    assert lib.nop_rms_norm_forward(d, 64, None, None, 64, None, None, None, None) == code, _lib.last_error()
    assert lib.nop_rms_norm_backward(d, 64, None, 64, None, 64, None, None, 0, None) == code
    assert lib.nop_rms_norm_backward_workspace_size(d, size) == code


def test_norm_pointers():
    lib, d = _lib.library(), norm_desc()
    fwd = lib.nop_rms_norm_forward
    assert fwd(None, 64, None, None, 64, None, None, None, None) == -1
    assert fwd(d, None, None, None, 64, None, None, None, None) == -1   # no x
    assert fwd(d, 64, None, None, None, None, None, None, None) == -1   # no output
    assert fwd(d, 64, None, None, 64, None, 64, 64, None) == -1         # two outputs
    assert fwd(d, 64, None, None, None, None, 64, None, None) == -1     # no scale
    assert fwd(d, 64, 64, None, 64, None, None, None, None) == -1       # a residual without r
    assert fwd(d, 66, None, None, 64, None, None, None, None) == -3
    assert fwd(norm_desc(batch=0), None, None, None, None, None, None, None, None) == 0
    bwd = lib.nop_rms_norm_backward
    assert bwd(d, None, None, 64, None, 64, None, None, 0, None) == -1
    assert bwd(d, 64, None, 64, None, None, None, None, 0, None) == 0   # nothing asked for
    assert bwd(d, 64, None, 65, None, 64, None, None, 0, None) == -3


def test_clip_pointers():
    lib, size = _lib.library(), ctypes.c_size_t()
    assert lib.nop_clip_workspace_size(-1, size) == -1
    assert lib.nop_clip_workspace_size(3, size) == 0 and size.value > 0

    def call(n=1, src=64, dst=64, numel=4, dtype=0, kind=0, limit=1.0, norm=64, ws=64, ws_bytes=None):
        p = lambda v: None if v is None else (ctypes.c_void_p * 1)(v)  # noqa: E731
        return lib.nop_clip_by_norm(n, p(src), p(dst), (ctypes.c_int64 * 1)(numel), (ctypes.c_int32 * 1)(dtype), kind,
                                    limit, norm, ws, size.value if ws_bytes is None else ws_bytes, None)

    assert call(n=-1) == -1 and call(src=None) == -1 and call(numel=-1) == -1 and call(dtype=3) == -1
    assert call(kind=2) == -1 and call(limit=-1.0) == -1 and call(limit=math.nan) == -1
    assert call(dst=None, norm=None) == -1 and call(src=0) == -1 and call(dst=0) == -1
    assert call(src=66) == -3 and call(dst=66) == -3 and call(ws=68) == -3
    assert call(ws=None) == -4 and call(ws_bytes=8) == -4
