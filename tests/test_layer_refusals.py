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


def gated_ops(c=4, h=6, o=3, dtype=f32):
    return [fake(h, c, dtype=dtype), fake(h, c, dtype=dtype), fake(o, h, dtype=dtype)]


def test_gated_mlp_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        nb.gated_mlp(fake(1, 4, 5), *gated_ops())


@pytest.mark.parametrize("case, error", [
    (dict(activation="relu"), ValueError),
    (dict(x=(4,)), ValueError),
    (dict(x=(1, 5, 7)), ValueError),
    (dict(w_up=(6, 5)), ValueError),
    (dict(w_down=(3, 7)), ValueError),
    (dict(w_gate=(6, 4, 2)), ValueError),
    (dict(b_gate=(5,)), ValueError),
    (dict(b_down=(6,)), ValueError),
    (dict(x=(1, 300, 7), w_gate=(6, 300), w_up=(6, 300)), ValueError),
    (dict(w_down=(257, 6)), ValueError),
    (dict(w_gate=(16385, 4), w_up=(16385, 4), w_down=(3, 16385)), ValueError),
    (dict(x=(1, 4, 7), dtype_x=torch.bfloat16), TypeError),
    (dict(dtype=torch.float64), TypeError),
    (dict(x_scale=(1, 1, 7)), TypeError),
    (dict(dtype_x=torch.float8_e4m3fn, x_scale=(1, 1, 7)), TypeError),
])
def test_gated_mlp_arguments(case, error, monkeypatch):
    """The checks run on the host; the tensors only claim to be on a device."""
    from neuraloperator_b200 import gated

    dtype = case.get("dtype", f32)
    t = {"x": (1, 4, 7), "w_gate": (6, 4), "w_up": (6, 4), "w_down": (3, 6), "b_gate": None, "b_up": None,
         "b_down": None, "x_scale": None, **{k: v for k, v in case.items() if isinstance(v, tuple)}}
    t = {k: None if v is None else torch.empty(v, dtype=dtype, device="meta") for k, v in t.items()}
    if "dtype_x" in case:
        t["x"] = t["x"].to(case["dtype_x"])
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    with pytest.raises(error):
        gated._check(t["x"], t["w_gate"], t["w_up"], t["w_down"], (t["b_gate"], t["b_up"], t["b_down"]),
                     case.get("activation", "silu"), t["x_scale"])


def gated_desc(**over):
    d = _lib.NopGatedDesc(_lib.ABI_VERSION, 0, 0, 0, 2, 16, 8, 12, 8, 0)
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over, code", [
    (dict(), 0), (dict(abi_version=7), -1), (dict(dtype=3), -1), (dict(x_dtype=1), -1), (dict(x_dtype=3), -2),
    (dict(dtype=1, x_dtype=3), 0), (dict(activation=2), -1), (dict(batch=-1), -1), (dict(points=-1), -1),
    (dict(channels=0), -1), (dict(hidden=0), -1), (dict(out_channels=0), -1), (dict(channels=257), -2),
    (dict(out_channels=257), -2), (dict(hidden=16385), -2), (dict(batch=1 << 16, points=1 << 16), -2)])
def test_gated_descriptor(over, code):
    lib, size = _lib.library(), ctypes.c_size_t()
    assert lib.nop_gated_workspace_size(gated_desc(**over), 0, size) == code, _lib.last_error()


def test_gated_plan_takes_every_width():
    """Every admitted combination of channels, hidden width, type and pass has a plan."""
    lib, size = _lib.library(), ctypes.c_size_t()
    for dtype in range(3):
        for c in (1, 16, 17, 64, 127, 128, 129, 250, 256):
            for o in (1, 16, 100, 128, 129, 256):
                for h in (1, 16, 17, 48, 64, 65, 100, 129, 500, 16384):
                    for backward in (0, 1):
                        d = gated_desc(dtype=dtype, x_dtype=dtype, channels=c, out_channels=o, hidden=h)
                        assert lib.nop_gated_workspace_size(d, backward, size) == 0, (dtype, c, o, h, backward)


def test_gated_pointers():
    lib, size = _lib.library(), ctypes.c_size_t()
    d = gated_desc()
    assert lib.nop_gated_workspace_size(d, 0, size) == 0
    full = dict(x=512, w_gate=512, w_up=512, w_down=512, y=512)
    ops = lambda **kw: _lib.NopGatedOperands(**{**full, **kw})  # noqa: E731
    fwd = lambda o, ws=512, n=None: lib.nop_gated_forward(d, o, ws, size.value if n is None else n, None)  # noqa: E731
    for name in full:
        assert fwd(ops(**{name: None})) == -1, name
    assert fwd(ops(x=514)) == -3 and fwd(ops(b_up=513)) == -3 and fwd(ops(), ws=520) == -3
    assert fwd(ops(), ws=None) == -4 and fwd(ops(), n=8) == -4
    assert lib.nop_gated_forward(gated_desc(dtype=1, x_dtype=3), ops(), 512, 1 << 30, None) == -1  # no scales
    g = _lib.NopGatedGrads(gy=None, gx=512)
    assert lib.nop_gated_backward(d, ops(), g, 512, 1 << 30, None) == -1
    assert lib.nop_gated_backward(d, ops(), None, 512, 1 << 30, None) == -1
    assert lib.nop_gated_backward(d, ops(), _lib.NopGatedGrads(gy=512, gx=513), 512, 1 << 30, None) == -3
    assert lib.nop_gated_backward(d, ops(), _lib.NopGatedGrads(gy=512, gx=512), 512, 8, None) == -4
    assert lib.nop_gated_backward(gated_desc(dtype=1, x_dtype=3), ops(), g, 512, 1 << 30, None) == -2


def test_block_options():
    kw = dict(n_modes=(4, 4), in_channels=1, out_channels=1, hidden_channels=8)
    with pytest.raises(NotImplementedError, match="norm"):
        nb.FNO(**kw, norm="group_norm")
    with pytest.raises(ValueError, match="channel_mlp_type"):
        nb.FNO(**kw, channel_mlp_type="glu")
    with pytest.raises(ValueError, match="dropout"):
        nb.FNO(**kw, channel_mlp_type="gated", channel_mlp_dropout=0.1)
    with pytest.raises(ValueError, match="channels"):
        nb.GatedChannelMLP(300)
    model = nb.FNO(**kw, n_layers=3, norm="rms_norm", channel_mlp_type="gated")
    assert len(model.fno_blocks.norm) == 6 and isinstance(model.fno_blocks.channel_mlp[0], nb.GatedChannelMLP)
    with pytest.raises(RuntimeError, match="CUDA"):
        model(fake(1, 1, 8, 8))
    assert nb.FNO(**kw).fno_blocks.norm is None  # the default is as it was


def test_gated_workspace_of_a_part():
    """dL/dx alone takes the packed weights and no scratch of the points; the backward checks what it is given."""
    lib, size = _lib.library(), ctypes.c_size_t()
    for dtype in range(3):
        sizes = {}
        for points in (16, 1 << 20):
            d = gated_desc(dtype=dtype, x_dtype=dtype, points=points)
            for which in (0, 1, 2):
                assert lib.nop_gated_workspace_size(d, which, size) == 0
                sizes[points, which] = size.value
        assert sizes[16, 2] == sizes[1 << 20, 2] < sizes[16, 1] < sizes[1 << 20, 1]
        ops = _lib.NopGatedOperands(x=512, w_gate=512, w_up=512, w_down=512)
        back = lambda n, **g: lib.nop_gated_backward(d, ops, _lib.NopGatedGrads(gy=512, **g), 512, n, None)  # noqa: E731
        assert back(sizes[1 << 20, 2], gx=512, gb_up=512) == -4 and back(sizes[1 << 20, 2] - 1, gx=512) == -4
    assert lib.nop_gated_workspace_size(gated_desc(), 3, size) == -1
    assert lib.nop_gated_workspace_size(gated_desc(), -1, size) == -1


@pytest.mark.parametrize("preactivation", [False, True])
@pytest.mark.parametrize("use_channel_mlp", [False, True])
def test_every_norm_is_used(preactivation, use_channel_mlp, monkeypatch):
    """Each layer's forward calls all of its norms, and no other's."""
    blocks = nb.FNOBlocks(4, 4, (2, 2), n_layers=2, norm="rms_norm", preactivation=preactivation,
                          use_channel_mlp=use_channel_mlp)
    called = []
    monkeypatch.setattr(nb.RMSNorm, "forward", lambda self, x, residual=None: (
        called.append(id(self)), x if residual is None else (x + residual, x))[1])
    monkeypatch.setattr(nb.SpectralConv, "forward", lambda self, x, output_shape=None: x)
    for index in range(2):
        blocks(torch.zeros(1, 4, 4, 4), index)
    assert called == [id(m) for m in blocks.norm]
