"""FNO and FNOBlocks with RMS norms and gated channel MLPs: forward and every gradient against the same model in
float64 on the CPU (the oracle's spectral convolution, plain torch layers), and a training loop with clipping."""

import pytest
import torch
import torch.nn.functional as F

import neuraloperator_b200 as nb
import oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def exact_convolutions():
    """The blocks' linear skips are torch Conv1d layers, which round their operands to tf32 (2^-11) by default."""
    kept = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    yield
    torch.backends.cudnn.allow_tf32 = kept


def rms(x, m, residual=None):
    r = x if residual is None else x + residual
    return r / torch.sqrt((r * r).mean(1, keepdim=True) + m.eps) * m.weight.view(1, -1, *[1] * (x.ndim - 2))


def mlp(x, m):
    size, x = x.shape, x.reshape(*x.shape[:2], -1)
    lin = lambda fc, t: F.conv1d(t, fc.weight, fc.bias)  # noqa: E731
    if isinstance(m, nb.GatedChannelMLP):
        y = lin(m.down, F.silu(lin(m.gate, x)) * lin(m.up, x))
    else:
        y = lin(m.fcs[1], F.gelu(lin(m.fcs[0], x)))
    return y.reshape(size[0], -1, *size[2:])



def block(fb, x, i, modes):
    """FNOBlocks.forward from its definition, on the CPU in float64."""
    last = i == fb.n_layers - 1
    norm = (lambda k, t, r=None: rms(t, fb.norm[2 * i + k], r)) if fb.norm is not None else None
    skip_lin = lambda t: F.conv1d(t.reshape(*t.shape[:2], -1), fb.fno_skips[i].conv.weight).reshape(t.shape)  # noqa: E731
    spectral = lambda t: oracle.spectral_conv(t, fb.convs[i].weight.tensor, fb.convs[i].bias, modes)  # noqa: E731
    gate = lambda t: fb.channel_mlp_skips[i].weight * t  # noqa: E731
    if fb.preactivation:
        x = F.gelu(x)
        if norm:
            x = norm(0, x)
        a, s = skip_lin(x), gate(x)
        x = spectral(x) + a
        if not last:
            x = F.gelu(x)
        if norm:
            x = norm(1, x)
        return mlp(x, fb.channel_mlp[i]) + s
    s, a = gate(x), skip_lin(x)
    x = spectral(x)
    x = (norm(0, x) if norm else x) + a
    if not last:
        x = F.gelu(x)
    x = mlp(x, fb.channel_mlp[i])
    x = norm(1, x, s) if norm else x + s
    return x if last else F.gelu(x)


def reference(model, x, modes):
    pe = model.positional_embedding
    x = torch.cat([x, *[g.to(x).expand(x.shape[0], 1, *x.shape[2:]) for g in pe.grid(x.shape[2:], "cpu", x.dtype)]], 1)
    x = mlp(x, model.lifting)
    for i in range(model.n_layers):
        x = block(model.fno_blocks, x, i, modes)
    return mlp(x, model.projection)


def rel(a, b):
    return float((a.detach().cpu().to(b.dtype) - b.detach()).norm() / b.detach().norm())


@pytest.mark.parametrize("kw", [dict(norm="rms_norm"), dict(channel_mlp_type="gated"),
                                dict(norm="rms_norm", channel_mlp_type="gated", channel_mlp_expansion=2.0),
                                dict(norm="rms_norm", channel_mlp_type="gated", preactivation=True),
                                dict(norm="rms_norm", preactivation=True)])
@pytest.mark.parametrize("grid, modes", [((64,), (16,)), ((24, 20), (8, 8)), ((15, 21), (6, 6))])
def test_model_against_definition(kw, grid, modes):
    torch.manual_seed(0)
    model = nb.FNO(n_modes=modes, in_channels=2, out_channels=1, hidden_channels=12, n_layers=2, **kw)
    ref = nb.FNO(n_modes=modes, in_channels=2, out_channels=1, hidden_channels=12, n_layers=2, **kw)
    with torch.no_grad():
        if model.fno_blocks.norm is not None:
            for m in model.fno_blocks.norm:
                m.weight.add_(0.3 * torch.randn(m.weight.shape))
    ref.load_state_dict(model.state_dict())
    ref = ref.double()  # (leaves complex parameters as they are)
    for p in ref.parameters():
        if p.is_complex():
            p.data = p.data.to(torch.complex128)
    x, gy = torch.randn(3, 2, *grid), torch.randn(3, 1, *grid)
    want = reference(ref, x.double(), modes)
    want.backward(gy.double())
    model = model.cuda()
    y = model(x.cuda())
    y.backward(gy.cuda())
    # the per-layer paths are held to 1e-5 each elsewhere; a model of two blocks has some ten of them in a row
    assert rel(y, want) <= 2e-5
    for (name, p), q in zip(model.named_parameters(), ref.parameters()):
        assert rel(p.grad, q.grad) <= 5e-5, name
    with torch.no_grad():
        assert rel(model(x.cuda()), want) <= 2e-5


def test_staged_model_and_state():
    model = nb.FNOStaged([(8, 8), (6, 6)], in_channels=1, out_channels=1, hidden_channels=8, norm="rms_norm",
                         channel_mlp_type="gated").cuda()
    x = torch.randn(2, 1, 16, 16, device="cuda")
    y = model(x)
    other = nb.FNOStaged([(8, 8), (6, 6)], in_channels=1, out_channels=1, hidden_channels=8, norm="rms_norm",
                         channel_mlp_type="gated").cuda()
    other.load_state_dict(model.state_dict())
    assert torch.equal(other(x), y)


def test_training_steps_with_clipping():
    """A few steps of a normed, gated model: backward, clip, step; runs, and every gradient is finite and clipped."""
    torch.manual_seed(1)
    model = nb.FNO(n_modes=(8, 8), in_channels=1, out_channels=1, hidden_channels=16, n_layers=2, norm="rms_norm",
                   channel_mlp_type="gated", channel_mlp_expansion=2.0).cuda()
    opt = torch.optim.SGD(model.parameters(), lr=1e-2)
    x, t = torch.randn(4, 1, 32, 32, device="cuda"), torch.randn(4, 1, 32, 32, device="cuda")
    for _ in range(3):
        opt.zero_grad()
        F.mse_loss(model(x), t).backward()
        norm = nb.clip_grad_norm_(model.parameters(), 1e-3, error_if_nonfinite=True)
        assert float(norm) > 1e-3
        assert abs(float(nb.global_norm([p.grad for p in model.parameters()])) - 1e-3) <= 1e-6
        opt.step()


@pytest.mark.parametrize("kw", [dict(channel_mlp_type="gated", channel_mlp_skip="linear"), dict(),
                                dict(channel_mlp_type="gated", preactivation=True)])
def test_normed_models_under_autocast(kw):
    """Autocast makes the torch layers' outputs bf16 and leaves this library's fp32: a skip of another type than the channel
    MLP's output is added in the wider one."""
    torch.manual_seed(0)
    model = nb.FNO(n_modes=(8, 8), in_channels=1, out_channels=1, hidden_channels=16, n_layers=2, norm="rms_norm",
                   **kw).cuda()
    x = torch.randn(2, 1, 16, 20, device="cuda")
    want = model(x)
    with torch.autocast("cuda", torch.bfloat16):
        y = model(x)
    # a dozen torch layers in a row round to bf16, 2^-8 each, and every gain is of the order of one
    assert rel(y, want.cpu()) <= 12 * 2.0 ** -8
    y.float().square().mean().backward()
    assert all(torch.isfinite(torch.view_as_real(p.grad) if p.is_complex() else p.grad).all() for p in model.parameters())
