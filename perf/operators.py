"""The per-point feed-forward operators and the gradient clipping, as cases that can be timed and compared.

Three operators on the framework's fields [batch, channels, *grid]:

* the root-mean-square norm over the channels of every point, with the residual's addition (``rms_norm``),
  and its output in 8 bits with one scale a point (``rms_norm_quantized``);
* the gated feed-forward block W_down (act(W_gate x + b_gate) * (W_up x + b_up)) + b_down (``gated_mlp``);
* the global norm over all gradients of a model, and their clipping (``clip_by_global_norm``).

``run`` computes them in elementary torch operations, or with ``own`` set through the package's entry points.
"""

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2, "e4m3": 1}


def listed():
    return [
        # the norm of one small coarse field, as at the end of a multi-resolution sweep: latency alone
        {"name": "norm_coarse_fp32", "op": "norm", "mode": "infer", "dtype": "fp32", "batch": 1, "channels": 32,
         "grid": "16x16", "residual": False},
        # a training step of the block norm at the 2D Navier-Stokes grid and width, the skip added on the way
        {"name": "norm_train_512_fp32", "op": "norm", "mode": "train", "dtype": "fp32", "batch": 8, "channels": 64,
         "grid": "512x512", "residual": True},
        # serving on an odd 3D grid in bf16, the normed field kept in 8 bits for the feed-forward block
        {"name": "norm_e4m3_3d_bf16", "op": "norm", "mode": "e4m3", "dtype": "bf16", "batch": 2, "channels": 96,
         "grid": "61x67x71", "residual": True},
        # the feed-forward block on one small coarse field: latency alone
        {"name": "gated_coarse_fp32", "op": "gated", "mode": "infer", "dtype": "fp32", "batch": 1, "channels": 32,
         "hidden": 16, "out": 32, "grid": "16x16", "act": "silu", "bias": True},
        # inference at the 2D Navier-Stokes grid and width, hidden layer twice the width
        {"name": "gated_infer_512_fp32", "op": "gated", "mode": "infer", "dtype": "fp32", "batch": 8, "channels": 64,
         "hidden": 128, "out": 64, "grid": "512x512", "act": "silu", "bias": True},
        # a training step at the 256 x 256 grid of the single-layer benchmark
        {"name": "gated_train_256_fp32", "op": "gated", "mode": "train", "dtype": "fp32", "batch": 16, "channels": 64,
         "hidden": 128, "out": 64, "grid": "256x256", "act": "silu", "bias": True},
        # a wide block in training, bf16, on an odd grid whose rows are not aligned
        {"name": "gated_train_odd_bf16", "op": "gated", "mode": "train", "dtype": "bf16", "batch": 32, "channels": 128,
         "hidden": 384, "out": 128, "grid": "85x85", "act": "gelu", "bias": False},
        # serving from the 8-bit field that the norm left
        {"name": "gated_e4m3_bf16", "op": "gated", "mode": "e4m3", "dtype": "bf16", "batch": 4, "channels": 96,
         "hidden": 256, "out": 96, "grid": "256x256", "act": "silu", "bias": True},
        # the gradients of the 2D Darcy model: 40 tensors, most of them a few numbers
        {"name": "clip_darcy_fp32", "op": "clip", "dtype": "fp32", "modes": "16x16", "channels": 32, "layers": 4,
         "rank": 0, "clips": True},
        # the gradients of the factorized 2D model in half precision: small odd tensors, the norm under the limit
        {"name": "clip_factorized_fp16", "op": "clip", "dtype": "fp16", "modes": "64x64", "channels": 64, "layers": 4,
         "rank": 9, "clips": False},
        # the gradients of the 3D model: 0.6 GB of spectral weights
        {"name": "clip_3d_fp32", "op": "clip", "dtype": "fp32", "modes": "32x32x32", "channels": 32, "layers": 4,
         "rank": 0, "clips": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _grid(rng, points):
    """A 1D, 2D or 3D grid of at most about `points` points, odd sizes among them."""
    nd = rng.choice((1, 2, 2, 3))
    side = points ** (1.0 / nd)
    return "x".join(str(max(1, int(side * rng.uniform(0.7, 1.0)))) for _ in range(nd))


def draw(rng):
    op = rng.choice(("norm", "norm", "gated", "gated", "gated", "clip"))
    if op == "clip":
        nd = rng.choice((1, 2, 3))
        modes = [_log(rng, 4, {1: 512, 2: 64, 3: 20}[nd]) for _ in range(nd)]
        return {"op": "clip", "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16")), "modes": "x".join(map(str, modes)),
                "channels": _log(rng, 8, 48), "layers": rng.randint(1, 4), "rank": rng.choice((0, 0, rng.randint(2, 8))),
                "clips": rng.random() < 0.7}
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    batch = _log(rng, 1, 16)
    if op == "norm":
        channels = _log(rng, 1, 512)
        points = _log(rng, 1, max(1, min(1 << 20, (1 << 26) // (channels * batch))))
        return {"op": "norm", "mode": rng.choice(("infer", "train", "train", "e4m3")), "dtype": dtype, "batch": batch,
                "channels": channels, "grid": _grid(rng, points), "residual": rng.random() < 0.6}
    channels, hidden = _log(rng, 3, 256), _log(rng, 4, 1024)
    out = channels if rng.random() < 0.7 else _log(rng, 1, 256)
    most = (1 << 32) // (hidden * (2 * channels + out) * batch)
    points = _log(rng, 1, max(1, min(1 << 18, most)))
    mode = rng.choice(("infer", "train", "e4m3") if dtype != "fp32" else ("infer", "train"))
    return {"op": "gated", "mode": mode, "dtype": dtype, "batch": batch, "channels": channels, "hidden": hidden,
            "out": out, "grid": _grid(rng, points), "act": rng.choice(("silu", "gelu")), "bias": rng.random() < 0.5}


def _sizes(text):
    return [int(n) for n in text.split("x")]


def _shapes(case):
    """The parameter shapes of a model of this width (spectral weights last axis halved), as (shape, complex)."""
    modes, c, r = _sizes(case["modes"]), case["channels"], case["rank"]
    kept = modes[:-1] + [modes[-1] // 2 + 1]
    nd = len(kept)
    shapes = [((2 * c, 1 + nd, 1), False), ((2 * c,), False), ((c, 2 * c, 1), False), ((c,), False)]
    for _ in range(case["layers"]):
        if r:
            shapes += [((r,) * (nd + 2), True), ((c, r), True), ((c, r), True)] + [((n, r), True) for n in kept]
        else:
            shapes += [((c, c, *kept), True)]
        shapes += [((c, *(1,) * nd), False), ((c, c, 1), False), ((c // 2, c, 1), False), ((c // 2,), False),
                   ((c, c // 2, 1), False), ((c,), False), ((1, c, *(1,) * nd), False)]
    return shapes + [((2 * c, c, 1), False), ((2 * c,), False), ((1, 2 * c, 1), False), ((1,), False)]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "clip":
        # complex gradients where the model is in fp32; a half-precision model holds them as pairs of reals
        dtype, grads = DTYPES[case["dtype"]], []
        for shape, cplx in _shapes(case):
            scale = 10 ** float(torch.rand((), generator=g, device="cuda") * 2 - 2)
            if cplx:
                pair = randn(*shape, 2, dtype=dtype, scale=scale)
                grads.append(torch.view_as_complex(pair) if dtype == torch.float32 else pair)
            else:
                grads.append(randn(*shape, dtype=dtype, scale=scale))
        total = math.sqrt(sum(float(_real(t).double().square().sum()) for t in grads))
        return {"case": case, "grads": grads, "max_norm": total * (0.3 if case["clips"] else 3.0)}
    dtype, c, b, grid = DTYPES[case["dtype"]], case["channels"], case["batch"], _sizes(case["grid"])
    train = case["mode"] == "train"
    s = {"case": case}
    if case["op"] == "norm":
        s["x"] = randn(b, c, *grid, dtype=dtype, scale=1.5)
        s["res"] = randn(b, c, *grid, dtype=dtype) if case["residual"] else None
        s["w"] = 1 + randn(c, scale=0.2)
        if train:
            s["gy"] = randn(b, c, *grid, dtype=dtype)
            s["gr"] = randn(b, c, *grid, dtype=dtype) if case["residual"] else None
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["res"], s["w"]) if t is not None]
        return s
    h, o = case["hidden"], case["out"]
    s["x"] = randn(b, c, *grid, dtype=dtype)
    s["wg"], s["wu"] = randn(h, c, dtype=dtype, scale=c ** -0.5), randn(h, c, dtype=dtype, scale=c ** -0.5)
    s["wd"] = randn(o, h, dtype=dtype, scale=h ** -0.5)
    for name, n in (("bg", h), ("bu", h), ("bd", o)):
        s[name] = randn(n, dtype=dtype, scale=0.3) if case["bias"] else None
    s["scale"] = None
    if case["mode"] == "e4m3":
        s["x"], s["scale"] = _quantize(s["x"].float())
    if train:
        s["gy"] = randn(b, o, *grid, dtype=dtype)
        s["leaves"] = [t.requires_grad_() for t in _mlp_operands(s) if t is not None]
    return s


def _mlp_operands(s):
    return [s[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd")]


def _real(t):
    return torch.view_as_real(t) if t.is_complex() else t


def _quantize(y):
    """y in e4m3 with one scale a point: the smallest power of two s with max over the channels of |y| <= 448 s."""
    most, e = torch.frexp(y.abs().amax(1, keepdim=True))
    scale = torch.ldexp(torch.ones_like(most), torch.where(most <= 0.875, e - 9, e - 8).clamp(min=-126))
    scale = torch.where(most > 0, scale, torch.ones_like(scale))
    return (y / scale).to(torch.float8_e4m3fn), scale.to(torch.float32)


def _stands_for(q, scale):
    """The values that 8-bit numbers with scales stand for: four significant bits each, exact in bf16."""
    return (q.float() * scale).to(torch.bfloat16)


# ---- the framework's calls --------------------------------------------------------------------------------


def _own(s):
    import neuraloperator_b200 as nb

    case = s["case"]
    if case["op"] == "clip":
        return nb.clip_by_global_norm(s["grads"], s["max_norm"])
    if case["op"] == "norm":
        if case["mode"] == "e4m3":
            q, scale, *r = nb.rms_norm_quantized(s["x"], s["w"], residual=s["res"], eps=EPS)
            return [_stands_for(q, scale), *r]
        y = nb.rms_norm(s["x"], s["w"], residual=s["res"], eps=EPS)
        y, r = y if case["residual"] else (y, None)
        if case["mode"] == "infer":
            return [y, r]
        outs, grads = ([y, r], [s["gy"], s["gr"]]) if case["residual"] else ([y], [s["gy"]])
        return [y, r, *torch.autograd.grad(outs, s["leaves"], grads)]
    y = nb.gated_mlp(s["x"], s["wg"], s["wu"], s["wd"], s["bg"], s["bu"], s["bd"], activation=case["act"],
                     x_scale=s["scale"])
    if case["mode"] != "train":
        return [y]
    return [y, *torch.autograd.grad(y, s["leaves"], s["gy"])]


# ---- the plain forms --------------------------------------------------------------------------------------


def _norm_plain(s):
    case, dtype = s["case"], s["x"].dtype
    shape = (1, -1) + (1,) * (s["x"].ndim - 2)
    x = s["x"].float() if s["res"] is None else s["x"].float() + s["res"].float()
    x = x.to(dtype).float()  # the sum that goes on as the residual is what is normed
    w = s["w"].view(shape)
    inv = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    hat = x * inv
    y, r = hat * w, None if s["res"] is None else x.to(dtype)
    if case["mode"] == "e4m3":
        return [_stands_for(*_quantize(y))] + ([r] if r is not None else [])
    if case["mode"] == "infer":
        return [y.to(dtype), r]
    gy = s["gy"].float()
    gw = (gy * hat).sum([0] + list(range(2, x.ndim)))
    gh = gy * w
    gx = inv * (gh - hat * (gh * hat).mean(1, keepdim=True))
    if r is None:
        return [y.to(dtype), r, gx.to(dtype), gw]
    gx = (gx + s["gr"].float()).to(dtype)
    return [y.to(dtype), r, gx, gx, gw]


def _act(z, kind):
    """The activation and its derivative."""
    if kind == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
    return z * p, p + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5


def _gated_plain(s):
    case, x = s["case"], s["x"]
    b, c, grid = x.shape[0], x.shape[1], x.shape[2:]
    dtype = s["wg"].dtype
    xf = x.float().reshape(b, c, -1)
    if s["scale"] is not None:
        xf = xf * s["scale"].reshape(b, 1, -1)
    wg, wu, wd = s["wg"].float(), s["wu"].float(), s["wd"].float()
    bias = [0.0 if t is None else t.float()[:, None] for t in (s["bg"], s["bu"], s["bd"])]
    gate, up = torch.matmul(wg, xf) + bias[0], torch.matmul(wu, xf) + bias[1]
    a, da = _act(gate, case["act"])
    h = a * up
    y = (torch.matmul(wd, h) + bias[2]).to(dtype).reshape(b, -1, *grid)
    if case["mode"] != "train":
        return [y]
    gy = s["gy"].float().reshape(b, wd.shape[0], -1)
    gh = torch.matmul(wd.t(), gy)
    ggate, gup = gh * up * da, gh * a
    gx = torch.matmul(wg.t(), ggate) + torch.matmul(wu.t(), gup)
    grads = [gx.reshape(x.shape), torch.matmul(ggate, xf.mT).sum(0), torch.matmul(gup, xf.mT).sum(0),
             torch.matmul(gy, h.mT).sum(0)]
    if case["bias"]:
        grads += [ggate.sum((0, 2)), gup.sum((0, 2)), gy.sum((0, 2))]
    return [y] + [t.to(dtype) for t in grads]


def _clip_plain(s):
    total = torch.stack([_real(t).float().square().sum() for t in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (total + 1e-6)).clamp(max=1.0)
    clipped = [t * coef if t.is_complex() else (t.float() * coef).to(t.dtype) for t in s["grads"]]
    return clipped, total


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    with torch.no_grad():
        return _norm_plain(state) if op == "norm" else _gated_plain(state) if op == "gated" else _clip_plain(state)


# ---- the same in 64 bits, from the definitions ------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        flat = torch.cat([_real(t).reshape(-1).double() for t in s["grads"]])
        total = torch.linalg.vector_norm(flat)
        coef = min(1.0, s["max_norm"] / (float(total) + 1e-6))
        return [t.to(torch.complex128 if t.is_complex() else torch.float64) * coef for t in s["grads"]], total
    leaf = {k: (v.detach().double().requires_grad_(v.requires_grad) if torch.is_tensor(v) else v)
            for k, v in s.items() if k != "leaves"}
    if case["op"] == "norm":
        r = leaf["x"] if leaf["res"] is None else leaf["x"] + leaf["res"]
        # the sum is held in the input's type; its rounding has derivative one
        r = r + (r.detach().float().to(s["x"].dtype).double() - r.detach())
        y = torch.movedim(r, 1, -1)
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * leaf["w"]
        y = torch.movedim(y, -1, 1)
        if case["mode"] == "e4m3":
            q, scale = _quantize(y)
            q = [q.double() * scale.double()]
            return q + ([r] if case["residual"] else [])
        if case["mode"] == "infer":
            return [y, r if case["residual"] else None]
        outs, grads = ([y, r], [leaf["gy"], leaf["gr"]]) if case["residual"] else ([y], [leaf["gy"]])
        want = [leaf[k] for k in ("x", "res", "w") if leaf[k] is not None]
        return [y, r if case["residual"] else None, *torch.autograd.grad(outs, want, grads)]
    x = leaf["x"] if leaf["scale"] is None else leaf["x"] * leaf["scale"]
    rows = torch.movedim(x, 1, -1)
    linear = torch.nn.functional.linear
    gate, up = linear(rows, leaf["wg"], leaf["bg"]), linear(rows, leaf["wu"], leaf["bu"])
    a = torch.nn.functional.silu(gate) if case["act"] == "silu" else torch.nn.functional.gelu(gate)
    y = torch.movedim(linear(a * up, leaf["wd"], leaf["bd"]), -1, 1)
    if case["mode"] != "train":
        return [y]
    want = [t for t in _mlp_operands(leaf) if t is not None]
    return [y, *torch.autograd.grad(y, want, leaf["gy"])]


def work(case):
    """Every input read once and every output written once; the products' operations, and ten a value elsewhere."""
    if case["op"] == "clip":
        n = sum(math.prod(shape) * (2 if cplx else 1) for shape, cplx in _shapes(case))
        return {"bytes": 2 * n * SIZES[case["dtype"]], "flops": 3 * n}
    size, points = SIZES[case["dtype"]], case["batch"] * math.prod(_sizes(case["grid"]))
    c = case["channels"]
    if case["op"] == "norm":
        field = points * c
        fields = 2 * size + (2 * size if case["residual"] else 0)  # x, y, and the residual in and out
        if case["mode"] == "train":
            fields += 3 * size + (size if case["residual"] else 0)  # the normed sum again, dL/dy (dL/dr), dL/dx
        if case["mode"] == "e4m3":
            fields += 1 - size
        return {"bytes": field * fields + 8 * c, "flops": 10 * field}
    h, o = case["hidden"], case["out"]
    weights, bias = h * (2 * c + o), (2 * h + o if case["bias"] else 0)
    if case["mode"] == "e4m3":
        return {"bytes": points * (c + 4 + o * size) + (weights + bias) * size,
                "flops": 2 * points * weights}
    io, flops = points * (c + o) * size + (weights + bias) * size, 2 * points * weights
    if case["mode"] == "train":
        # again x and dL/dy, dL/dx and the weight gradients; the products of the gradients are twice the forward's
        io, flops = io + points * (2 * c + o) * size + (2 * weights + bias) * size, 3 * flops
    return {"bytes": io, "flops": flops}
