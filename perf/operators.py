"""The operators that networks of any width are built of and trained with: linear layers with bias, activation and residual in one
pass, layer norm, both with their backward passes, and the global norm of many tensors' gradients with clipping.

listed() and draw() give the cases, prepare() what a program holds before the call, run() one pass (through the framework where
``own`` is true, in elementary torch operations where it is not), exact() the same outputs from the definitions in 64 bits, and
work() the bytes and operations a pass cannot do without."""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # one point through one layer: latency
        dict(name="linear 1x256x256", kind="linear", rows=1, n_in=256, n_out=256, dtype="fp16", activation="ReLU", residual=False, save=False),
        # a few queries through a wide layer: the weights' bytes
        dict(name="linear 16x2048x2048", kind="linear", rows=16, n_in=2048, n_out=2048, dtype="bf16", activation="SiLU", residual=False, save=False),
        # the framework's batch of 2^18 points through the second layer of a residual block 256 wide
        dict(name="linear 2^18x256x256 residual", kind="linear", rows=1 << 18, n_in=256, n_out=256, dtype="fp16", activation="None", residual=True, save=False),
        # the widest layers, in training: the matrix product itself
        dict(name="linear 16384x2048x2048", kind="linear", rows=16384, n_in=2048, n_out=2048, dtype="bf16", activation="GELU", residual=False, save=True),
        # backward of a block's first layer at the framework's batch
        dict(name="linear backward 2^18x256x256", kind="linear_backward", rows=1 << 18, n_in=256, n_out=256, dtype="fp16", activation="ReLU"),
        # a ragged batch and the output width of an SDF with its feature vector, 256 + 1
        dict(name="linear backward 5003x320x257", kind="linear_backward", rows=5003, n_in=320, n_out=257, dtype="bf16", activation="SiLU"),
        # a small batch of narrow rows: latency
        dict(name="norm 1000x64", kind="norm", rows=1000, width=64, dtype="fp16", weights="fp16"),
        # the framework's batch, 256 wide
        dict(name="norm 2^18x256", kind="norm", rows=1 << 18, width=256, dtype="fp16", weights="fp16"),
        # its backward pass, with the skip connection's gradient
        dict(name="norm backward 2^18x256", kind="norm_backward", rows=1 << 18, width=256, dtype="fp16", weights="fp16", skip=True),
        # a ragged batch of odd rows, weights kept in fp32
        dict(name="norm backward 5003x1001", kind="norm_backward", rows=5003, width=1001, dtype="bf16", weights="fp32", skip=False),
        # one field's gradients, networks and table, clipped into buffers of their own
        dict(name="clip 4 tensors", kind="clip", tensors=4, total=12612212, dtype="fp16", sizes=1, clips=True),
        # many tensors of a large network, below the limit: most steps of a training
        dict(name="clip 60 tensors", kind="clip", tensors=60, total=50000000, dtype="mixed", sizes=2, clips=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.4 else max(lo, w // 8 * 8)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_backward", "linear_backward", "norm", "norm_backward", "clip"])
    if kind in ("linear", "linear_backward"):
        n_in, n_out = _width(rng, 16, 4096), _width(rng, 16, 4096)
        most = min(1 << 18, (16384 * 2048 * 2048 if kind == "linear" else 8192 * 2048 * 2048) // (n_in * n_out), (1 << 26) // max(n_in, n_out))
        case = dict(kind=kind, rows=_log(rng, 1, most), n_in=n_in, n_out=n_out, dtype=rng.choice(["fp16", "bf16"]), activation=rng.choice(["None", "ReLU", "SiLU", "GELU"]))
        if kind == "linear":
            case.update(residual=rng.random() < 0.5, save=rng.random() < 0.5)
        return case
    if kind in ("norm", "norm_backward"):
        width, dtype = _width(rng, 16, 8192), rng.choice(["fp16", "bf16", "fp32"])
        case = dict(kind=kind, rows=_log(rng, 1, min(1 << 18, (1 << 26) // width)), width=width, dtype=dtype, weights=rng.choice([dtype, "fp32"]))
        if kind == "norm_backward":
            case.update(skip=rng.random() < 0.5)
        return case
    return dict(kind=kind, tensors=rng.randint(1, 60), total=_log(rng, 10000, 50000000), dtype=rng.choice(["fp16", "bf16", "fp32", "mixed"]), sizes=rng.randrange(1000),
                clips=rng.random() < 0.5)


def _clip_sizes(case):
    """Element counts of the tensors: a few large ones, many small ones, as networks have them."""
    rng = random.Random(case["sizes"])
    share = [math.exp(rng.uniform(0, 6)) for _ in range(case["tensors"])]
    scale = case["total"] / sum(share)
    names = ["fp16", "bf16", "fp32"]
    return [(max(1, int(s * scale)), names[rng.randrange(3)] if case["dtype"] == "mixed" else case["dtype"]) for s in share]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    """The tensors that a case's call reads."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    kind = case["kind"]
    if kind == "clip":
        # gradients under the framework's loss scale, tensors of different magnitudes
        tensors = [(normal(n) * (128 * 0.001 * math.exp(0.5 * (i % 5)))).to(DTYPES[t]) for i, (n, t) in enumerate(_clip_sizes(case))]
        return dict(gradients=tensors)
    t, rows = DTYPES[case["dtype"]], case["rows"]
    if kind in ("linear", "linear_backward"):
        n_in, n_out = case["n_in"], case["n_out"]
        bound = math.sqrt(6.0 / (n_in + n_out))
        w = (torch.rand(n_out, n_in, device="cuda", generator=gen) * 2 - 1) * bound
        params = torch.cat([w.reshape(-1), normal(n_out) * 0.1]).to(t)
        d = dict(x=normal(rows, n_in).to(t), params=params)
        if kind == "linear":
            d["residual"] = normal(rows, n_out).to(t) if case["residual"] else None
        else:
            d["pre"] = normal(rows, n_out).to(t) if case["activation"] != "None" else None
            d["dy"] = (normal(rows, n_out) * (128.0 / rows)).to(t)
        return d
    width, tw = case["width"], DTYPES[case["weights"]]
    # rows as a residual stream has them: columns of different means, rows of different sizes
    x = normal(rows, width) * torch.exp(0.5 * normal(rows, 1)) + 0.5 * normal(width)
    d = dict(x=x.to(t), params=torch.cat([1 + 0.1 * normal(width), 0.1 * normal(width)]).to(tw))
    if kind == "norm_backward":
        d["dy"] = (normal(rows, width) * (128.0 / rows)).to(t)
        d["skip"] = (normal(rows, width) * (128.0 / rows)).to(t) if case["skip"] else None
        f = d["x"].float()
        mean = f.mean(1)
        d["mean"], d["rstd"] = mean, torch.rsqrt((f - mean[:, None]).square().mean(1) + 1e-5)
    return d


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    kind = case["kind"]
    if kind == "clip":
        total = math.sqrt(sum(float(g.double().square().sum()) for g in s["gradients"])) / 128.0
        s["max_norm"] = total * (0.37 if case["clips"] else 1.5)
        s["into"] = [torch.empty_like(g) for g in s["gradients"]] if case["clips"] else None
    elif kind in ("linear", "linear_backward"):
        s["w"], s["b"] = s["params"][:case["n_in"] * case["n_out"]].view(case["n_out"], case["n_in"]), s["params"][case["n_in"] * case["n_out"]:]
        s["gradients"] = torch.zeros_like(s["params"]) if kind == "linear_backward" else None
    else:
        s["scale"], s["shift"] = s["params"][:case["width"]], s["params"][case["width"]:]
        s["gradients"] = torch.zeros_like(s["params"]) if kind == "norm_backward" else None
    if own:
        from neus2_amd.layers import GradientClip, LayerNorm, Linear
        if kind == "clip":
            s["op"] = GradientClip(s["gradients"], out=s["into"])
        elif kind in ("linear", "linear_backward"):
            s["op"] = Linear(case["n_in"], case["n_out"], activation=case["activation"], dtype=DTYPES[case["dtype"]])
            s["op"].set_params(s["params"], s["gradients"])
        else:
            s["op"] = LayerNorm(case["width"], dtype=DTYPES[case["dtype"]], param_dtype=DTYPES[case["weights"]])
            s["op"].set_params(s["params"], s["gradients"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _activation(z, name):
    if name == "ReLU":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "SiLU":
        return z * torch.sigmoid(z)
    if name == "GELU":
        return z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    return z


def _slope(z, name):
    if name == "ReLU":
        return (z > 0).to(z.dtype)
    if name == "SiLU":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "GELU":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    kind = case["kind"]
    if kind == "clip":
        norm = torch.sqrt(torch.stack([(g.float() / 128.0).square().sum() for g in s["gradients"]]).sum())
        factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        return dict(norm=norm, gradients=[(g.float() * factor).to(g.dtype) for g in s["gradients"]])
    t = DTYPES[case["dtype"]]
    if kind == "linear":
        z = s["x"].float() @ s["w"].float().t() + s["b"].float()
        y = _activation(z, case["activation"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return dict(y=y.to(t), pre=z.to(t)) if case["save"] else dict(y=y.to(t))
    if kind == "linear_backward":
        dz = s["dy"].float()
        if s["pre"] is not None:
            dz = dz * _slope(s["pre"].float(), case["activation"])
        return dict(dx=(dz @ s["w"].float()).to(t), dw=(dz.t() @ s["x"].float()).to(t), db=dz.sum(0).to(t))
    x, scale, shift = s["x"].float(), s["scale"].float(), s["shift"].float()
    if kind == "norm":
        mean = x.mean(1)
        centred = x - mean[:, None]
        rstd = torch.rsqrt(centred.square().mean(1) + 1e-5)
        return dict(y=(centred * rstd[:, None] * scale + shift).to(t), mean=mean, rstd=rstd)
    xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["dy"].float()
    h = dy * scale
    dx = s["rstd"][:, None] * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
    if s["skip"] is not None:
        dx = dx + s["skip"].float()
    return dict(dx=dx.to(t), dscale=(dy * xh).sum(0).to(s["scale"].dtype), dshift=dy.sum(0).to(s["scale"].dtype))


def _run_own(s):
    case, op = s["case"], s["op"]
    kind = case["kind"]
    if kind == "clip":
        norm = op.clip(s["max_norm"], loss_scale=128.0)
        return dict(norm=norm, gradients=s["gradients"] if s["into"] is None else s["into"])
    if kind == "linear":
        y, pre = op.forward(s["x"], residual=s["residual"], want_pre_activation=case["save"])
        return dict(y=y, pre=pre) if case["save"] else dict(y=y)
    if kind == "linear_backward":
        dx = op.backward(s["x"], s["pre"], s["dy"])
        n = s["w"].numel()
        return dict(dx=dx, dw=s["gradients"][:n].view(s["w"].shape), db=s["gradients"][n:])
    if kind == "norm":
        y, (mean, rstd) = op.forward(s["x"], want_ctx=True)
        return dict(y=y, mean=mean, rstd=rstd)
    dx = op.backward((s["mean"], s["rstd"]), s["x"], s["dy"], dL_dskip=s["skip"])
    return dict(dx=dx, dscale=s["gradients"][:case["width"]], dshift=s["gradients"][case["width"]:])


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, and what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    d = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "clip":
        gradients = [g.double() for g in d["gradients"]]
        norm = sum(float((g * g).sum()) for g in gradients) ** 0.5 / 128.0
        limit = norm * (0.37 if case["clips"] else 1.5)
        factor = min(1.0, limit / (norm + 1e-6))
        return dict(norm=torch.tensor(norm, dtype=torch.float64, device="cuda"), gradients=[g * factor for g in gradients])
    if kind in ("linear", "linear_backward"):
        n_in, n_out, name = case["n_in"], case["n_out"], case["activation"]
        w, b = d["params"][:n_in * n_out].reshape(n_out, n_in), d["params"][n_in * n_out:]
        if kind == "linear":
            z = torch.addmm(b, d["x"], w.T.contiguous())
            y = {"None": lambda: z, "ReLU": lambda: z.clamp(min=0), "SiLU": lambda: z / (1 + (-z).exp()), "GELU": lambda: z * torch.erfc(z * -(0.5 ** 0.5)) / 2}[name]()
            y = y if d["residual"] is None else y + d["residual"]
            return dict(y=y, pre=z) if case["save"] else dict(y=y)
        z, dz = d["pre"], d["dy"]
        if name == "ReLU":
            dz = dz.masked_fill(z <= 0, 0)
        elif name == "SiLU":
            e = 1 + (-z).exp()
            dz = dz * (1 / e + z * (e - 1) / e ** 2)
        elif name == "GELU":
            dz = dz * (torch.erfc(z * -(0.5 ** 0.5)) / 2 + z * (z * z / -2).exp() / (2 * math.pi) ** 0.5)
        return dict(dx=torch.mm(dz, w), dw=torch.mm(dz.T.contiguous(), d["x"]), db=dz.sum(0))
    x, scale, shift = d["x"], d["params"][:case["width"]], d["params"][case["width"]:]
    if kind == "norm":
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + 1e-5) ** -0.5
        return dict(y=(x - mean.unsqueeze(1)) * (rstd.unsqueeze(1) * scale) + shift, mean=mean, rstd=rstd)
    mean, rstd, dy, n = d["mean"].unsqueeze(1), d["rstd"].unsqueeze(1), d["dy"], case["width"]
    xh = (x - mean) * rstd
    h = dy * scale
    dx = (h * n - h.sum(1, True) - xh * (h * xh).sum(1, True)) * (rstd / n)
    dx = dx if d["skip"] is None else dx + d["skip"]
    return dict(dx=dx, dscale=(dy * xh).sum(0), dshift=dy.sum(0))


def work(case):
    kind = case["kind"]
    if kind == "clip":
        n = [(count, SIZE[t]) for count, t in _clip_sizes(case)]
        elements, moved = sum(c for c, _ in n), sum(c * b for c, b in n)
        # (read once and, where something is clipped, written once)
        return dict(bytes=moved * (2 if case["clips"] else 1) + 4, flops=elements * (3 if case["clips"] else 2))
    b, rows = SIZE[case["dtype"]], case["rows"]
    if kind == "linear":
        i, o = case["n_in"], case["n_out"]
        return dict(bytes=b * (rows * i + o * i + o + rows * o * (1 + case["residual"] + case["save"])), flops=2 * rows * i * o)
    if kind == "linear_backward":
        i, o = case["n_in"], case["n_out"]
        return dict(bytes=b * (2 * rows * i + rows * o * (1 if case["activation"] == "None" else 2) + 2 * o * i + o), flops=4 * rows * i * o)
    w, p = case["width"], SIZE[case["weights"]]
    if kind == "norm":
        return dict(bytes=b * 2 * rows * w + 2 * p * w + 8 * rows, flops=8 * rows * w)
    return dict(bytes=b * rows * w * (3 + case["skip"]) + 3 * p * w + 8 * rows, flops=14 * rows * w)
