"""The layers' formulas in 64 bits, and how far fp32 sums and one rounding may be from them."""
import math

import torch

U32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the distance between the smallest numbers of a type: what rounding may move where a relative step does not hold."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def act(z, kind):
    if kind == "ReLU":
        return torch.where(z > 0, z, 0.0)
    if kind == "SiLU":
        return z * torch.sigmoid(z)
    if kind == "GELU":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    return z


def slope(z, kind):
    if kind == "ReLU":
        return (z > 0).double()
    if kind == "SiLU":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if kind == "GELU":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def within(got, exact, error, what, dtype=None):
    """|got - exact| <= error before the rounding, plus that rounding: half a step of the value, or of the smallest numbers."""
    dtype = got.dtype if dtype is None else dtype
    got, exact = got.double().cpu(), exact.cpu()
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    error = torch.as_tensor(error).double().cpu()
    bound = error + half_step(dtype) * (exact.abs() + error) + least(dtype)
    off = (got - exact).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = int((off - bound).nan_to_num(nan=math.inf).reshape(-1).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; at {i} got {got.reshape(-1)[i]:.9g}, exact {exact.reshape(-1)[i]:.9g}, bound {bound.reshape(-1)[i]:.3g}")


def linear_forward(x, w, b, r, kind):
    """(y, z, bound on the fp32 error of y, of z): k products and their sum in fp32 are off by at most 2 (k + 2) half steps of the sum of
    magnitudes (every addition counted with a whole step: the matrix cores may cut off); the activations have slopes below 1.13 and are
    evaluated within 16 half steps of a value no larger than |z|."""
    x, w = x.double(), w.double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device) if b is None else b.double()
    z = x @ w.T + b
    dz = 2 * (x.shape[1] + 2) * U32 * (x.abs() @ w.abs().T + b.abs())
    y = act(z, kind)
    dy = 1.13 * dz + 16 * U32 * z.abs()
    if r is not None:
        y = y + r.double()
        dy = dy + U32 * y.abs()
    return y, z, dy, dz


def linear_backward(x, w, z, dy, kind):
    """dict(dx, dw, db) with bounds: dz is rounded to the type (half a step) after its slope, which is off by at most 2^-20, has met dy."""
    dtype = dy.dtype
    x, w, g = x.double(), w.double(), dy.double()
    dz = g if kind == "None" else g * slope(z.double(), kind)
    slope_error = 0.0 if kind in ("None", "ReLU") else 2.0 ** -20 * g.abs()
    rounded = slope_error if kind in ("None", "ReLU") else slope_error + half_step(dtype) * (dz.abs() + slope_error) + least(dtype)
    error = rounded + torch.zeros_like(dz)
    n, o = x.shape[0], w.shape[0]
    size = dz.abs() + error
    dx = (dz @ w, error @ w.abs() + 2 * (o + 2) * U32 * (size @ w.abs()))
    dw = (dz.T @ x, error.T @ x.abs() + 2 * (n + 66) * U32 * (size.T @ x.abs()))
    db = (dz.sum(0), (slope_error + torch.zeros_like(dz)).sum(0) + 2 * (n + 66) * U32 * dz.abs().sum(0))
    return dict(dx=dx, dw=dw, db=db)


def norm_forward(x, scale, shift, epsilon):
    """(y, mean, rstd) each with its bound.  The mean is off by at most w + 1 half steps of the mean magnitude; the centred values by that
    and a half step of theirs; the variance by w + 4 half steps and twice the mean's error squared (the sum of the centred values is
    zero); 1 / sqrt halves a relative error and adds two steps."""
    x, scale, shift = x.double(), scale.double(), shift.double()
    w = x.shape[1]
    mean = x.mean(1, keepdim=True)
    dmean = (w + 2) * U32 * x.abs().mean(1, keepdim=True)
    c = x - mean
    var = c.square().mean(1, keepdim=True)
    dvar = (w + 6) * U32 * var + 2 * dmean.square() + 2 * U32 * c.abs().mean(1, keepdim=True) * dmean
    rstd = 1 / (var + epsilon).sqrt()
    drstd = rstd * (0.5 * dvar / (var + epsilon) * 1.1 + 6 * U32)
    y = c * rstd * scale + shift
    dy = scale.abs() * (dmean * rstd + c.abs() * drstd) * 1.01 + 6 * U32 * ((c * rstd * scale).abs() + shift.abs())
    return (y, dy), (mean[:, 0], dmean[:, 0]), (rstd[:, 0], drstd[:, 0])


def norm_backward(x, mean, rstd, scale, dy, skip):
    """dict(dx, dscale, dshift) with bounds, for the statistics that are given: xh within three half steps and the cancellation of x - mean;
    means over w values within w + 4 half steps of the mean magnitude; a column's sum over n values within n + 66."""
    x, mean, rstd, scale, g = x.double(), mean.double()[:, None], rstd.double()[:, None], scale.double(), dy.double()
    n, w = x.shape
    xh = (x - mean) * rstd
    dxh = 4 * U32 * xh.abs()
    h = g * scale
    a, b = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    da = (w + 4) * U32 * h.abs().mean(1, keepdim=True)
    db = (w + 10) * U32 * (h * xh).abs().mean(1, keepdim=True)
    dx = rstd * (h - a - xh * b)
    size = h.abs() + a.abs() + (xh * b).abs()
    ddx = rstd * (da + xh.abs() * db + dxh * b.abs() + 6 * U32 * size)
    if skip is not None:
        dx = dx + skip.double()
        ddx = ddx + U32 * dx.abs()
    return dict(dx=(dx, ddx), dscale=((g * xh).sum(0), (2 * (n + 66) + 8) * U32 * (g * xh).abs().sum(0)), dshift=(g.sum(0), 2 * (n + 66) * U32 * g.abs().sum(0)))
