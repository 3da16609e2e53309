"""What the layers refuse, before anything is launched: no GPU needed (the addresses are never read)."""
import ctypes as C

import pytest
import torch

from neus2_amd import capi, layers
from neus2_amd.capi import N2Error

INVALID = 1
A, B, D, E, F, G, W = (0x10000000 * k for k in range(1, 8))


def lib():
    return capi.lib()


def refused(rc, text):
    assert rc == INVALID and text in lib().n2_last_error().decode(), (rc, lib().n2_last_error())


def accepted(rc):
    """Nothing to do, or the launch itself fails for want of a device: the checks have let it through."""
    assert rc != INVALID, lib().n2_last_error()


def linear(dtype=0, act=0, n=64, i=32, o=48, w=A, b=0, x=B, xs=None, r=0, rs=None, y=D, ys=None, z=0, zs=None, ws=W, nbytes=1 << 40):
    d = lambda s, width: width if s is None else s
    return lib().n2_linear_forward(None, dtype, act, n, i, o, w, b, x, d(xs, i), r, d(rs, o), y, d(ys, o), z, d(zs, o), ws, nbytes)


def linear_backward(dtype=0, act=2, n=64, i=32, o=48, w=A, x=B, xs=None, z=D, zs=None, dy=E, dys=None, dx=F, dxs=None, dw=G, db=G + 0x100000, mode=1, ws=W, nbytes=1 << 24):
    d = lambda s, width: width if s is None else s
    return lib().n2_linear_backward(None, dtype, act, n, i, o, w, x, d(xs, i), z, d(zs, o), dy, d(dys, o), dx, d(dxs, i), dw, db, mode, ws, nbytes)


def norm(dtype=0, weights=0, n=64, w=32, eps=1e-5, scale=A, shift=A + 64, x=B, xs=None, y=D, ys=None, mean=E, rstd=F):
    return lib().n2_layer_norm_forward(None, dtype, weights, n, w, eps, scale, shift, x, w if xs is None else xs, y, w if ys is None else ys, mean, rstd)


def norm_backward(dtype=0, weights=0, n=64, w=32, scale=A, x=B, xs=None, mean=D, rstd=D + 0x1000, dy=E, dys=None, skip=0, ss=None, dx=F, dxs=None, ds=G, db=G + 64, mode=1, ws=W, nbytes=1 << 24):
    d = lambda s: w if s is None else s
    return lib().n2_layer_norm_backward(None, dtype, weights, n, w, scale, x, d(xs), mean, rstd, dy, d(dys), skip, d(ss), dx, d(dxs), ds, db, mode, ws, nbytes)


def test_linear_forward_refuses():
    accepted(linear(n=0, x=0, y=0))
    for kw, text in ((dict(dtype=2), "neither"), (dict(dtype=7), "neither"), (dict(act=4), "activation"), (dict(act=-1), "activation"), (dict(i=0), "widths"), (dict(o=0), "widths"), (dict(i=65537), "widths"), (dict(n=1 << 31), "rows"),
                     (dict(w=0), "null"), (dict(x=0), "null"), (dict(y=0), "null"), (dict(xs=31), "the input"), (dict(ys=47), "the output"), (dict(r=E, rs=40), "residual"),
                     (dict(z=E, zs=1), "saved"), (dict(xs=1 << 61), "the input"),
                     (dict(y=B), "overlaps"), (dict(y=A), "overlaps"), (dict(y=B + 64 * 64 - 2), "overlaps"), (dict(z=D), "overlaps"), (dict(z=B), "overlaps"), (dict(r=D, rs=50), "overlaps"),
                     (dict(r=D + 2), "overlaps"), (dict(b=D + 100), "overlaps"), (dict(x=D, xs=100, ys=100), "overlaps"), (dict(x=D, xs=100, y=D + 62, ys=100), "overlaps")):
        refused(linear(**kw), text)


def test_linear_backward_refuses():
    need = lib().n2_linear_backward_workspace_bytes(64, 32, 48)
    assert need > 0
    for kw, text in ((dict(dtype=2), "neither"), (dict(act=9), "activation"), (dict(mode=3), "mode"), (dict(o=1 << 20), "widths"), (dict(w=0), "null"), (dict(x=0), "null"), (dict(dy=0), "null"),
                     (dict(z=0), "null"), (dict(zs=47), "saved"), (dict(dys=47), "output's gradient"), (dict(dxs=31), "input's gradient"), (dict(xs=3), "the input"),
                     (dict(ws=0), "workspace"), (dict(ws=W + 8), "workspace"), (dict(nbytes=need - 1), "workspace"), (dict(dx=B), "overlaps"), (dict(dx=E), "overlaps"), (dict(dw=A), "overlaps"),
                     (dict(db=G), "overlaps"), (dict(ws=E), "overlaps"), (dict(dx=W), "overlaps"), (dict(z=F), "overlaps")):
        refused(linear_backward(**kw), text)


def test_layer_norm_refuses():
    accepted(norm(n=0, x=0, y=0))
    for kw, text in ((dict(dtype=3), "type"), (dict(dtype=0, weights=1), "type"), (dict(dtype=2, weights=0), "type"), (dict(w=0), "width"), (dict(w=16385), "width"), (dict(eps=0.0), "epsilon"),
                     (dict(eps=float("nan")), "epsilon"), (dict(eps=float("inf")), "epsilon"), (dict(x=0), "null"), (dict(scale=0), "null"), (dict(shift=0), "null"), (dict(y=0), "null"),
                     (dict(xs=31), "stride"), (dict(ys=31), "stride"), (dict(xs=1 << 62), "beyond"), (dict(y=B), "overlaps"), (dict(y=A), "overlaps"), (dict(mean=F), "overlaps"), (dict(rstd=D), "overlaps")):
        refused(norm(**kw), text)
    need = lib().n2_layer_norm_workspace_bytes(0, 64, 32)
    assert need > 0
    for kw, text in ((dict(dtype=5), "type"), (dict(mode=-1), "mode"), (dict(ds=0), "null"), (dict(db=0), "null"), (dict(mean=0), "null"), (dict(rstd=0), "null"), (dict(dy=0), "null"),
                     (dict(dys=31), "stride"), (dict(skip=G + 0x10000, ss=31), "stride"), (dict(dxs=31), "stride"), (dict(ws=0), "workspace"), (dict(ws=W + 4), "workspace"),
                     (dict(nbytes=need - 1), "workspace"), (dict(dx=B), "overlaps"), (dict(dx=E), "overlaps"), (dict(skip=F, ss=40), "overlaps"), (dict(ds=G + 64, db=G + 66), "overlaps"),
                     (dict(ws=F), "overlaps"), (dict(ds=A), "overlaps")):
        refused(norm_backward(**kw), text)


def create(tensors, table=W, nbytes=1 << 30, count=None):
    arr = (capi.GradientTensor * max(1, len(tensors)))(*[capi.GradientTensor(*t) for t in tensors])
    h = C.c_void_p()
    rc = lib().n2_gradients_create(None, len(tensors) if count is None else count, arr, table, nbytes, C.byref(h))
    assert rc == 0 or not h.value
    return rc, h


def test_gradients_refuse():
    for tensors, text in (([(A, A, 8, 3)], "type"), ([(0, A, 8, 0)], "null"), ([(A, 0, 8, 0)], "null"), ([(A + 1, A + 1, 8, 0)], "aligned"), ([(A + 2, A + 2, 8, 2)], "aligned"),
                          ([(A, A, 8, 0), (A, A, 8, 0)], "overlap"), ([(A, A, 8, 0), (A + 14, A + 14, 8, 0)], "overlap"), ([(A, A + 2, 8, 0)], "overlap"), ([(A, B, 8, 0), (D, A, 8, 0)], "overlap"),
                          ([(A, A, 1 << 50, 0)], "values")):
        refused(create(tensors)[0], text)
    refused(create([(A, A, 8, 0)], table=0)[0], "table")
    refused(create([(A, A, 8, 0)], table=W + 8)[0], "table")
    refused(create([(A, A, 8193, 0)], nbytes=31)[0], "table")
    rc, h = create([(0, 0, 0, 0)])  # no values: nothing to upload
    assert rc == 0
    L = lib()
    ws = capi.GRADIENTS_WORKSPACE_BYTES
    refused(L.n2_gradients_clip(h, None, -1.0, 1.0, A, W, ws), "max_norm")
    refused(L.n2_gradients_clip(h, None, float("nan"), 1.0, A, W, ws), "max_norm")
    refused(L.n2_gradients_clip(h, None, 1.0, 0.0, A, W, ws), "loss_scale")
    refused(L.n2_gradients_clip(h, None, 1.0, float("inf"), A, W, ws), "loss_scale")
    refused(L.n2_gradients_clip(h, None, 1.0, 1.0, None, W, ws), "null")
    refused(L.n2_gradients_norm(h, None, 1.0, A, W, ws - 1), "workspace")
    refused(L.n2_gradients_norm(h, None, 1.0, A, W + 8, ws), "workspace")
    refused(L.n2_gradients_norm(None, None, 1.0, A, W, ws), "null")
    L.n2_gradients_destroy(h)
    L.n2_gradients_destroy(None)


def test_workspaces():
    L = lib()
    assert L.n2_linear_backward_workspace_bytes(0, 8, 8) == 0 and L.n2_linear_backward_workspace_bytes(8, 0, 8) == 0 and L.n2_layer_norm_workspace_bytes(0, 8, 16385) == 0
    # dz, and fp32 sums that stay small beside the operands
    for n, i, o in ((1, 1, 1), (1 << 18, 256, 256), (5003, 320, 257), (16384, 2048, 2048), (1 << 20, 64, 64)):
        assert L.n2_linear_backward_workspace_bytes(n, i, o) <= 2 * n * (o + 7) + 4 * 1024 * (o + 4) + 4 * 600 * max(i * o, 128 * 128) + 64


def test_python_refuses():
    for kw in (dict(activation="Sine"), dict(dtype=torch.float32), dict(n_input_dims=0), dict(n_output_dims=65537)):
        with pytest.raises(N2Error):
            layers.Linear(**{**dict(n_input_dims=8, n_output_dims=8), **kw})
    for args in ((0,), (16385,), (8, 0.0), (8, float("nan")), (8, 1e-5, torch.float64), (8, 1e-5, torch.float32, torch.float16), (8, 1e-5, torch.float16, torch.bfloat16)):
        with pytest.raises(N2Error):
            layers.LayerNorm(*args)
    lin = layers.Linear(8, 4)
    assert lin.n_params() == 36 and layers.Linear(8, 4, bias=False).n_params() == 32 and layers.LayerNorm(8).n_params() == 16
    x = torch.zeros(2, 8, dtype=torch.float16)
    for call in (lambda: lin.forward(x), lambda: lin.set_params(torch.zeros(36, dtype=torch.float16)), lambda: layers.LayerNorm(8).forward(x), lambda: layers.GradientClip([x])):
        with pytest.raises(N2Error):
            call()
