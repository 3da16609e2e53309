"""The layers of any width and the clipping on the GPU, against their formulas in 64 bits (tests/layers_ref.py)."""
import math

import pytest
import torch

import layers_ref as ref

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]
KINDS = ["None", "ReLU", "SiLU", "GELU"]


def _rows(gen, n, w, dtype, extra=0, first=0, scale=1.0):
    """[n, w] values inside a wider matrix: `extra` columns beside them, starting at element `first`."""
    whole = (torch.randn(n, w + extra, generator=gen) * scale).to(dtype).cuda() if n else torch.empty(0, w + extra, dtype=dtype, device="cuda")
    return whole[:, first:first + w]


def _canvas(n, w, dtype, extra, first):
    """An output inside a wider and longer matrix of marks, and the check that only the output was written."""
    whole = torch.full((n + 3, w + extra), 77.0, dtype=dtype, device="cuda")
    out = whole[:n, first:first + w]

    def check():
        rest = whole.clone()
        rest[:n, first:first + w] = 77.0
        assert bool((rest == 77.0).all()), "written outside the output"
    return out, check


def _linear(gen, i, o, kind, bias, dtype):
    from neus2_amd.layers import Linear
    op = Linear(i, o, activation=kind, bias=bias, dtype=dtype)
    w = torch.randn(o * i, generator=gen) / math.sqrt(i)
    params = torch.cat([w, torch.randn(o, generator=gen) * 0.3] if bias else [w]).to(dtype).cuda()
    op.set_params(params, torch.zeros_like(params))
    return op, params[:o * i].view(o, i), params[o * i:] if bias else None


# rows, in, out, extra columns, first column
SHAPES = [(1, 1, 1, 0, 0), (1, 256, 256, 0, 0), (2, 3, 5, 3, 1), (16, 512, 96, 8, 8), (17, 200, 33, 0, 0), (64, 64, 64, 0, 0), (65, 63, 129, 1, 1), (128, 128, 128, 0, 0),
          (130, 257, 31, 0, 0), (300, 72, 257, 8, 0), (513, 320, 257, 7, 3), (1000, 40, 24, 0, 0), (257, 1032, 264, 0, 0), (1500, 16, 8, 0, 0), (700, 500, 300, 4, 4), (20, 2056, 64, 0, 0), (33, 1000, 136, 8, 8)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,i,o,extra,first", SHAPES)
def test_linear_forward(n, i, o, extra, first, kind, dtype):
    gen = torch.Generator().manual_seed(n * 31 + i + o)
    residual = (n + i) % 2 == 0
    op, w, b = _linear(gen, i, o, kind, bias=o % 3 != 0, dtype=dtype)
    x = _rows(gen, n, i, dtype, extra, first)
    r = _rows(gen, n, o, dtype, extra, first) if residual else None
    out, check = _canvas(n, o, dtype, extra, first)
    y, z = op.forward(x, residual=r, want_pre_activation=True, out=out)
    ye, ze, dy, dz = ref.linear_forward(x, w, b, r, kind)
    ref.within(y, ye, dy, "y")
    ref.within(z, ze, dz, "z")
    check()
    assert torch.equal(op.forward(x, residual=r)[0], y)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,i,o,extra,first", SHAPES)
def test_linear_backward(n, i, o, extra, first, kind, dtype):
    from neus2_amd.capi import GRAD_ACCUMULATE, GRAD_IGNORE
    gen = torch.Generator().manual_seed(n * 17 + i + o)
    op, w, b = _linear(gen, i, o, kind, bias=True, dtype=dtype)
    x, dy = _rows(gen, n, i, dtype, extra, first), _rows(gen, n, o, dtype, extra, first)
    z = _rows(gen, n, o, dtype, extra, first) if kind != "None" else None
    e = ref.linear_backward(x, w, z, dy, kind)
    out, check = _canvas(n, i, dtype, extra, first)
    op._grads.fill_(float("nan"))  # overwritten, whatever stands there
    op.backward(x, z, dy, out=out)
    check()
    grads = op._grads.clone()
    ref.within(out, *e["dx"], "dx")
    ref.within(grads[:o * i].view(o, i), *e["dw"], "dw")
    ref.within(grads[o * i:], *e["db"], "db")
    # the parts on their own give the same bits
    op._grads.zero_()
    assert op.backward(x, z, dy, want_input_grad=False) is None and torch.equal(op._grads, grads)
    op._grads.fill_(5.0)
    assert torch.equal(op.backward(x, z, dy, mode=GRAD_IGNORE), out) and bool((op._grads == 5.0).all())
    # added to what is there, rounded once
    before = (torch.randn(op.n_params(), generator=gen)).to(dtype).cuda()
    op._grads.copy_(before)
    op.backward(x, z, dy, mode=GRAD_ACCUMULATE)
    old = before.double()
    ref.within(op._grads[:o * i].view(o, i), e["dw"][0] + old[:o * i].view(o, i), e["dw"][1] + ref.U32 * (e["dw"][0].abs() + old[:o * i].view(o, i).abs()), "dw added")
    ref.within(op._grads[o * i:], e["db"][0] + old[o * i:], e["db"][1] + ref.U32 * (e["db"][0].abs() + old[o * i:].abs()), "db added")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,i,o", [(20000, 24, 16), (9001, 130, 257), (4096, 256, 256), (2048, 512, 768)])
def test_linear_backward_sums_many_rows(n, i, o, dtype):
    """Rows dealt out to several workgroups for each tile of the weights' gradient; twice the same bits."""
    gen = torch.Generator().manual_seed(n)
    op, w, b = _linear(gen, i, o, "GELU", bias=True, dtype=dtype)
    x, z, dy = _rows(gen, n, i, dtype), _rows(gen, n, o, dtype), _rows(gen, n, o, dtype, scale=0.01)
    dx = op.backward(x, z, dy)
    grads = op._grads.clone()
    e = {k: v for k, v in ref.linear_backward(x, w, z, dy, "GELU").items()}
    ref.within(dx, *e["dx"], "dx")
    ref.within(grads[:o * i].view(o, i), *e["dw"], "dw")
    ref.within(grads[o * i:], *e["db"], "db")
    op._grads.zero_()
    assert torch.equal(op.backward(x, z, dy), dx) and torch.equal(op._grads, grads)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,i,o,residual,kind", [(49152, 256, 256, True, "None"), (49155, 64, 64, False, "SiLU"), (50001, 200, 136, True, "GELU"), (60000, 8, 8, False, "None"), (50000, 72, 256, True, "ReLU"),
                                                 (70001, 128, 24, False, "GELU"), (49200, 256, 64, True, "SiLU"), (49200, 40, 128, True, "None"), (49153, 36, 68, True, "None")])
def test_linear_forward_of_many_rows(n, i, o, residual, kind, dtype):
    """Narrow layers of many rows keep their weights in LDS and pass over the rows: widths inside their steps, ragged last rows, the residual in place."""
    gen = torch.Generator().manual_seed(n + i)
    op, w, b = _linear(gen, i, o, kind, bias=i != 64, dtype=dtype)
    x, r = _rows(gen, n, i, dtype, 8, 8), _rows(gen, n, o, dtype) if residual else None
    out, check = _canvas(n, o, dtype, 16, 8)
    y, z = op.forward(x, residual=r, want_pre_activation=True, out=out)
    ye, ze, dy, dz = ref.linear_forward(x, w, b, r, kind)
    ref.within(y, ye, dy, "y")
    ref.within(z, ze, dz, "z")
    check()
    if residual:
        op.forward(x, residual=r, out=r)
        assert torch.equal(r, y)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,i,o,kind,mode", [(49152, 256, 256, "ReLU", 1), (49155, 64, 64, "SiLU", 2), (50001, 200, 136, "GELU", 1), (60000, 8, 8, "None", 1), (50000, 72, 256, "None", 2), (70001, 24, 128, "ReLU", 1),
                                             (49200, 256, 64, "SiLU", 0), (49153, 36, 68, "GELU", 1), (49160, 33, 64, "ReLU", 1)])
def test_linear_backward_of_many_rows(n, i, o, kind, mode, dtype):
    """Narrow layers of many rows form dz, its column sums and dx in one pass; the parts on their own, the last rows ragged."""
    gen = torch.Generator().manual_seed(n + o)
    op, w, b = _linear(gen, i, o, kind, bias=True, dtype=dtype)
    x, dy = _rows(gen, n, i, dtype), _rows(gen, n, o, dtype, 8, 8, scale=0.02)
    z = _rows(gen, n, o, dtype, 8, 0) if kind != "None" else None
    out, check = _canvas(n, i, dtype, 8, 8)
    before = torch.randn(op.n_params(), generator=gen).to(dtype).cuda()
    op._grads.copy_(before)
    op.backward(x, z, dy, mode=mode, out=out)
    check()
    e = ref.linear_backward(x, w, z, dy, kind)
    ref.within(out, *e["dx"], "dx")
    old = before.double() * (mode == 2)
    if mode == 0:
        assert torch.equal(op._grads, before)
    else:
        for name, got, was in (("dw", op._grads[:o * i].view(o, i), old[:o * i].view(o, i)), ("db", op._grads[o * i:], old[o * i:])):
            ref.within(got, e[name][0] + was, e[name][1] + ref.U32 * (e[name][0].abs() + was.abs()), name)
    first = op._grads.clone()
    op._grads.copy_(before)
    assert torch.equal(op.backward(x, z, dy, mode=mode), out) and torch.equal(op._grads, first)


@pytest.mark.parametrize("dtype", HALVES)
def test_linear_of_no_rows(dtype):
    from neus2_amd.capi import GRAD_ACCUMULATE
    gen = torch.Generator().manual_seed(1)
    op, w, b = _linear(gen, 40, 24, "SiLU", bias=True, dtype=dtype)
    x, g = torch.empty(0, 40, dtype=dtype, device="cuda"), torch.empty(0, 24, dtype=dtype, device="cuda")
    y, z = op.forward(x, want_pre_activation=True)
    assert y.shape == z.shape == (0, 24)
    op._grads.fill_(3.0)
    op.backward(x, z, g, mode=GRAD_ACCUMULATE)
    assert bool((op._grads == 3.0).all())
    assert op.backward(x, z, g).shape == (0, 40) and not bool(op._grads.any())


@pytest.mark.parametrize("n", [1, 5, 16, 40, 300])
def test_infinities_and_nans_stay_in_their_rows(n):
    """A row of no numbers, beside rows of numbers and behind the last row of the batch, changes no other row."""
    gen = torch.Generator().manual_seed(n)
    op, w, b = _linear(gen, 72, 40, "None", bias=True, dtype=torch.float16)
    whole = _rows(gen, n + 2, 72, torch.float16)
    clean = op.forward(whole[:n].clone())[0]
    whole[n:] = float("nan")
    assert torch.equal(op.forward(whole[:n])[0], clean)
    if n > 1:
        whole[n // 2] = float("inf")
        got = op.forward(whole[:n])[0]
        others = torch.arange(n) != n // 2
        assert torch.equal(got[others], clean[others]) and not bool(torch.isfinite(got[n // 2]).any())


def test_columns_behind_a_row_are_not_read():
    """What stands between a row's end and the next row's start may be anything."""
    gen = torch.Generator().manual_seed(3)
    for i, o, first in ((72, 40, 0), (65, 33, 1), (8, 8, 8)):
        op, w, b = _linear(gen, i, o, "ReLU", bias=True, dtype=torch.bfloat16)
        x, z, dy = (_rows(gen, 90, c, torch.bfloat16) for c in (i, o, o))
        wide = []
        for t in (x, z, dy):
            m = torch.full((90, t.shape[1] + first + 5), float("nan"), dtype=torch.bfloat16, device="cuda")
            m[:, first:first + t.shape[1]] = t
            wide.append(m[:, first:first + t.shape[1]])
        assert torch.equal(op.forward(wide[0])[0], op.forward(x)[0])
        dx = op.backward(x, z, dy)
        grads = op._grads.clone()
        assert torch.equal(op.backward(*wide), dx) and torch.equal(op._grads, grads)


@pytest.mark.parametrize("n,i,o", [(40, 72, 24), (300, 200, 136), (3000, 256, 256), (50000, 64, 128)])
def test_linear_without_bias(n, i, o):
    gen = torch.Generator().manual_seed(n + 1)
    for dtype, kind in ((torch.float16, "ReLU"), (torch.bfloat16, "None")):
        op, w, b = _linear(gen, i, o, kind, bias=False, dtype=dtype)
        assert b is None and op.n_params() == i * o
        x, dy = _rows(gen, n, i, dtype), _rows(gen, n, o, dtype, scale=0.1)
        y, z = op.forward(x, want_pre_activation=True)
        ye, _, error, _ = ref.linear_forward(x, w, None, None, kind)
        ref.within(y, ye, error, "y")
        dx = op.backward(x, z, dy)
        e = ref.linear_backward(x, w, z, dy, kind)
        ref.within(dx, *e["dx"], "dx")
        ref.within(op._grads.view(o, i), *e["dw"], "dw")


@pytest.mark.parametrize("n,i,o,extra,first,kind", [(100003, 256, 256, 0, 0, "ReLU"), (100003, 256, 257, 0, 0, "None"), (100010, 256, 256, 9, 1, "SiLU"), (33001, 512, 1024, 8, 8, "GELU"), (600001, 64, 64, 0, 0, "ReLU")])
def test_linear_backward_of_more_than_the_cache_holds(n, i, o, extra, first, kind):
    """dz formed by loads that pass by the last-level cache: whole vectors, odd widths, rows that start anywhere."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    make = lambda w, scale: (torch.randn(n, w + extra, generator=gen, device="cuda") * scale).half()[:, first:first + w]
    op, w, b = _linear(torch.Generator().manual_seed(n), i, o, kind, bias=True, dtype=torch.float16)
    x, z, dy = make(i, 1.0), make(o, 1.0) if kind != "None" else None, make(o, 0.01)
    dx = op.backward(x, z, dy)
    e = ref.linear_backward(x, w, z, dy, kind)
    ref.within(dx, *e["dx"], "dx")
    ref.within(op._grads[:o * i].view(o, i), *e["dw"], "dw")
    ref.within(op._grads[o * i:], *e["db"], "db")
    first_grads = op._grads.clone()
    assert torch.equal(op.backward(x, z, dy), dx) and torch.equal(op._grads, first_grads)


@pytest.mark.parametrize("n", [2, 40])
def test_rows_a_long_way_apart(n):
    """Strides beyond the 32-bit offsets of a tile's rows: 2^22 values and more from row to row."""
    gen = torch.Generator().manual_seed(n + 5)
    stride, i, o = (1 << 22) + 8, 72, 136
    op, w, b = _linear(gen, i, o, "SiLU", bias=True, dtype=torch.bfloat16)
    norm, *_ = _norm(gen, i, torch.bfloat16, torch.float32)
    x, z, dy = (_rows(gen, n, c, torch.bfloat16) for c in (i, o, o))
    whole = torch.full((n, stride), float("nan"), dtype=torch.bfloat16, device="cuda")
    at = 0
    wide = []
    for t in (x, z, dy, x, z):  # (the last two: outputs)
        view = whole[:, at:at + t.shape[1]]
        at += t.shape[1] + 8
        view.copy_(t)
        wide.append(view)
    far_x, far_z, far_dy, out_x, out_y = wide
    y = op.forward(x, residual=dy)[0]
    assert torch.equal(op.forward(far_x, residual=far_dy, out=out_y)[0], y)
    dx = op.backward(x, z, dy)
    grads = op._grads.clone()
    assert torch.equal(op.backward(far_x, far_z, far_dy, out=out_x), dx)
    e = ref.linear_backward(x, w, z, dy, "SiLU")
    ref.within(out_x, *e["dx"], "dx")
    ref.within(op._grads[:o * i].view(o, i), *e["dw"], "dw")
    assert torch.equal(op._grads[o * i:], grads[o * i:])
    h, ctx = norm.forward(x, want_ctx=True)
    assert torch.equal(norm.forward(far_x, out=out_x)[0], h)
    dh = norm.backward(ctx, x, h)
    assert torch.equal(norm.backward(ctx, far_x, out_x, out=out_y[:, :i]), dh)
    assert torch.equal(far_x, x) and torch.equal(far_z, z) and torch.equal(far_dy, dy)


@pytest.mark.parametrize("n,i,o", [(1, 72, 40), (16, 72, 264), (50, 200, 136), (300, 328, 72), (3000, 264, 520), (49155, 72, 200), (49153, 256, 64), (50000, 264, 72)])
def test_nothing_around_a_matrix_is_read(n, i, o):
    """No numbers beside the columns and behind the last row of every operand, at strides of whole vectors."""
    gen = torch.Generator().manual_seed(n + i + o)
    op, w, b = _linear(gen, i, o, "ReLU", bias=True, dtype=torch.bfloat16)
    x, z, dy, r = (_rows(gen, n, c, torch.bfloat16) for c in (i, o, o, o))
    wide = []
    for t in (x, z, dy, r):
        m = torch.full((n + 70, t.shape[1] + 64), float("nan"), dtype=torch.bfloat16, device="cuda")
        m[:n, :t.shape[1]] = t
        wide.append(m[:n, :t.shape[1]])
    assert torch.equal(op.forward(wide[0], residual=wide[3])[0], op.forward(x, residual=r)[0])
    assert torch.equal(op.forward(wide[0])[0], op.forward(x)[0])
    dx = op.backward(x, z, dy)
    grads = op._grads.clone()
    assert torch.equal(op.backward(*wide[:3]), dx) and torch.equal(op._grads, grads)
    from neus2_amd.capi import GRAD_IGNORE
    assert torch.equal(op.backward(*wide[:3], mode=GRAD_IGNORE), dx)
    norm, *_ = _norm(gen, i, torch.bfloat16, torch.float32)
    h, ctx = norm.forward(x, want_ctx=True)
    assert torch.equal(norm.forward(wide[0])[0], h)
    dh = norm.backward(ctx, x, x)
    grads = norm._grads.clone()
    assert torch.equal(norm.backward(ctx, wide[0], wide[0]), dh) and torch.equal(norm._grads, grads)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", HALVES)
def test_activations_over_the_types_whole_range(kind, dtype):
    """Every finite value of the type through the epilogue and through the slope, one layer of a single weight 1: no overflow on the way
    turns a finite result into none."""
    from neus2_amd.layers import Linear
    values = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    values = values[torch.isfinite(values)].cuda()[:, None]
    op = Linear(1, 1, activation=kind, bias=False, dtype=dtype)
    one = torch.ones(1, dtype=dtype, device="cuda")
    op.set_params(one, torch.zeros_like(one))
    y, z = op.forward(values, want_pre_activation=True)
    assert torch.equal(z.float(), values.float())
    ye, _, error, _ = ref.linear_forward(values, one[:, None], None, None, kind)
    ref.within(y, ye, error, "y")
    dy = torch.full_like(values, 0.5)
    dx = op.backward(values, z, dy, mode=0)
    e = ref.linear_backward(values, one[:, None], values, dy, kind)
    ref.within(dx, *e["dx"], "dx")


@pytest.mark.parametrize("n,i,o", [(3, 72, 40), (100, 256, 136), (5000, 64, 64), (50000, 64, 128)])
def test_parameters_anywhere_in_a_larger_vector(n, i, o):
    """A layer's parameters and gradients inside the vector of a whole network, at odd places: what stands beside them stays."""
    from neus2_amd.layers import LayerNorm, Linear
    gen = torch.Generator().manual_seed(n + 9)
    dtype = torch.float16
    lin, norm = Linear(i, o, activation="SiLU", dtype=dtype), LayerNorm(i, dtype=dtype)
    at, after = 1, 1 + lin.n_params() + 2
    size = after + norm.n_params() + 1
    params = (torch.randn(size, generator=gen) * 0.1).to(dtype).cuda()
    grads = torch.full((size,), 7.0, dtype=dtype, device="cuda")
    lin.set_params(params[at:at + lin.n_params()], grads[at:at + lin.n_params()])
    norm.set_params(params[after:after + norm.n_params()], grads[after:after + norm.n_params()])
    x, dy = _rows(gen, n, i, dtype), _rows(gen, n, o, dtype, scale=0.05)
    h, ctx = norm.forward(x, want_ctx=True)
    y, z = lin.forward(h, want_pre_activation=True)
    w, b = params[at:at + i * o].view(o, i), params[at + i * o:at + i * o + o]
    scale, shift = params[after:after + i], params[after + i:after + 2 * i]
    ref.within(h, *ref.norm_forward(x, scale, shift, 1e-5)[0], "h")
    ye, _, error, _ = ref.linear_forward(h, w, b, None, "SiLU")
    ref.within(y, ye, error, "y")
    dh = lin.backward(h, z, dy)
    e = ref.linear_backward(h, w, z, dy, "SiLU")
    ref.within(dh, *e["dx"], "dh")
    ref.within(grads[at:at + i * o].view(o, i), *e["dw"], "dw")
    ref.within(grads[at + i * o:at + i * o + o], *e["db"], "db")
    dx = norm.backward(ctx, x, dh)
    e = ref.norm_backward(x, *ctx, scale, dh, None)
    ref.within(dx, *e["dx"], "dx")
    ref.within(grads[after:after + i], *e["dscale"], "dscale")
    ref.within(grads[after + i:after + 2 * i], *e["dshift"], "dshift")
    beside = torch.cat([grads[:at], grads[at + lin.n_params():after], grads[after + norm.n_params():]])
    assert beside.numel() == 4 and bool((beside == 7.0).all())


@pytest.mark.parametrize("n,i,o,extra,first", [(50001, 513, 510, 0, 0), (100001, 255, 127, 2, 1), (20011, 1003, 300, 0, 0), (3001, 2047, 65, 5, 5), (18, 1, 3, 0, 0), (40, 2, 1, 0, 0)])
def test_odd_rows_in_tiles_of_every_size(n, i, o, extra, first):
    """Rows that start anywhere, through registers: the last piece of the matrix ends with it, what stands between rows is cut off."""
    gen = torch.Generator().manual_seed(n + i)
    op, w, b = _linear(gen, i, o, "GELU", bias=True, dtype=torch.bfloat16)
    whole = torch.full((n, i + extra), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = whole[:, first:first + i]
    x.copy_(torch.randn(n, i, generator=gen))
    y, z = op.forward(x, want_pre_activation=True)
    ye, ze, error, z_error = ref.linear_forward(x, w, b, None, "GELU")
    ref.within(y, ye, error, "y")
    ref.within(z, ze, z_error, "z")
    dy = _rows(gen, n, o, torch.bfloat16, scale=0.05)
    dx = op.backward(x, z, dy)
    e = ref.linear_backward(x, w, z, dy, "GELU")
    ref.within(dx, *e["dx"], "dx")
    ref.within(op._grads[:o * i].view(o, i), *e["dw"], "dw")
    ref.within(op._grads[o * i:], *e["db"], "db")


def test_residual_in_place_and_columns_of_one_matrix():
    gen = torch.Generator().manual_seed(4)
    op, w, b = _linear(gen, 64, 64, "SiLU", bias=True, dtype=torch.float16)
    x, r = _rows(gen, 200, 64, torch.float16), _rows(gen, 200, 64, torch.float16)
    y = op.forward(x, residual=r)[0]
    stream = r.clone()
    assert op.forward(x, residual=stream, out=stream)[0] is stream and torch.equal(stream, y)
    both = torch.cat([x, r], 1)  # input and output side by side
    op.forward(both[:, :64], residual=both[:, 64:], out=both[:, 64:])
    assert torch.equal(both[:, 64:], y) and torch.equal(both[:, :64], x)


@pytest.mark.parametrize("kind", KINDS)
def test_linear_gradients_against_differences(kind):
    """<dx, d> against (L(x + h d) - L(x - h d)) / 2h of the forward pass in 64 bits, L = sum(dy * y), and the same for the weights:
    off by the gradient's own bound along d and the differences' h^2 / 6 times the third derivative (activations: below 2)."""
    dtype = torch.float16
    gen = torch.Generator().manual_seed(8)
    op, w, b = _linear(gen, 24, 20, kind, bias=True, dtype=dtype)
    x, dy = _rows(gen, 33, 24, dtype), _rows(gen, 33, 20, dtype)
    z = (x.double() @ w.double().T + b.double())
    if kind == "ReLU":  # (differences across the corner say nothing)
        x = x[(z.abs() > 1e-2).all(1)]
        dy = dy[:x.shape[0]]
        z = (x.double() @ w.double().T + b.double())
    zq = z.to(dtype)
    dx = op.backward(x, zq, dy)
    dw, db = op._grads[:480].view(20, 24), op._grads[480:]
    e = ref.linear_backward(x, w, zq, dy, kind)
    h = 1e-5
    L = lambda x_, w_, b_: float((dy.double() * ref.act(x_ @ w_.T + b_, kind)).sum())
    for name, got, at in (("dx", dx, 0), ("dw", dw, 1), ("db", db, 2)):
        parts = [x.double(), w.double(), b.double()]
        d = torch.randn(parts[at].shape, generator=gen).double().cuda()
        up, down = list(parts), list(parts)
        up[at], down[at] = parts[at] + h * d, parts[at] - h * d
        numeric = (L(*up) - L(*down)) / (2 * h)
        bound = e[name][1] + ref.half_step(dtype) * (e[name][0].abs() + e[name][1]) + ref.least(dtype)
        # (the saved z is rounded: the slope moves by half a step of z times a curvature below 1.2)
        curvature = 0.0 if kind in ("None", "ReLU") else 1.2
        moved = curvature * (ref.half_step(dtype) * z.abs()) * dy.double().abs()
        turned = {"dx": lambda: moved @ w.double().abs(), "dw": lambda: moved.T @ x.double().abs(), "db": lambda: moved.sum(0)}[name]()
        third = 0.0 if curvature == 0.0 else 2 * h * h / 6 * float((dy.double().abs() * (x.double().abs() @ w.double().abs().T + x.double().abs().sum(1, True) + w.double().abs().sum(1) + 1) ** 3).sum()) * 64
        assert abs(float((got.double() * d).sum()) - numeric) <= float(((bound + turned) * d.abs()).sum()) + third + 1e-7 * abs(numeric), name


# ---------------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------------
TYPES = [(torch.float16, torch.float16), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]
NORMS = [(1, 1, 0, 0), (3, 2, 3, 1), (1000, 64, 0, 0), (257, 63, 1, 1), (33, 129, 0, 0), (64, 256, 8, 8), (50, 257, 0, 0), (40, 1000, 8, 0), (21, 1537, 0, 0), (9, 2048, 0, 0), (7, 4097, 3, 2),
         (5, 8192, 0, 0), (3, 16384, 0, 0), (2100, 24, 0, 0)]


def _norm(gen, w, dtype, weights):
    from neus2_amd.layers import LayerNorm
    op = LayerNorm(w, dtype=dtype, param_dtype=weights)
    params = torch.cat([1 + 0.2 * torch.randn(w, generator=gen), 0.3 * torch.randn(w, generator=gen)]).to(weights).cuda()
    op.set_params(params, torch.zeros_like(params))
    return op, params[:w], params[w:]


@pytest.mark.parametrize("dtype,weights", TYPES)
@pytest.mark.parametrize("n,w,extra,first", NORMS)
def test_norm_forward_and_backward(n, w, extra, first, dtype, weights):
    from neus2_amd.capi import GRAD_ACCUMULATE, GRAD_IGNORE
    gen = torch.Generator().manual_seed(n + w)
    op, scale, shift = _norm(gen, w, dtype, weights)
    x = _rows(gen, n, w, dtype, extra, first)
    out, check = _canvas(n, w, dtype, extra, first)
    y, (mean, rstd) = op.forward(x, want_ctx=True, out=out)
    ye, me, se = ref.norm_forward(x, scale, shift, 1e-5)
    ref.within(y, *ye, "y")
    ref.within(mean, *me, "mean")
    ref.within(rstd, *se, "rstd")
    check()
    assert torch.equal(op.forward(x)[0], y)
    dy, skip = _rows(gen, n, w, dtype, extra, first), _rows(gen, n, w, dtype, extra, first) if w % 2 else None
    e = ref.norm_backward(x, mean, rstd, scale, dy, skip)
    dx, check = _canvas(n, w, dtype, extra, first)
    op._grads.fill_(float("nan"))
    op.backward((mean, rstd), x, dy, dL_dskip=skip, out=dx)
    check()
    grads = op._grads.clone()
    ref.within(dx, *e["dx"], "dx")
    ref.within(grads[:w], *e["dscale"], "dscale")
    ref.within(grads[w:], *e["dshift"], "dshift")
    assert op.backward((mean, rstd), x, dy, want_input_grad=False) is None and torch.equal(op._grads, grads)
    op._grads.fill_(2.0)
    assert torch.equal(op.backward((mean, rstd), x, dy, dL_dskip=skip, mode=GRAD_IGNORE), dx) and bool((op._grads == 2.0).all())
    op.backward((mean, rstd), x, dy, mode=GRAD_ACCUMULATE)
    for name, got in (("dscale", op._grads[:w]), ("dshift", op._grads[w:])):
        ref.within(got, e[name][0] + 2.0, e[name][1] + ref.U32 * (e[name][0].abs() + 2.0), name + " added")


def test_norm_of_many_rows():
    gen = torch.Generator().manual_seed(6)
    op, scale, shift = _norm(gen, 256, torch.float16, torch.float16)
    x, dy, skip = (_rows(gen, 30011, 256, torch.float16) for _ in range(3))
    y, ctx = op.forward(x, want_ctx=True)
    ref.within(y, *ref.norm_forward(x, scale, shift, 1e-5)[0], "y")
    dx = op.backward(ctx, x, dy, dL_dskip=skip)
    e = ref.norm_backward(x, *ctx, scale, dy, skip)
    ref.within(dx, *e["dx"], "dx")
    ref.within(op._grads[:256], *e["dscale"], "dscale")
    ref.within(op._grads[256:], *e["dshift"], "dshift")
    into = skip.clone()  # the gradient stream in place
    assert op.backward(ctx, x, dy, dL_dskip=into, out=into) is into and torch.equal(into, dx)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_norm_of_rows_far_from_zero_and_of_equal_values(dtype):
    """The variance comes of the centred values: a mean a thousand times the deviation takes nothing from it.  Equal values have none."""
    gen = torch.Generator().manual_seed(7)
    op, scale, shift = _norm(gen, 96, dtype, torch.float32)
    x = (torch.randn(20, 96, generator=gen) + 1000).to(dtype).cuda()
    x[3] = 12.0
    y, (mean, rstd) = op.forward(x, want_ctx=True)
    ye, me, se = ref.norm_forward(x, scale, shift, 1e-5)
    ref.within(y, *ye, "y")
    ref.within(rstd, *se, "rstd")
    assert torch.equal(y[3], shift.to(dtype)) and float(rstd[3]) == pytest.approx(1e-5 ** -0.5, rel=1e-6)
    x[5, 7] = float("inf")
    x[6, 1] = float("nan")
    got = op.forward(x)[0]
    others = torch.tensor([i not in (5, 6) for i in range(20)])
    assert torch.equal(got[others], y[others]) and bool(got[6].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_norm_of_no_rows(dtype):
    gen = torch.Generator().manual_seed(9)
    op, scale, shift = _norm(gen, 48, dtype, dtype)
    x = torch.empty(0, 48, dtype=dtype, device="cuda")
    y, ctx = op.forward(x, want_ctx=True)
    op._grads.fill_(1.0)
    assert op.backward(ctx, x, y).shape == (0, 48) and not bool(op._grads.any())


def test_norm_gradients_against_differences():
    """Central differences of the forward pass in 64 bits with statistics of its own: h = 1e-5 leaves an error of third derivatives times
    h^2 (below 1e-7 here) and of cancellation (1e-11 of the sum)."""
    gen = torch.Generator().manual_seed(10)
    op, scale, shift = _norm(gen, 40, torch.float32, torch.float32)
    x, dy, skip = (_rows(gen, 17, 40, torch.float32) for _ in range(3))
    y, ctx = op.forward(x, want_ctx=True)
    dx = op.backward(ctx, x, dy, dL_dskip=skip)
    e = ref.norm_backward(x, *ctx, scale, dy, skip)

    def loss(x_, s_, b_):
        mean = x_.mean(1, keepdim=True)
        xh = (x_ - mean) / ((x_ - mean).square().mean(1, keepdim=True) + 1e-5).sqrt()
        return float((dy.double() * (xh * s_ + b_)).sum() + (skip.double() * x_).sum())

    parts = [x.double(), scale.double(), shift.double()]
    for at, name, got in ((0, "dx", dx), (1, "dscale", op._grads[:40]), (2, "dshift", op._grads[40:])):
        d = torch.randn(parts[at].shape, generator=gen).double().cuda()
        up, down = list(parts), list(parts)
        up[at], down[at] = parts[at] + 1e-5 * d, parts[at] - 1e-5 * d
        numeric = (loss(*up) - loss(*down)) / 2e-5
        # (mean and rstd are the kernel's: relative errors of 50 half steps of fp32)
        bound = float(((e[name][1] + ref.U32 * e[name][0].abs()) * d.abs()).sum()) + 200 * ref.U32 * float((e[name][0].abs() * d.abs()).sum() + (dy.abs().sum() if at < 2 else 0))
        assert abs(float((got.double() * d).sum()) - numeric) <= bound + 1e-5, name


# ---------------------------------------------------------------------------------------------------------------------
# clipping
# ---------------------------------------------------------------------------------------------------------------------
def _gradients(gen, sizes, dtypes, scale=1.0):
    return [(torch.randn(n, generator=gen) * scale).to(dtypes[i % len(dtypes)]).cuda() for i, n in enumerate(sizes)]


ALL = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("sizes", [[1], [7, 0, 8193], [8192] * 3, [100003, 3, 64, 16385, 1], [5] * 700, [9000001, 2049, 17, 4097]])
@pytest.mark.parametrize("dtypes", [[t] for t in ALL] + [ALL])
@pytest.mark.parametrize("apart", [False, True])
def test_clip(sizes, dtypes, apart):
    from neus2_amd.layers import GradientClip
    gen = torch.Generator().manual_seed(sum(sizes))
    g = _gradients(gen, sizes, dtypes)
    before = [t.clone() for t in g]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in g)) / 128
    out = [torch.full_like(t, 9.0) for t in g] if apart else None
    clip = GradientClip(g, out=out)
    # sums in fp64 (fp16: eight squares at a time in fp32, 8 half steps): the norm rounded once
    near = pytest.approx(norm, rel=10 * ref.U32)
    assert float(clip.norm(loss_scale=128.0)) == near
    assert all(torch.equal(a, b) for a, b in zip(g, before))
    assert float(clip.clip(2 * norm, loss_scale=128.0)) == near  # below the limit
    assert all(torch.equal(a, b) for a, b in zip(out if apart else g, before))
    assert float(clip.clip(0.3 * norm, loss_scale=128.0)) == near
    factor = 0.3 * norm / (norm + 1e-6)
    for a, b in zip(out if apart else g, before):
        ref.within(a, b.double() * factor, 12 * ref.U32 * b.double().abs() * factor, "clipped")
    if apart:
        assert all(torch.equal(a, b) for a, b in zip(g, before))


def test_clip_reads_what_the_tensors_hold_then():
    from neus2_amd.layers import GradientClip
    g = [torch.zeros(5000, device="cuda"), torch.zeros(3, 7, dtype=torch.float16, device="cuda")]
    clip = GradientClip(g)
    assert float(clip.norm()) == 0.0 and float(clip.clip(1.0)) == 0.0 and not any(bool(t.any()) for t in g)
    g[0][17], g[1][2, 3] = 3.0, 4.0
    assert float(clip.clip(0.5)) == 5.0
    assert float(g[0][17]) == pytest.approx(0.3, rel=1e-6) and float(g[1][2, 3]) == pytest.approx(0.4, rel=2 ** -11)
    assert float(GradientClip([]).norm()) == 0.0 and float(GradientClip([]).clip(1.0)) == 0.0


@pytest.mark.parametrize("dtype,size", [(torch.float32, 1e30), (torch.float32, 1e-30), (torch.bfloat16, 1e30), (torch.bfloat16, 1e-30), (torch.float16, 6e4), (torch.float16, 6e-8)])
def test_norm_of_values_whose_squares_leave_fp32(dtype, size):
    from neus2_amd.layers import GradientClip
    g = torch.full((4096,), size, device="cuda").to(dtype)
    exact = 64 * float(g[0])
    assert float(GradientClip([g]).norm()) == pytest.approx(exact, rel=10 * ref.U32)


def test_gradients_that_are_no_numbers():
    from neus2_amd.layers import GradientClip
    g = torch.ones(100, device="cuda")
    g[3] = float("inf")
    clip = GradientClip([g])
    assert float(clip.clip(1.0)) == math.inf
    assert bool(g[3].isnan()) and float(g.nan_to_num(0.0).abs().sum()) == 0.0
    assert math.isnan(float(clip.clip(1.0))) and bool(g.isnan().all())


def test_clipping_is_the_same_every_time():
    from neus2_amd.layers import GradientClip
    gen = torch.Generator().manual_seed(2)
    g = _gradients(gen, [70000, 1 << 20, 333, 12345], ALL)
    clip = GradientClip(g, out=[torch.empty_like(t) for t in g])
    runs = [(clip.clip(1.0).clone(), [t.clone() for t in clip._keep[1]]) for _ in range(3)]
    for norm, out in runs[1:]:
        assert torch.equal(norm, runs[0][0]) and all(torch.equal(a, b) for a, b in zip(out, runs[0][1]))


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
class Block:
    """x + W2 gelu(W1 norm(x) + b1) + b2, its parameters and gradients in one vector, as the optimiser takes them."""

    def __init__(self, gen, width, hidden):
        from neus2_amd.layers import LayerNorm, Linear
        self.ops = [LayerNorm(width), Linear(width, hidden, activation="GELU"), Linear(hidden, width)]
        sizes = [op.n_params() for op in self.ops]
        master = [torch.cat([torch.ones(width), torch.zeros(width)])]
        for i, o in ((width, hidden), (hidden, width)):
            master.append(torch.cat([torch.randn(o * i, generator=gen) / math.sqrt(i), torch.zeros(o)]))
        self.master = torch.cat(master).cuda()
        self.params, self.grads = self.master.half(), torch.zeros(sum(sizes), dtype=torch.float16, device="cuda")
        self.slices = [slice(sum(sizes[:k]), sum(sizes[:k + 1])) for k in range(3)]
        for op, s in zip(self.ops, self.slices):
            op.set_params(self.params[s], self.grads[s])

    def forward(self, x):
        norm, up, down = self.ops
        y, ctx = norm.forward(x, want_ctx=True)
        h, z = up.forward(y, want_pre_activation=True)
        out, _ = down.forward(h, residual=x)
        return out, (x, y, ctx, h, z)

    def backward(self, saved, dL_dout):
        norm, up, down = self.ops
        x, y, ctx, h, z = saved
        dh = down.backward(h, None, dL_dout)
        dy = up.backward(y, z, dh)
        return norm.backward(ctx, x, dy, dL_dskip=dL_dout), dh, dy


@pytest.mark.parametrize("n,width,hidden", [(300, 64, 256), (77, 41, 90)])
def test_a_training_step_of_a_residual_block(n, width, hidden):
    """Norm, two linear layers with the residual, backward through all, clipping, Adam: every stage against 64 bits on its own inputs."""
    from neus2_amd.layers import GradientClip
    from neus2_amd.tcnn_api import Adam
    gen = torch.Generator().manual_seed(n)
    block = Block(gen, width, hidden)
    adam, clip = Adam(block.master, block.master.numel()), GradientClip([block.grads[s] for s in block.slices])
    x, g = _rows(gen, n, width, torch.float16), _rows(gen, n, width, torch.float16, scale=128.0 / n)
    for _ in range(2):
        out, saved = block.forward(x)
        _, y, ctx, h, z = saved
        p = [block.params[s] for s in block.slices]
        w1, b1 = p[1][:width * hidden].view(hidden, width), p[1][width * hidden:]
        w2, b2 = p[2][:width * hidden].view(width, hidden), p[2][width * hidden:]
        ref.within(y, *ref.norm_forward(x, p[0][:width], p[0][width:], 1e-5)[0], "norm")
        he, ze, dh_, dz_ = ref.linear_forward(y, w1, b1, None, "GELU")
        ref.within(h, he, dh_, "hidden")
        oe, _, do_, _ = ref.linear_forward(h, w2, b2, x, "None")
        ref.within(out, oe, do_, "out")
        dx, dh, dy = block.backward(saved, g)
        e2, e1 = ref.linear_backward(h, w2, None, g, "None"), ref.linear_backward(y, w1, z, dh, "GELU")
        e0 = ref.norm_backward(x, *ctx, p[0][:width], dy, g)
        for what, got, e in (("dh", dh, e2["dx"]), ("dy", dy, e1["dx"]), ("dx", dx, e0["dx"])):
            ref.within(got, *e, what)
        grads = [block.grads[s] for s in block.slices]
        for what, got, e in (("dw2", grads[2][:-width].view(width, hidden), e2["dw"]), ("db2", grads[2][-width:], e2["db"]), ("dw1", grads[1][:-hidden].view(hidden, width), e1["dw"]),
                             ("db1", grads[1][-hidden:], e1["db"]), ("dscale", grads[0][:width], e0["dscale"]), ("dshift", grads[0][width:], e0["dshift"])):
            ref.within(got, *e, what)
        before, exact = block.grads.clone(), float(block.grads.double().norm()) / 128
        assert float(clip.clip(0.5 * exact, loss_scale=128.0)) == pytest.approx(exact, rel=10 * ref.U32)
        ref.within(block.grads, before.double() * 0.5, before.double().abs() * 0.5 * (12 * ref.U32 + 1e-6 / exact), "clipped")
        old = block.master.clone()
        adam.step(block.params, block.grads)
        assert bool((block.master != old).any()) and torch.equal(block.params, block.master.half())


def test_a_captured_step_of_a_residual_block_replays():
    """Forward, backward and clipping in a graph: every replay on new inputs gives what the eager calls give, with eager work between."""
    from neus2_amd.layers import GradientClip
    gen = torch.Generator().manual_seed(12)
    block = Block(gen, 64, 192)
    clip = GradientClip([block.grads])
    x, g = _rows(gen, 500, 64, torch.float16), _rows(gen, 500, 64, torch.float16, scale=0.25)

    def step():
        out, saved = block.forward(x)
        dx, _, _ = block.backward(saved, g)
        return out, dx, clip.clip(0.01, loss_scale=128.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        x.copy_(_rows(gen, 500, 64, torch.float16))
        eager = [t.clone() for t in step()] + [block.grads.clone()]
        block.grads.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*captured, block.grads], eager)), k


def test_two_streams_at_once():
    """Calls of one layer's shape on two streams at the same time, each with its own parameters' gradients."""
    gen = torch.Generator().manual_seed(13)
    pairs = []
    for _ in range(2):
        op, w, b = _linear(gen, 160, 96, "SiLU", bias=True, dtype=torch.float16)
        pairs.append((op, _rows(gen, 3000, 160, torch.float16), _rows(gen, 3000, 96, torch.float16), _rows(gen, 3000, 96, torch.float16)))
    alone = []
    for op, x, z, dy in pairs:
        alone.append((op.backward(x, z, dy), op._grads.clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for op, *_ in pairs:
        op._grads.zero_()
    torch.cuda.synchronize()
    together = []
    for _ in range(3):
        for s, (op, x, z, dy) in zip(streams, pairs):
            with torch.cuda.stream(s):
                together.append(op.backward(x, z, dy))
    torch.cuda.synchronize()
    for k, (op, *_) in enumerate(pairs):
        assert torch.equal(op._grads, alone[k][1])
        assert all(torch.equal(t, alone[k][0]) for t in together[k::2])


def test_rows_beyond_32_bits():
    """More than 2^32 values in a matrix: the last rows are found by every pass (all others are zero, or checked by a sample)."""
    n, i, last = 17_000_000, 256, 50
    gen = torch.Generator().manual_seed(21)
    x = torch.zeros(n, i, dtype=torch.float16, device="cuda")
    x[-last:] = torch.randn(last, i, generator=gen).half().cuda()
    for o in (8, 264):  # with the weights in LDS, and in tiles
        op, w, b = _linear(gen, i, o, "None", bias=True, dtype=torch.float16)
        y = op.forward(x)[0]
        ye, _, dy_, _ = ref.linear_forward(x[-last:], w, b, None, "None")
        ref.within(y[-last:], ye, dy_, "y")
        ref.within(y[:1000], b.double().expand(1000, o), 0.0, "y of zeros")
        dy = torch.randn(1000, o, generator=gen).half().cuda().repeat(n // 1000, 1)
        dx = op.backward(x, None, dy)
        e = ref.linear_backward(x[-last:], w, None, dy[-last:], "None")
        ref.within(dx[-last:], *e["dx"], "dx")
        ref.within(dx[n // 2 - 500:n // 2 + 500], *ref.linear_backward(x[:1000], w, None, dy[n // 2 - 500:n // 2 + 500], "None")["dx"], "dx of a sample")
        ref.within(op._grads[:o * i].view(o, i), *e["dw"], "dw")
        del y, dy, dx
    op, scale, shift = _norm(gen, i, torch.float16, torch.float16)
    y, (mean, rstd) = op.forward(x, want_ctx=True)
    ref.within(y[-last:], *ref.norm_forward(x[-last:], scale, shift, 1e-5)[0], "norm")
    ref.within(y[:1000], shift.double().expand(1000, i), 0.0, "norm of zeros")
    dy = torch.zeros_like(x)
    dy[-last:] = torch.randn(last, i, generator=gen).half().cuda()
    dx = op.backward((mean, rstd), x, dy, dL_dskip=x)
    e = ref.norm_backward(x[-last:], mean[-last:], rstd[-last:], scale, dy[-last:], x[-last:])
    ref.within(dx[-last:], *e["dx"], "norm dx")
    ref.within(op._grads[:i], *e["dscale"], "dscale")
    assert not bool(dx[:-last].any())
    del y, dx, dy


def test_clip_of_one_tensor_beyond_32_bits():
    from neus2_amd.layers import GradientClip
    n = (1 << 32) + 12345
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-3:] = torch.tensor([3.0, 0.0, 4.0])
    clip = GradientClip([g])
    assert float(clip.clip(1.0)) == 5.0
    assert [float(v) for v in g[-3:]] == pytest.approx([0.6, 0.0, 0.8], rel=2 ** -8) and not bool(g[:-3].any())


def test_a_clip_is_not_made_under_capture():
    from neus2_amd.capi import N2Error
    from neus2_amd.layers import GradientClip
    g = torch.ones(100, device="cuda")
    graph, refused = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        try:
            GradientClip([g])
        except N2Error as e:
            refused.append(str(e))
        g.mul_(2.0)
    assert len(refused) == 1 and "captured" in refused[0]
    graph.replay()
    torch.cuda.synchronize()
    assert float(g[0]) == 2.0 and float(GradientClip([g]).norm()) == 20.0


def test_layers_refuse_other_types_shapes_and_orders():
    from neus2_amd.capi import N2Error
    from neus2_amd.layers import GradientClip, LayerNorm, Linear
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    lin, norm = Linear(8, 4, activation="ReLU"), LayerNorm(8)
    for call in (lambda: lin.set_params(h(35)), lambda: lin.set_params(h(36).float()), lambda: lin.set_params(h(72)[::2]), lambda: norm.set_params(h(15)), lambda: norm.set_params(h(16).float())):
        with pytest.raises(N2Error):
            call()
    lin.set_params(h(36)), norm.set_params(h(16))
    x, y = h(5, 8), h(5, 4)
    ctx = norm.forward(x, want_ctx=True)[1]
    for call in (lambda: lin.forward(h(5, 7)), lambda: lin.forward(x.float()), lambda: lin.forward(h(8, 5).t()), lambda: lin.forward(x, residual=h(4, 4)), lambda: lin.forward(x, out=h(5, 5)),
                 lambda: lin.forward(x, residual=h(1, 4).expand(5, 4)), lambda: lin.forward(x.cpu()), lambda: lin.backward(x, None, y), lambda: lin.backward(x, y, y),  # (no gradients were set)
                 lambda: lin.forward(x, out=x[:, :4]), lambda: norm.forward(x, out=x), lambda: norm.backward(None, x, x), lambda: norm.backward(ctx, x, x), lambda: norm.forward(h(5, 9)),
                 lambda: norm.backward((ctx[0][:4], ctx[1]), x, x, mode=0), lambda: norm.backward(ctx, x, x, dL_dskip=x, want_input_grad=False, mode=0),
                 lambda: GradientClip([h(4, 4).t()[:2]]), lambda: GradientClip([x, x]), lambda: GradientClip([x], out=[y]), lambda: GradientClip([x, y], out=[x]),
                 lambda: GradientClip([torch.zeros(3, dtype=torch.int32, device="cuda")]), lambda: GradientClip([x[:, ::2]])):
        with pytest.raises(N2Error):
            call()
