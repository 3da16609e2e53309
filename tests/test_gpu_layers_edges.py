"""The layers and the clipping where their numbers leave what fp32 holds easily, against their formulas in 64 bits."""
import math

import pytest
import torch

import layers_ref as ref

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", ["GELU", "SiLU"])
def test_activations_keep_their_tails(kind, dtype):
    """Every finite value of the type through the epilogue and through the slope, one layer of a single weight 1: the negative tails are as
    exact as their own size asks for, down to the smallest numbers of the type.

    The bound before the rounding is relative to |y|, or to the two terms of the slope: 16 half steps of fp32 for what is computed, and for
    the exponent -z or -z^2 / 2, formed with at most three roundings, three half steps of it, which is what they move the exponential by."""
    from neus2_amd.layers import Linear
    values = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    values = values[torch.isfinite(values)].cuda()[:, None]
    op = Linear(1, 1, activation=kind, bias=False, dtype=dtype)
    op.set_params(torch.ones(1, dtype=dtype, device="cuda"))
    y = op.forward(values)[0]
    z = values.double()
    if kind == "GELU":
        below, exponent = torch.special.erfc(-z * math.sqrt(0.5)) / 2, z * z / 2
        second = z * torch.exp(-exponent) / math.sqrt(2 * math.pi)
    else:
        below, exponent = torch.exp(torch.minimum(z, torch.zeros_like(z))) / (1 + torch.exp(-z.abs())), z.abs()
        second = z * below * torch.exp(-torch.maximum(z, torch.zeros_like(z))) / (1 + torch.exp(-z.abs()))
    relative = (16 + 3 * exponent.clamp(max=200.0)) * ref.U32
    ref.within(y, z * below, relative * (z * below).abs(), "y")
    dx = op.backward(values, values, torch.ones_like(values), mode=0)
    ref.within(dx, below + second, relative * (below + second.abs()), "slope")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [8, 12, 1001])
def test_norm_keeps_an_infinite_mean(width, dtype):
    """A row with infinities of one sign has that infinity for its mean; the other rows are as without it."""
    from neus2_amd.layers import LayerNorm
    gen = torch.Generator().manual_seed(width)
    x = torch.randn(7, width, generator=gen).to(dtype).cuda()
    op = LayerNorm(width, dtype=dtype)
    op.set_params(torch.cat([torch.ones(width), torch.zeros(width)]).to(dtype).cuda())
    y, (mean, rstd) = op.forward(x, want_ctx=True)
    x[2, 5], x[4, 0], x[4, 3], x[6, 1], x[6, 2] = math.inf, -math.inf, -math.inf, math.inf, -math.inf
    y2, (mean2, rstd2) = op.forward(x, want_ctx=True)
    assert float(mean2[2]) == math.inf and float(mean2[4]) == -math.inf and math.isnan(float(mean2[6]))
    assert bool(y2[[2, 4, 6]].isnan().all()) and bool(rstd2[[2, 4, 6]].isnan().all())
    rest = [0, 1, 3, 5]
    assert torch.equal(y2[rest], y[rest]) and torch.equal(mean2[rest], mean[rest]) and torch.equal(rstd2[rest], rstd[rest])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [1, 12, 63, 1001, 2056, 5000])
def test_norm_backward_of_equal_values_far_from_zero(width, dtype):
    """Rows whose mean times 1 / deviation leaves fp32: what stands past the rows' ends in the lanes' vectors has no part in the sums."""
    from neus2_amd.layers import LayerNorm
    gen = torch.Generator().manual_seed(width)
    op = LayerNorm(width, epsilon=1e-12, dtype=dtype)
    params = torch.cat([1 + 0.1 * torch.randn(width, generator=gen), torch.zeros(width)]).to(dtype).cuda()
    op.set_params(params, torch.zeros_like(params))
    x = torch.full((5, width), 1e34, device="cuda").to(dtype)
    x[1] = torch.randn(width, generator=gen).to(dtype).cuda()
    dy = torch.randn(5, width, generator=gen).to(dtype).cuda()
    _, (mean, rstd) = op.forward(x, want_ctx=True)
    assert bool((rstd[[0, 2, 3, 4]] > 9e5).all())
    dx = op.backward((mean, rstd), x, dy)
    e = ref.norm_backward(x, mean, rstd, params[:width], dy, None)
    ref.within(dx, *e["dx"], "dx")
    ref.within(op._grads[:width], *e["dscale"], "dscale")
    ref.within(op._grads[width:], *e["dshift"], "dshift")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size,loss_scale,max_norm", [(1e19, 1e-25, 1.0), (1e30, 1e-30, 0.5), (1e5, 1.0, 1e-39), (3e37, 1.0, 1e-2)])
def test_clip_by_a_factor_below_fp32(size, loss_scale, max_norm, dtype):
    """max_norm / norm is no normal number of fp32, or zero, where the clipped gradients are: bound, half a step for the factor in fp64 and the product each."""
    from neus2_amd.layers import GradientClip
    gen = torch.Generator().manual_seed(3)
    g = (torch.randn(5003, generator=gen) * size).to(dtype).cuda()
    before = g.double()
    norm = float(before.square().sum().sqrt()) / torch.tensor(loss_scale, dtype=torch.float32).double().item()
    factor = torch.tensor(max_norm, dtype=torch.float32).double().item() / (norm + 1e-6)
    assert factor < 1.2e-38
    GradientClip([g]).clip(max_norm, loss_scale=loss_scale)
    exact = before * factor
    ref.within(g, exact, 4 * ref.U32 * exact.abs(), "clipped")


def test_the_norm_of_fp16_gradients_loses_no_small_square():
    """Squares of 10.5 beside those of 60 000, a step of fp32 for 256: the sum is fp64's, so the norm is off by its own rounding alone (and 2^-40 for the sum's)."""
    from neus2_amd.layers import GradientClip
    g = torch.full((4096, 8), 10.5, dtype=torch.float16, device="cuda")
    g[:, 3] = 60000.0
    exact = math.sqrt(float(g.double().square().sum()))
    clip = GradientClip([g], out=[torch.empty_like(g)])
    for norm in (clip.norm(), clip.clip(1.0)):
        assert abs(float(norm) - exact) <= (ref.U32 + 2.0 ** -40) * exact


def test_a_dropped_clips_table_waits_for_the_streams_that_read_it():
    """The table is made on one stream and read on another, where the call waits behind a long piece of work: dropped then, its memory is not
    handed out again before that call is done, and the clipped gradients are right."""
    from neus2_amd.layers import GradientClip
    tensors = [torch.full((64,), 1.0, device="cuda") for _ in range(2000)]
    big = torch.ones(1 << 28, device="cuda")
    side = torch.cuda.Stream()
    clip = GradientClip(tensors)
    table, size = clip._table.data_ptr(), clip._table.numel()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(200):
            big.mul_(1.0)
        norm = clip.clip(1.0)
        done = side.record_event()
    del clip
    new = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(8)]
    early = not done.query()
    assert early and all(t.data_ptr() != table for t in new)
    torch.cuda.synchronize()
    assert float(norm) == pytest.approx(math.sqrt(128000.0), rel=1e-6)
    assert all(float(t[0]) == pytest.approx(1 / math.sqrt(128000.0), rel=1e-5) for t in tensors[::100])


@pytest.mark.parametrize("residual", [False, True])
def test_as_many_rows_as_there_can_be(residual):
    """2^31 - 1 rows of one value, in tiles: more workgroups than one launch has threads for.  Every value is checked: all are small whole
    numbers, exact in fp16 but for the weight's gradient, which is rounded once."""
    from neus2_amd.layers import Linear
    n = (1 << 31) - 1
    op = Linear(1, 1, activation="ReLU", dtype=torch.float16)
    params = torch.tensor([2.0, -8.0], dtype=torch.float16, device="cuda")
    op.set_params(params, torch.zeros_like(params))
    x = torch.arange(13, dtype=torch.float16, device="cuda").repeat(n // 13 + 1)[:n, None]
    y, z = op.forward(x, residual=x if residual else None, want_pre_activation=True)
    assert torch.equal(z, x * 2 - 8)
    assert torch.equal(y, z.clamp(min=0) + x if residual else z.clamp(min=0))
    if residual:
        return
    del y
    dy = torch.zeros_like(x)
    dy[::1 << 20] = 1.0  # 2048 rows of a gradient
    dy[-5:] = 1.0
    dx = op.backward(x, z, dy)
    on = (z > 0) & (dy > 0)
    assert torch.equal(dx, on.half() * 2)
    assert float(op._grads[0]) == float(torch.tensor(float(x[on].double().sum())).half()) and float(op._grads[1]) == float(torch.tensor(float(on.sum())).half())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", ["SiLU", "GELU"])
@pytest.mark.parametrize("n,i,o", [(5, 24, 40), (300, 72, 96), (5003, 320, 257), (3000, 264, 520), (50000, 64, 128), (49155, 200, 72)])
def test_the_backward_pass_rounds_dz_once(n, i, o, kind, dtype):
    """dL/dz meets the matrix cores in the layer's type, the one rounding besides the results' own: with the identity for weights the input's
    gradient is dL/dz as it was rounded, and from that the gradients of any weights are off by their fp32 sums and their own rounding alone."""
    from neus2_amd.layers import Linear
    gen = torch.Generator().manual_seed(n + i)
    z, dy = (torch.randn(n, o, generator=gen).to(dtype).cuda() for _ in range(2))
    x = torch.randn(n, i, generator=gen).to(dtype).cuda()
    identity = Linear(o, o, activation=kind, bias=False, dtype=dtype)
    identity.set_params(torch.eye(o, dtype=dtype, device="cuda").reshape(-1))
    dz = identity.backward(torch.zeros(n, o, dtype=dtype, device="cuda"), z, dy, mode=0)
    g = dy.double()
    ref.within(dz, g * ref.slope(z.double(), kind), 2.0 ** -20 * g.abs(), "dz")
    op = Linear(i, o, activation=kind, dtype=dtype)
    w = (torch.randn(o, i, generator=gen) / math.sqrt(o)).to(dtype).cuda()
    params = torch.cat([w.reshape(-1), torch.zeros(o, dtype=dtype, device="cuda")])
    op.set_params(params, torch.zeros_like(params))
    dx = op.backward(x, z, dy)
    d = dz.double()
    ref.within(dx, d @ w.double(), 2 * (o + 2) * ref.U32 * (d.abs() @ w.double().abs()), "dx")
    ref.within(op._grads[:o * i].view(o, i), d.T @ x.double(), 2 * (n + 66) * ref.U32 * (d.abs().T @ x.double().abs()), "dw")
    if n > 40000:
        dx = op.backward(x, z, dy, mode=0)  # (formed on the way to dx)
        ref.within(dx, d @ w.double(), 2 * (o + 2) * ref.U32 * (d.abs() @ w.double().abs()), "dx alone")


def test_an_infinite_limit_clips_nothing():
    from neus2_amd.layers import GradientClip
    g = torch.arange(1.0, 101.0, device="cuda")
    clip = GradientClip([g])
    assert float(clip.clip(math.inf)) == pytest.approx(math.sqrt(338350.0), rel=2 * ref.U32) and torch.equal(g, torch.arange(1.0, 101.0, device="cuda"))
    g[7] = math.inf
    assert float(clip.clip(math.inf)) == math.inf and bool(g.isnan().all())


def test_a_captured_clip_replays_and_is_dropped():
    """Made on one stream, captured on another: every replay clips what the tensors hold then, as eager calls do, and the object goes behind its graph."""
    from neus2_amd.layers import GradientClip
    gen = torch.Generator().manual_seed(4)
    sizes = [70000, 333, 1]
    g = [torch.zeros(k, device="cuda") for k in sizes]
    clip = GradientClip(g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip.clip(0.5, loss_scale=2.0)
    for _ in range(4):
        fresh = [torch.randn(k, generator=gen).cuda() for k in sizes]
        [t.copy_(f) for t, f in zip(g, fresh)]
        graph.replay()
        torch.cuda.synchronize()
        replayed, n = [t.clone() for t in g], norm.clone()
        [t.copy_(f) for t, f in zip(g, fresh)]
        assert torch.equal(clip.clip(0.5, loss_scale=2.0), n) and all(torch.equal(a, b) for a, b in zip(g, replayed))
    del graph
    del clip
    torch.cuda.synchronize()
    assert float(GradientClip(g).norm()) == pytest.approx(1.0, rel=1e-5)
