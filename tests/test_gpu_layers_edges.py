"""The layers and the clipping where their numbers leave what fp32 holds easily, against their formulas in 64 bits."""
import math

import pytest
import torch

import layers_ref as ref

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", ["GELU"])
def test_activations_keep_their_tails(kind, dtype):
    """Every finite value of the type through the epilogue, one layer of a single weight 1: the negative tail is as exact as its own size
    asks for, down to the smallest numbers of the type.

    The bound before the rounding is relative to |y|: 16 half steps of fp32 for what the epilogue computes, and for the exponent -z or
    -z^2 / 2, formed with at most three roundings, three half steps of it, which is what they move the exponential by."""
    from neus2_amd.layers import Linear
    values = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    values = values[torch.isfinite(values)].cuda()[:, None]
    op = Linear(1, 1, activation=kind, bias=False, dtype=dtype)
    op.set_params(torch.ones(1, dtype=dtype, device="cuda"))
    y = op.forward(values)[0]
    z = values.double()
    exact = z * torch.special.erfc(-z * math.sqrt(0.5)) / 2 if kind == "GELU" else z / (1 + torch.exp(-z))
    exponent = torch.minimum(z * z / 2 if kind == "GELU" else z.abs(), torch.full_like(z, 200.0))
    ref.within(y, exact, (16 + 3 * exponent) * ref.U32 * exact.abs(), "y")
