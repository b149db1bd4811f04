"""The gated activation's gradient where its factors are the type's largest: a masked gate, and products of two of them that
pass the range of fp32 while the gradient does not."""

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _grad(gate, up, gy):
    x = torch.tensor([[gate, up]], dtype=gy.dtype, device="cuda").requires_grad_()
    got, = torch.autograd.grad(fo.silu_mul(x), x, gy)
    g, u = x.detach().double()[0]
    s, d = torch.sigmoid(g), gy.double()[0, 0]
    return got[0], torch.stack([d * u * (s * (1 + g * (1 - s))), d * (g * s)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gy", [-3.0, 1.0, 64.0])
def test_masked_gate(cuda_device, dtype, gy):
    """The type's lowest value as a gate's mask: silu and its slope are zero there, so both gradients are."""
    lowest = torch.finfo(dtype).min
    for up in (-2.0, 0.0, 5.0, torch.finfo(dtype).max):
        got, want = _grad(lowest, up, torch.full((1, 1), gy, dtype=dtype, device="cuda"))
        assert (want == 0).all() and (got == 0).all(), (up, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate,up,gy", [(-60.0, 1e30, 1e20), (-40.0, -1e25, 1e18), (-1e25, 1e30, 1e20), (-80.0, 3e38, 1e10),
                                        (1.5, 3.3e38, 0.5), (1.5, 0.5, 2.7e38), (-60.0, 1e-20, 1e30), (-60.0, 1e30, 1e-20)])
def test_products_past_the_range(cuda_device, dtype, gate, up, gy):
    """At most 16 roundings and the exponential's argument's, as everywhere, where the result is in range."""
    got, want = _grad(gate, up, torch.full((1, 1), gy, dtype=dtype, device="cuda"))
    unit = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24
    assert want.abs().max() < 0.99 * torch.finfo(dtype).max
    limit = (unit + 2.0**-20 + abs(gate) * 2.0**-22 if gate > -100 else 0.0) * want.abs() + 2.0**-125
    assert ((got.double() - want).abs() <= limit).all(), (got, want)
