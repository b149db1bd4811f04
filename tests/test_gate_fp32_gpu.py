"""The gated activation of fp32 values is as exact as fp32 is, at gates of any size."""

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu
UNIT = 2.0**-24
# In units: the exponential 2 (an ulp), 1 + t 1 and the quotient 1 (t's own error reaches it by t / (1 + t) at most), s = t q 1,
# g s 1, times up 1; one of the two is no product (g > 0), one more is spare for the terms of second order.
FORWARD = 8 * UNIT


def _x(m, n, seed, spread):
    g = torch.Generator("cuda").manual_seed(seed)
    gate = (torch.rand((m, n), generator=g, device="cuda") * 2 - 1) * spread
    return torch.cat([gate, torch.randn((m, n), generator=g, device="cuda")], -1)


def _parts(x):
    g, u = x.double().chunk(2, -1)
    return g, u, torch.sigmoid(g), torch.sigmoid(-g)


@pytest.mark.parametrize("spread", [1.0, 20.0, 80.0])
def test_forward(cuda_device, spread):
    x = _x(300, 1000, 1, spread)
    g, u, s, _ = _parts(x)
    want = g * s * u
    assert ((fo.silu_mul(x).double() - want).abs() <= FORWARD * want.abs() + 2.0**-126).all()


@pytest.mark.parametrize("spread", [1.0, 20.0, 80.0])
def test_gradient(cuda_device, spread):
    """The slope's 1 + g (1 - s) is a sum whose terms may cancel: its error is that of the terms."""
    x = _x(300, 1000, 2, spread).requires_grad_()
    gy = torch.randn((300, 1000), generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    got, = torch.autograd.grad(fo.silu_mul(x), x, gy)
    g, u, s, c = _parts(x.detach())
    d = gy.double()
    want = torch.cat([d * u * s * (1 + g * c), d * g * s], -1)
    size = torch.cat([(d * u * s).abs() * (1 + g.abs() * c), (d * g * s).abs()], -1)
    # s or c 5, g c 1, the sum 1, times s 5 and 1, times each factor 1
    assert ((got.double() - want).abs() <= 16 * UNIT * size + 2.0**-126).all()
