"""Derivatives that the operators with one scale for each block of 128 do not have are refused on the GPU, never left out."""

import pytest
import torch
from torch.autograd import forward_ad

import feather_ops as fo

pytestmark = pytest.mark.gpu


@pytest.fixture
def leaves(cuda_device):
    g = torch.Generator("cpu").manual_seed(1)
    return [torch.randn(shape, generator=g).bfloat16().cuda().requires_grad_() for shape in ((6, 256), (20, 256), (20,))]


def test_gradient_penalty_on_the_last_layer(leaves):
    x, w, b = leaves
    y = fo.block_scaled_linear(x, w, b)
    gx, gw = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
    for penalty, inputs in ((gx, w), (gw, x), (gx, (w, b))):
        with pytest.raises(RuntimeError, match="not implemented"):
            torch.autograd.grad(y.float().mean() + penalty.float().square().sum(), inputs, retain_graph=True)
    for outs, inputs in (((fo.silu_mul(x),), (x,)), (fo.rms_norm(x, w[0].detach(), w[:6].detach()), (x,))):
        gx, = torch.autograd.grad(sum(out.sum() for out in outs), inputs, create_graph=True)
        with pytest.raises(RuntimeError, match="not implemented"):
            torch.autograd.grad(sum(out.float().mean() for out in outs) + gx.float().square().sum(), inputs)
    plain = torch.autograd.grad(fo.block_scaled_linear(x, w, b).sum(), leaves)
    kept = torch.autograd.grad(fo.block_scaled_linear(x, w, b).sum(), leaves, create_graph=True)
    assert all(torch.equal(a, c) for a, c in zip(plain, kept))


def test_forward_mode_is_refused(leaves):
    x, w, b = (leaf.detach() for leaf in leaves)
    calls = {"silu_mul": fo.silu_mul, "rms_norm": lambda t: fo.rms_norm(t, w[0]),
             "block_scaled_linear": lambda t: fo.block_scaled_linear(t, w, b)}
    for name, call in calls.items():
        with pytest.raises(NotImplementedError, match=f"forward-mode derivatives of {name}"):
            torch.func.jvp(call, (x,), (x,))
        leaf = x.clone().requires_grad_()
        y = call(leaf)
        with forward_ad.dual_level():
            for tensor in (x, leaf):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(forward_ad.make_dual(tensor, x))
            with pytest.raises(RuntimeError, match="forward"):   # the tangent of a gradient that comes in
                torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
