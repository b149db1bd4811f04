"""The fp8 feed-forward example with frozen weights: what needs a gradient gets it, and the weights may change."""

import importlib.util
import pathlib

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = pathlib.Path(__file__).resolve().parents[1] / "feather-ops_amd" / "examples" / "block_scaled_mlp.py"


@pytest.fixture
def mlp(cuda_device):
    spec = importlib.util.spec_from_file_location("block_scaled_mlp", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    torch.manual_seed(1)
    return module.BlockScaledMLP(640, 1000)


def _inputs():
    g = torch.Generator("cuda").manual_seed(2)
    return [torch.randn((30, 640), generator=g, device="cuda").bfloat16() for _ in range(2)]


def test_gradient_through_frozen_weights(mlp):
    x, residual = _inputs()
    want_y, _ = mlp(x.requires_grad_(), residual)
    gy = torch.randn_like(want_y)
    want, = torch.autograd.grad(want_y, x, gy)
    mlp.freeze_()
    for leaf, other in ((x, residual), (x.detach(), residual.clone().requires_grad_())):
        y, h = mlp(leaf, other)
        got, = torch.autograd.grad(y, leaf if leaf.requires_grad else other, gy)
        assert torch.equal(y, want_y) and torch.equal(got, want)
    y, _ = mlp(x.detach(), residual)
    with torch.no_grad():
        assert torch.equal(mlp(x, residual)[0], y) and y.grad_fn is None
    mlp.norm.requires_grad_(True)   # the norm's weight alone
    y, _ = mlp(x.detach(), residual)
    assert torch.autograd.grad(y, mlp.norm, gy)[0].abs().sum() > 0


def test_frozen_without_kept_codes(mlp):
    x, residual = _inputs()
    mlp.requires_grad_(False)
    y, _ = mlp(x, residual)
    frozen, _ = mlp.freeze_()(x, residual)
    assert ((y.float() - frozen.float()).norm() / frozen.float().norm()).item() < 0.1


def test_weights_that_change(mlp):
    x, residual = _inputs()
    mlp.freeze_()
    with torch.no_grad():
        before, _ = mlp(x, residual)
        mlp.load_state_dict({name: value * 2 for name, value in mlp.state_dict().items()})
        after, _ = mlp(x, residual)
        want, _ = mlp.freeze_()(x, residual)
    assert torch.equal(after, want) and not torch.equal(after, before)
