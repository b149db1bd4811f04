"""The fp8 feed-forward example: inference and training run the operators together, and both are as near the 32-bit layer as
their quantization allows."""

import importlib.util
import pathlib
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = pathlib.Path(__file__).resolve().parents[1] / "feather-ops_amd" / "examples" / "block_scaled_mlp.py"
# A code of 4 significant bits is off by at most 2^-4 of its value, about 2^-4 / sqrt(3) in the mean square and less after
# scaling; each product has two such operands, and the gated activation multiplies two products: with the three products'
# errors added as squares, under 0.1.
OFF = 0.1


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("block_scaled_mlp", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_inference_and_training(example, tokens):
    torch.manual_seed(tokens)
    mlp = example.BlockScaledMLP(640, 1000)
    x, residual = (torch.randn(tokens, 640, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    y, h = mlp(x, residual)
    gy = torch.randn_like(y)
    got = torch.autograd.grad((y, h), (x, mlp.norm, mlp.gate_up.weight, mlp.down.weight), (gy, torch.zeros_like(h)))
    plain = [t.detach().clone().requires_grad_() for t in (x, mlp.norm, mlp.gate_up.weight, mlp.down.weight)]
    copy = example.BlockScaledMLP(640, 1000)
    copy.norm, copy.gate_up.weight, copy.down.weight = (torch.nn.Parameter(t.detach()) for t in plain[1:])
    want_y = example.reference(copy, plain[0], residual.detach())
    want = torch.autograd.grad(want_y, (plain[0], copy.norm, copy.gate_up.weight, copy.down.weight), gy.float())
    for a, b in [(y, want_y), *zip(got, want)]:
        assert ((a.float() - b.float()).norm() / b.float().norm()).item() < OFF
    assert torch.equal(h, x + residual)
    with torch.no_grad():
        frozen, stream = mlp.freeze_()(x, residual)
    assert ((frozen.float() - want_y).norm() / want_y.norm()).item() < OFF and torch.equal(stream, h)


def test_command():
    run = subprocess.run([sys.executable, str(PATH), "--tokens", "3", "--width", "256", "--hidden", "384"],
                         capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr[-2000:]
    assert "training:" in run.stdout and "inference:" in run.stdout
