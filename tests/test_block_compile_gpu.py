"""The operators with one scale for each block of 128 under torch.compile: one node for a product and for a layer, values
and gradients those of the eager calls."""

import pytest
import torch
from torch import nn
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import feather_ops as fo

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def fresh(cuda_device):
    torch._dynamo.reset()


def _randn(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def _operands(m, n, k, by_row=False):
    return (*fo.quantize_blocks(_randn(m, k, seed=1)), *fo.quantize_blocks(_randn(n, k, seed=2), square=not by_row))


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 512), (64, 256, 4096), (300, 500, 700), (1000, 264, 768)])
def test_product(m, n, k, dynamic):
    operands, bias = _operands(m, n, k), _randn(n, seed=3)

    def run(*args):
        return fo.block_scaled_mm(*args)

    compiled = torch.compile(run, fullgraph=True, dynamic=dynamic)
    assert torch.equal(compiled(*operands, bias), run(*operands, bias))
    assert torch.equal(compiled(*_operands(m, n, k, True), None, torch.float32), run(*_operands(m, n, k, True), None, torch.float32))
    a, sa, b, sb = operands   # rows off the boundaries: copied inside the node
    apart = torch.cat([a[:, :1], a], 1)[:, 1:]
    assert torch.equal(compiled(apart, sa, b, sb, bias), run(*operands, bias))


def _nodes(run, *args):
    graphs = []

    def backend(gm, example_inputs):
        graphs.append(gm)
        return gm.forward

    out = torch.compile(run, backend=backend, fullgraph=True)(*args)
    assert len(graphs) == 1
    return out, [str(n.target) for n in graphs[0].graph.nodes if "feather_ops" in str(n.target)]


def test_one_node_each():
    a, sa, b, sb = _operands(40, 256, 4096)
    out, nodes = _nodes(lambda *args: fo.block_scaled_mm(*args), a, sa, b, sb)
    assert len(nodes) == 1 and torch.equal(out, fo.block_scaled_mm(a, sa, b, sb))
    layer = nn.Linear(256, 130, device="cuda", dtype=torch.bfloat16)
    fo.to_block_scaled_linear(layer)
    x = _randn(2, 9, 256, seed=4)
    out, nodes = _nodes(layer, x)
    assert len(nodes) == 1 and torch.equal(out, layer(x))


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("shape", [(20, 300), (2, 33, 300), (300,)])
def test_layer_inference(shape, frozen, dynamic):
    torch.manual_seed(5)
    layer = nn.Linear(300, 200, device="cuda", dtype=torch.bfloat16).requires_grad_(not frozen)
    fo.to_block_scaled_linear(layer)
    x = _randn(*shape, seed=6)
    with torch.no_grad():
        assert torch.equal(torch.compile(layer, fullgraph=True, dynamic=dynamic)(x), layer(x))


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("q", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_training_step(dtype, q, bias):
    x, w, gy = _randn(2, 70, 300, seed=7, dtype=dtype), _randn(200, 300, seed=8, dtype=dtype), _randn(2, 70, 200, seed=9, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, *([_randn(200, seed=10, dtype=dtype)] if bias else []))]
    compiled = torch.compile(lambda *args: fo.block_scaled_linear(*args, dtype=q), fullgraph=True)
    want = torch.autograd.grad(fo.block_scaled_linear(*leaves, dtype=q), leaves, gy)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(compiled(*leaves), leaves, gy), want))
    for i, leaf in enumerate(leaves):
        args = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(compiled(*args), leaf, gy)[0], want[i])


def test_frozen_layer_gives_its_input_gradient():
    torch.manual_seed(11)
    layer = nn.Linear(300, 200, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    fo.to_block_scaled_linear(layer, torch.float8_e5m2)
    x, gy = _randn(20, 300, seed=12).requires_grad_(), _randn(20, 200, seed=13)
    want = layer(x)
    got = torch.compile(layer, fullgraph=True)(x)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got, x, gy)[0], torch.autograd.grad(want, x, gy)[0])


@pytest.mark.parametrize("assign", [False, True])
def test_frozen_layer_that_changes(assign):
    torch.manual_seed(14)
    layer = nn.Linear(300, 200, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    fo.to_block_scaled_linear(layer)
    compiled, x = torch.compile(layer, fullgraph=True), _randn(20, 300, seed=15)
    with torch.no_grad():
        before = compiled(x)
        for _ in range(2):
            layer.load_state_dict({k: v * 2 + 1 for k, v in layer.state_dict().items()}, assign=assign)
            layer.requires_grad_(False)
            got = compiled(x)
            assert torch.equal(got, fo.block_scaled_linear(x, layer.weight, layer.bias)) and not torch.equal(got, before)
            assert torch.equal(layer(x), got) and torch.equal(compiled(x), got)
            before = got


def test_norm_and_gate():
    x, res, w = _randn(33, 512, seed=16), _randn(33, 512, seed=17), _randn(512, seed=18)

    def inference(x, res, w):
        codes, scale, h = fo.rms_norm_quantized(x, w, res)
        c2, s2 = fo.silu_mul_quantized(h)
        c3, s3 = fo.quantize_blocks(h)
        return codes.float() * scale.repeat_interleave(128, 1), h, c2.float(), s2, c3.float(), s3

    for a, b in zip(torch.compile(inference, fullgraph=True)(x, res, w), inference(x, res, w)):
        assert torch.equal(a, b)

    def training(x, res, w):
        y, h = fo.rms_norm(x, w, res)
        return fo.silu_mul(y), h

    leaves = [t.requires_grad_() for t in (x, res, w)]
    gy, gh = _randn(33, 256, seed=19), _randn(33, 512, seed=20)
    got, want = torch.compile(training, fullgraph=True)(*leaves), training(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(torch.autograd.grad(got, leaves, (gy, gh)), torch.autograd.grad(want, leaves, (gy, gh))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("backend", ["eager", "aot_eager", "inductor"])
def test_derivatives_that_are_not_there_are_refused(backend):
    x, w = _randn(20, 300, seed=21).requires_grad_(), _randn(200, 300, seed=22).requires_grad_()
    compiled = torch.compile(lambda x, w: fo.block_scaled_linear(x, w), fullgraph=True, backend=backend)
    y = compiled(x, w)
    with pytest.raises(RuntimeError, match="no autograd formula|double backward"):
        gx, = torch.autograd.grad(y.sum(), x, create_graph=True)
        torch.autograd.grad(y.float().mean() + gx.float().square().sum(), w)
    for tensor in (x, x.detach()):
        for shape in ((20, 300), (2, 10, 300)):
            with forward_ad.dual_level(), pytest.raises(NotImplementedError):
                compiled(forward_ad.make_dual(tensor.view(shape), torch.ones_like(x).view(shape)), w.detach())


def test_traced_program_runs_again():
    """Products that are split along K: the program's own workspace, cleared where it has to be in each run."""
    operands = _operands(64, 256, 4096)
    traced = make_fx(lambda *a: fo.block_scaled_mm(*a), tracing_mode="fake")(*operands)
    for seed in range(3):
        fresh_ones = (*fo.quantize_blocks(_randn(64, 4096, seed=30 + seed)), *operands[2:])
        assert torch.equal(traced(*fresh_ones), fo.block_scaled_mm(*fresh_ones))
