"""What the autograd nodes of the norm and the gate do beside their gradients' values: graphs built or not, second
derivatives refused, saved tensors that change noticed, gradients of any layout, hooks and accumulation."""

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu


@pytest.fixture
def leaves(cuda_device):
    g = torch.Generator("cpu").manual_seed(5)
    new = lambda *shape: torch.randn(shape, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    return new(6, 256), new(256), new(6, 256)


def test_no_graph_without_a_reason(leaves):
    x, w, r = leaves
    with torch.no_grad():
        assert fo.silu_mul(x).grad_fn is None and fo.rms_norm(x, w, r)[0].grad_fn is None
    with torch.inference_mode():
        assert torch.equal(fo.silu_mul(x), fo.silu_mul(x.detach()))
    assert fo.silu_mul(x.detach()).grad_fn is None
    y, h = fo.rms_norm(x.detach(), w.detach(), r.detach())
    assert not y.requires_grad and not h.requires_grad
    y, h = fo.rms_norm(x.detach(), w, r.detach())
    assert y.requires_grad and y.grad_fn is not None


@pytest.mark.parametrize("shape", [(6, 256), (2, 3, 256), (256,)])
def test_values_are_those_without_a_graph(leaves, shape):
    x, w, r = (t.detach() for t in leaves)
    x, r = (x[:1] if len(shape) == 1 else x).reshape(shape), (r[:1] if len(shape) == 1 else r).reshape(shape)
    assert torch.equal(fo.silu_mul(x.clone().requires_grad_()), fo.silu_mul(x))
    for got, want in zip(fo.rms_norm(x.clone().requires_grad_(), w, r), fo.rms_norm(x, w, r)):
        assert torch.equal(got, want) and got.shape == torch.Size(shape)


def test_second_derivatives_are_refused(leaves):
    x, w, r = leaves
    for outs, ins in (((fo.silu_mul(x),), (x,)), (fo.rms_norm(x, w, r), (x, w, r)), ((fo.rms_norm(x, w),), (x, w))):
        first = torch.autograd.grad(sum(out.float().square().sum() for out in outs), ins, create_graph=True)
        with pytest.raises(RuntimeError, match="not implemented"):
            torch.autograd.grad(sum(grad.float().sum() for grad in first), ins)


def test_a_saved_tensor_that_changes_is_noticed(leaves):
    x, w, r = leaves
    kept = x * 1
    y = fo.silu_mul(kept)
    with torch.no_grad():
        kept.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, h = fo.rms_norm(x, w, r)   # h is kept for the backward
    with torch.no_grad():
        h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_of_any_layout(leaves):
    x, w, r = leaves
    plain = torch.randn(6, 256, generator=torch.Generator("cpu").manual_seed(6)).to(torch.bfloat16).cuda()
    apart = plain.t().contiguous().t()                          # columns side by side
    wide = torch.cat([plain, plain], 1)[:, :256]                # rows apart
    want = torch.autograd.grad(fo.rms_norm(x, w, r), (x, w, r), (plain, plain))
    gate = torch.autograd.grad(fo.silu_mul(x), x, plain[:, :128].contiguous())[0]
    for g in (apart, wide):
        for got, grad in zip(torch.autograd.grad(fo.rms_norm(x, w, r), (x, w, r), (g, g)), want):
            assert torch.equal(got, grad)
        assert torch.equal(torch.autograd.grad(fo.silu_mul(x), x, g[:, :128])[0], gate)
    one = plain[:1].expand(6, 256)                              # one row for all
    got = torch.autograd.grad(fo.rms_norm(x, w, r), (x, w, r), (one, one))
    want = torch.autograd.grad(fo.rms_norm(x, w, r), (x, w, r), (one.contiguous(), one.contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_accumulation_and_reuse(leaves):
    x, w, r = leaves
    plain = torch.ones(6, 256, dtype=torch.bfloat16, device="cuda")
    want = torch.autograd.grad(fo.rms_norm(x, w, r)[0], (x, w, r), plain)
    y, _ = fo.rms_norm(x, w, r)
    y.backward(plain, retain_graph=True)
    for leaf, grad in zip((x, w, r), want):
        assert torch.equal(leaf.grad, grad)
    assert x.grad.data_ptr() != r.grad.data_ptr()               # the two share a gradient, not its memory
    y.backward(plain)
    for leaf, grad in zip((x, w, r), want):
        assert torch.equal(leaf.grad, grad + grad)
    with pytest.raises(RuntimeError, match="second time"):
        y.backward(plain)


def _layer(m, n, k, seed=8):
    g = torch.Generator("cpu").manual_seed(seed)
    return [torch.randn(shape, generator=g).to(torch.bfloat16).cuda().requires_grad_() for shape in ((m, k), (n, k), (n,))]


def test_layer_second_derivatives_are_refused(cuda_device):
    args = _layer(20, 64, 256)
    first = torch.autograd.grad(fo.block_scaled_linear(*args).float().square().sum(), args, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(sum(grad.float().sum() for grad in first), args)


def test_layer_with_and_without_a_graph(cuda_device):
    x, w, b = _layer(20, 64, 256)
    with torch.no_grad():
        want = fo.block_scaled_linear(x, w, b)
    assert want.grad_fn is None and torch.equal(fo.block_scaled_linear(x, w, b), want)
    with torch.inference_mode():
        assert torch.equal(fo.block_scaled_linear(x.detach(), w.detach(), b.detach()), want)
    codes = fo.quantize_blocks(w, square=True)
    assert torch.equal(fo.block_scaled_linear(x, w, b, quantized_weight=codes), want)
    assert torch.equal(fo.block_scaled_linear(x.detach(), w.detach(), b.detach(), quantized_weight=codes), want)
    with pytest.raises(RuntimeError, match="go together"):
        torch.ops.feather_ops.block_scaled_linear(x, w, b, False, codes[0], None, None)


@pytest.mark.parametrize("apart", [False, True])
def test_layer_captured(cuda_device, apart):
    """A training pass in one graph, and forward and backward in two that share their memory; with split products. Replays
    with new inputs, eager passes between them."""
    from feather_ops import block_scaled

    m, n, k = 64, 256, 4096
    assert block_scaled._train_workspace_bytes(m, n, k) > 0
    x, w, b = _layer(m, n, k)
    gy = torch.randn(m, n, generator=torch.Generator("cpu").manual_seed(9)).to(torch.bfloat16).cuda()

    def eager():
        y = fo.block_scaled_linear(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph()]
    if apart:
        graphs.append(torch.cuda.CUDAGraph())
        pool = torch.cuda.graph_pool_handle()
        with torch.cuda.graph(graphs[0], pool=pool, stream=side):
            y = fo.block_scaled_linear(x, w, b)
        with torch.cuda.graph(graphs[1], pool=pool, stream=side):
            grads = torch.autograd.grad(y, (x, w, b), gy)
    else:
        with torch.cuda.graph(graphs[0], stream=side):
            y = fo.block_scaled_linear(x, w, b)
            grads = torch.autograd.grad(y, (x, w, b), gy)
    for replay in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(m, k, generator=torch.Generator("cpu").manual_seed(10 + replay)).to(torch.bfloat16))
            gy.copy_(torch.randn(m, n, generator=torch.Generator("cpu").manual_seed(20 + replay)).to(torch.bfloat16))
        want = eager()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip((y.detach(), *grads), want):
            assert torch.equal(got, expected), replay
