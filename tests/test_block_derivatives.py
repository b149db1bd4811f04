"""Derivatives that the fp8 layer does not have, without a GPU: the real autograd node over plain forms of the ops in it.
They are refused, never left out of a sum."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

import feather_ops as fo

M, N, K = 6, 20, 256


def _values(codes, scale):
    if scale.shape[0] != codes.shape[0]:
        scale = scale.repeat_interleave(128, 0)[:codes.shape[0]]
    return codes.float() * scale.repeat_interleave(128, 1)[:, :codes.shape[1]]


def _quantized(x, e5m2, square):
    """Scales of one: what these tests look at does not depend on them."""
    codes = x.float().to(torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn)
    return codes, torch.ones(-(-x.shape[0] // 128) if square else x.shape[0], -(-x.shape[1] // 128))


def _quantize_tiles(x, e5m2, square, plain, transposed, sums):
    none = x.new_empty((0, 0))
    return (*(_quantized(x, e5m2, square) if plain else (none, none)),
            *(_quantized(x.t(), e5m2, square) if transposed else (none, none)),
            torch.stack([part.float().sum(0) for part in x.split(128)]) if sums else none)


def _mm(a, a_scale, b, b_scale, bias, out_type, workspace):
    y = _values(a, a_scale) @ _values(b, b_scale).t()
    return (y if bias is None else y + bias).to((torch.bfloat16, torch.float16, torch.float32)[out_type])


@pytest.fixture
def plain_ops():
    library = torch.library.Library("feather_ops", "IMPL", "CPU")
    library.impl("quantize_tiles", _quantize_tiles)
    library.impl("quantize_blocks", lambda x, e5m2: _quantized(x, e5m2, False))
    library.impl("block_scaled_mm", _mm)
    library.impl("sum_rows", lambda part, out_type: part.sum(0))
    yield
    library._destroy()


@pytest.fixture
def leaves():
    g = torch.Generator().manual_seed(1)
    return [torch.randn(shape, generator=g).requires_grad_() for shape in ((M, K), (N, K), (N,))]


def test_gradient_of_a_gradient_as_last_layer(plain_ops, leaves):
    """The gradient that a sum sends back is a constant; dx depends on the weight all the same, and dW on x."""
    x, w, b = leaves
    gx, = torch.autograd.grad(fo.block_scaled_linear(x, w, b).sum(), x, create_graph=True)
    assert gx.requires_grad
    assert torch.autograd.grad(gx.square().sum(), x, allow_unused=True, retain_graph=True) == (None,)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(gx.square().sum(), w, allow_unused=True)
    y = fo.block_scaled_linear(x, w, b)
    gx, gw = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
    for penalty, inputs in ((gx, w), (gw, x), (gx, (w, b))):   # with the first derivative's own way to the inputs
        with pytest.raises(RuntimeError, match="not implemented"):
            torch.autograd.grad(y.mean() + penalty.square().sum(), inputs)
    with pytest.raises(RuntimeError, match="not implemented"):
        (y.mean() + gx.square().sum()).backward()


@pytest.mark.parametrize("which", [0, 1])
def test_gradient_of_a_gradient_with_one_operand_of_constants(plain_ops, leaves, which):
    """By a constant weight dx depends on x only through the gradient that comes in."""
    args = [leaf if i == which else leaf.detach() for i, leaf in enumerate(leaves)]
    grad, = torch.autograd.grad(fo.block_scaled_linear(*args).square().sum(), args[which], create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(grad.sum(), args[which])
    grad, = torch.autograd.grad(fo.block_scaled_linear(*args).sum(), args[which], create_graph=True)
    assert not grad.requires_grad


def test_first_gradients_with_a_graph_have_the_same_values(plain_ops, leaves):
    g = torch.randn(M, N, generator=torch.Generator().manual_seed(2))
    for grad in (g, g.clone().requires_grad_()):
        plain = torch.autograd.grad(fo.block_scaled_linear(*leaves), leaves, grad)
        kept = torch.autograd.grad(fo.block_scaled_linear(*leaves), leaves, grad, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, kept))
        assert not any(t.requires_grad for t in plain)
        assert [t.requires_grad for t in kept] == [True, True, grad.requires_grad]   # the bias's is the sum of grad alone
    for again in kept:
        with pytest.raises(RuntimeError, match="not implemented"):
            torch.autograd.grad(again.sum(), grad, retain_graph=True)


# ---- forward mode ----


def _entry_points(x, w, b):
    norm = w[0]
    return {"silu_mul": lambda x=x: fo.silu_mul(x), "silu_mul batch": lambda x=x: fo.silu_mul(x[None]),
            "rms_norm": lambda x=x: fo.rms_norm(x, norm), "rms_norm weight": lambda x=norm: fo.rms_norm(b, x),
            "rms_norm residual": lambda x=x: fo.rms_norm(w[:M], norm, x),
            "linear": lambda x=x: fo.block_scaled_linear(x, w), "linear weight": lambda x=w: fo.block_scaled_linear(b, x),
            "linear bias": lambda x=norm[:N]: fo.block_scaled_linear(b, w, x)}


NAMES = ["silu_mul", "silu_mul batch", "rms_norm", "rms_norm weight", "rms_norm residual", "linear", "linear weight",
         "linear bias"]


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, graph):
    """A dual tensor's tangent, of any operand, with and without a gradient beside it and outside of grad mode."""
    with FakeTensorMode():
        x, w, b = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for shape in ((M, K), (N, K), (M, K)))
        call = _entry_points(x, w, b)[name]
        primal, = call.__defaults__
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(primal.clone().requires_grad_(graph), torch.empty_like(primal))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
            call()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (primal,), (torch.empty_like(primal),))


def test_tangent_of_the_layers_gradient_is_refused(plain_ops, leaves):
    y = fo.block_scaled_linear(*leaves)
    with forward_ad.dual_level():
        grad = forward_ad.make_dual(torch.ones(M, N), torch.ones(M, N))
        for inputs in (leaves, leaves[0], leaves[2]):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, inputs, grad, retain_graph=True)
