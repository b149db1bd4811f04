"""The feed-forward operators' nodes in traced programs: what they say of their results, and gradients for inputs of any shape."""

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu
SHAPES = [(5, 70), (2, 3, 70), (70,), (5, 72), (90, 70)]


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").bfloat16()


def _same_layout(op, *args):
    """A node's results lie as its shape function says they do."""
    torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_layouts_of_the_gated_blocks_nodes(fo, shape):
    x, w, b = _randn(*shape), _randn(24, shape[-1], seed=1), _randn(24, seed=2)
    ops = torch.ops.feather_ops
    _same_layout(ops.gated_linear_auto.default, x, w, b, 1)
    gy = _randn(*shape[:-1], 12, seed=3)
    for needs in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        _same_layout(ops.gated_linear_auto_backward.default, gy, x, w, b, 1, *needs)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_layouts_of_the_4_bit_products_nodes(fo, shape):
    x, b = _randn(*shape), _randn(24, seed=2)
    codes, scale, zero = fo.quantize_int4(_randn(24, shape[-1], seed=1), 32, zeros=True)
    ops = torch.ops.feather_ops
    _same_layout(ops.int4_linear_auto.default, x, codes, scale, zero, b)
    _same_layout(ops.int4_gated_auto.default, x, codes, scale, zero, b, 1)
    _same_layout(ops.int4_linear_auto_backward.default, _randn(*shape[:-1], 24, seed=3), codes, scale, zero, shape[-1])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["gated", "int4"])
def test_compiled_gradients(fo, kind, shape):
    """A vector's too. They are the eager ones (of the 4-bit product's bias but for the order of the sum: it is rounded once either way)."""
    x, w, b = _randn(*shape), _randn(24, shape[-1], seed=1), _randn(24, seed=2)
    int4 = fo.quantize_int4(w, 32, zeros=True)
    gy = _randn(*shape[:-1], 12 if kind == "gated" else 24, seed=3)

    def step(t, u, v):
        return fo.gated_linear(t * 2, u, v) if kind == "gated" else fo.int4_linear(t * 2, *int4, v)

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    wanted = leaves if kind == "gated" else [leaves[0], leaves[2]]
    want, got = step(*leaves), compiled(*leaves)
    assert torch.equal(got, want)
    expected, mine = (torch.autograd.grad(y, wanted, gy) for y in (want, got))
    for p, q, leaf in zip(mine, expected, wanted):
        assert p.shape == leaf.shape
        exact = kind == "gated" or leaf is leaves[0]
        if exact:
            assert torch.equal(p, q)
        else:   # two fp32 sums of the same values, and two roundings
            rows = gy.reshape(-1, 24).double().abs()
            sums = 2 * (rows.shape[0] + 34) * ref.ULP * rows.sum(0)
            assert ((p.double() - q.double()).abs() <= sums + 2 * ref.half_step(p.dtype, q.double().abs() + sums)).all()
