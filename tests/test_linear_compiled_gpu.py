"""The feed-forward operators' nodes in traced programs: what they say of their results, and gradients for inputs of any shape."""

import pytest
import torch

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
