"""What the feed-forward operators' gradients cannot sum is refused by the forward that would need them, without a GPU."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import feather_ops as fo

LONG = (1 << 21) + 8


@pytest.fixture
def new():
    with FakeTensorMode():
        yield lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="cuda")


def test_rows_of_x_that_the_weights_gradient_sums(new):
    x, w = new(LONG, 64), new(48, 64)
    with pytest.raises(ValueError, match="gradient of the weight"):
        fo.gated_linear(x, w.requires_grad_())
    with pytest.raises(ValueError, match="gradient of the weight"):
        fo.gated_linear(x.view(2, LONG // 2, 64), w)
    with torch.no_grad():
        assert fo.gated_linear(x, w).shape == (LONG, 24)
    assert fo.gated_linear(x.requires_grad_(), w.detach(), new(48).requires_grad_()).shape == (LONG, 24)
    assert fo.gated_linear(new(LONG - 8, 64), w).shape == (LONG - 8, 24)


def test_rows_of_the_weight_that_the_inputs_gradient_sums(new):
    x, w = new(4, 64), new(LONG, 64)
    codes, scale = new(LONG, 32, dtype=torch.uint8), new(LONG, 1)
    assert fo.gated_linear(x, w.requires_grad_()).shape == (4, LONG // 2)
    assert fo.int4_linear(x, codes, scale, None, new(LONG).requires_grad_()).shape == (4, LONG)
    x.requires_grad_()
    with pytest.raises(ValueError, match="gradient of x"):
        fo.gated_linear(x, w)
    for call in (fo.int4_linear, fo.int4_gated_linear):
        with pytest.raises(ValueError, match="gradient of x"):
            call(x, codes, scale)
    with torch.no_grad():
        assert fo.gated_linear(x, w).shape == (4, LONG // 2) and fo.int4_linear(x, codes, scale).shape == (4, LONG)


def test_sizes_that_no_product_takes(new):
    x, codes, scale = new(4, LONG), new(8, LONG // 2, dtype=torch.uint8), new(8, -(-LONG // 128))
    for call in (lambda: fo.gated_linear(x, new(8, LONG)), lambda: fo.int4_linear(x, codes, scale),
                 lambda: fo.int4_gated_linear(x, codes, scale)):
        with pytest.raises(ValueError, match="out of range"):
            call()
