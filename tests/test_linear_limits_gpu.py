"""The longest sums that the feed-forward operators' gradients take."""

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu
LONGEST = 1 << 21


def _randn(*shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * scale).bfloat16()


def test_weights_gradient_over_the_most_rows(cuda_device):
    import feather_ops as fo

    x, w, gy = _randn(LONGEST, 16, seed=1), _randn(16, 16, seed=2, scale=0.25).requires_grad_(), _randn(LONGEST, 8, seed=3)
    (gw,) = torch.autograd.grad(fo.gated_linear(x, w), w, gy)
    ref.check(gw, *ref.gated_gradients(x, w.detach(), None, "silu", gy)[1])


def test_inputs_gradient_over_the_most_rows_of_a_weight(cuda_device):
    import feather_ops as fo

    x, w, gy = _randn(3, 16, seed=1).requires_grad_(), _randn(LONGEST, 16, seed=2, scale=0.25), _randn(3, LONGEST // 2, seed=3)
    (gx,) = torch.autograd.grad(fo.gated_linear(x, w), x, gy)
    ref.check(gx, *ref.gated_gradients(x.detach(), w, None, "silu", gy)[0])
    int4, gy = fo.quantize_int4(w, 32), _randn(3, LONGEST, seed=4)
    (gx,) = torch.autograd.grad(fo.int4_linear(x, *int4), x, gy)
    v = ref.int4_values(*int4, 16)
    size = gy.double().abs() @ v.abs()
    ref.check(gx, gy.double() @ v, gy.double().abs() @ ref.half_step(torch.bfloat16, v) + ref.sum_error(LONGEST, size))
