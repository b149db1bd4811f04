"""4-bit weights of values at the ends of their type's range."""

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", ref.HALVES)
def test_weights_of_the_largest_values(cuda_device, dtype, zeros, group):
    """A group's range may be twice the type's largest value, in bfloat16 past fp32's."""
    import feather_ops as fo

    largest = torch.finfo(dtype).max
    w = (torch.rand((9, 300), generator=torch.Generator("cuda").manual_seed(group), device="cuda") * 1.8 - 0.9).double() * largest
    w = w.to(dtype)
    codes, scale, zero = fo.quantize_int4(w, group, zeros=zeros)
    assert scale.isfinite().all() and (scale > 0).all()
    values = ref.int4_values(codes, scale, zero, 300)
    # a step, of which rounding codes costs half and rounding zero points the rest, and the scale's own rounding, 15 times
    step = scale.double().repeat_interleave(group, 1)[:, :300]
    assert ((values - w.double()).abs() <= step * (1.0 if zeros else 0.5) + 16 * ref.half_step(dtype, step)).all()
    assert torch.equal(fo.dequantize_int4(codes, scale, zero), values.to(dtype))
