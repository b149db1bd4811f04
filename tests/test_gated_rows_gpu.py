"""Rows of the same input come out alike, in every value: infinities and NaN too."""

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m", [2, 20, 40, 70, 300])
def test_rows_with_extreme_gates_are_alike(cuda_device, m, dtype, act):
    import feather_ops as fo

    low, large = torch.finfo(dtype).min, torch.finfo(dtype).max
    gates = torch.tensor([low, large, float("-inf"), float("nan"), 0.0, -200.0, float("inf"), 1.0])
    ups = torch.tensor([large, 0.5, 2.0, 1.0, float("inf"), 1.0, -3.0, low])
    w = torch.zeros(16, 8, dtype=dtype, device="cuda")
    w[:8, 0], w[8:, 0] = gates.to(dtype), ups.to(dtype)
    x = torch.zeros(m, 8, dtype=dtype, device="cuda")
    x[:, 0] = 1
    y = fo.gated_linear(x, w, None, act)
    want = torch.tensor([0.0, large / 2, 0.0, float("nan"), float("nan"), 0.0, float("-inf"), 0.0], dtype=torch.float64, device="cuda")
    value = ref.activation(torch.ones(1, dtype=torch.float64, device="cuda"), act)[0] * low
    row = y[0].double()
    assert torch.equal(row.isnan(), want.isnan())
    assert torch.equal(row[[0, 1, 2, 6]], want[[0, 1, 2, 6]].to(dtype).double()) and row[5].abs() < 1e-6
    assert (row[7] - value).abs() <= value.abs() * ref.ACT + ref.half_step(dtype, value)
    assert torch.allclose(y, y[:1].expand_as(y), rtol=0, atol=0, equal_nan=True)
