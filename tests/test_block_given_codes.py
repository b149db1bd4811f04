"""Codes that are passed to block_scaled_linear beside the weight, under fake tensors."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import feather_ops as fo


def test_codes_of_another_weight_are_refused():
    with FakeTensorMode():
        x, w = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for shape in ((5, 300), (200, 300)))
        codes, scale = fo.quantize_blocks(w, square=True)
        assert fo.block_scaled_linear(x, w, quantized_weight=(codes, scale)).shape == (5, 200)
        other, other_scale = fo.quantize_blocks(torch.empty((130, 300), dtype=torch.bfloat16, device="cuda"), square=True)
        rows = fo.quantize_blocks(w)
        for given, dtype in (((other, other_scale), torch.float8_e4m3fn), ((codes[:, :200], scale[:, :2]), torch.float8_e4m3fn),
                             ((codes[:130], scale), torch.float8_e4m3fn), ((codes, scale), torch.float8_e5m2),
                             ((codes.view(torch.uint8), scale), torch.float8_e4m3fn)):
            for leaf in (w, w.clone().requires_grad_()):
                with pytest.raises(ValueError, match="quantized_weight"):
                    fo.block_scaled_linear(x, leaf, None, dtype, quantized_weight=given)
        # scales by row are a product like any other, but not what the backward takes the weight in
        assert fo.block_scaled_linear(x, w, quantized_weight=rows).shape == (5, 200)
        for given in (rows, (codes, scale[:1])):
            with pytest.raises(ValueError, match="quantized_weight"):
                fo.block_scaled_linear(x.clone().requires_grad_(), w, quantized_weight=given)
