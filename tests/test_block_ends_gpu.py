"""Matrices whose last value is the last of their memory: nothing past it is read."""

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (130, 77), (129, 200), (5, 1003)])
def test_quantized_tiles(cuda_device, rows, cols, dtype):
    """64 MiB of its own, a whole number of the allocator's pieces, with rows apart and off the 16-byte boundaries."""
    total = (64 << 20) // dtype.itemsize
    buffer = torch.empty(total, dtype=dtype, device="cuda")
    ld = cols + 3
    x = buffer.as_strided((rows, cols), (ld, 1), total - ((rows - 1) * ld + cols))
    x.copy_(torch.randn((rows, cols), generator=torch.Generator("cuda").manual_seed(1), device="cuda"))
    assert x.data_ptr() + ((rows - 1) * ld + cols) * dtype.itemsize == buffer.data_ptr() + (64 << 20)
    for square in (False, True):
        got, want = (torch.ops.feather_ops.quantize_tiles(t, False, square, True, True, True) for t in (x, x.contiguous()))
        for a, b in zip(got, want):
            same = [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b)]
            assert torch.equal(*same)
    assert torch.equal(fo.quantize_blocks(x)[1], fo.quantize_blocks(x.contiguous())[1])
