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


def _at_end(rows, cols, seed, dtype=torch.bfloat16, pad=0):
    """Values whose last one is the last of 64 MiB of its own, rows `pad` further apart than they are long."""
    total = (64 << 20) // dtype.itemsize
    buffer = torch.empty(total, dtype=dtype, device="cuda")
    view = buffer.as_strided((rows, cols), (cols + pad, 1), total - ((rows - 1) * (cols + pad) + cols))
    return view.copy_(torch.randn((rows, cols), generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (5, 513), (7, 1003), (3, 2049), (300, 4100), (2, 9001), (2, 17001), (4, 256)])
def test_norm_and_gate(cuda_device, rows, cols, dtype):
    for pad in (0, 3):
        x, res, gy = (_at_end(rows, cols, seed, dtype, pad) for seed in (1, 2, 3))
        w = _at_end(1, cols, 4, dtype)[0]
        ends, plain = ([t if same else t.clone() for t in (x, res, w, gy)] for same in (True, False))
        results = []
        for x, res, w, gy in (ends, plain):
            leaves = [t.detach().requires_grad_() for t in (x, res, w)]
            y, h = fo.rms_norm(leaves[0], leaves[2], leaves[1])
            results.append((y, h, *torch.autograd.grad((y, h), leaves, (gy, gy)), fo.rms_norm_quantized(x, w, res)[1]))
            if cols % 2 == 0:
                leaf = x.detach().requires_grad_()
                y = fo.silu_mul(leaf)
                results[-1] += (y, *torch.autograd.grad(y, leaf, gy[:, :cols // 2]), fo.silu_mul_quantized(x)[1])
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("m,n,k", [(1, 5, 100), (1, 390, 3504), (20, 100, 1008), (40, 100, 1008), (70, 130, 400), (300, 260, 1008),
                                   (1500, 2600, 400)])
def test_product(cuda_device, m, n, k):
    """Codes and scales at the end of theirs, the output's bias too."""
    def at_end(t):
        # rows of codes start on 16-byte boundaries: a K that is no multiple of 16 only for a single row
        buffer = torch.empty((64 << 20) // t.dtype.itemsize, dtype=t.dtype, device="cuda")
        return buffer[-t.numel():].view(t.shape).copy_(t)

    g = torch.Generator("cuda").manual_seed(5)
    a, sa = fo.quantize_blocks(torch.randn((m, k), generator=g, device="cuda"))
    bias = torch.randn(n, generator=g, device="cuda").bfloat16()
    if k % 16:
        n, bias = 1, bias[:1]
    for square in (True, False):
        b, sb = fo.quantize_blocks(torch.randn((n, k), generator=g, device="cuda"), square=square)
        want = fo.block_scaled_mm(a, sa, b, sb, bias)
        ends = [at_end(t.contiguous()) for t in (a, sa, b, sb, bias)]
        assert torch.equal(fo.block_scaled_mm(*ends), want)
