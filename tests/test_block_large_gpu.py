"""Operands, outputs and gradients past 2^32 bytes: the last rows, against the same rows alone, and the rows before them."""

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def freed(cuda_device):
    yield
    torch.cuda.empty_cache()


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("by_row", [False, True])
def test_output_of_a_product(by_row):
    """300,003 x 8,200 bf16: 4.9 GB. Its rows do not depend on how many there are but for the tile that takes them."""
    m, n, k, last = 300_003, 8200, 128, 700
    a, sa = fo.quantize_blocks(_randn(1, last, k))
    b, sb = fo.quantize_blocks(_randn(2, n, k), square=not by_row)
    bias = _randn(3, n)
    codes = torch.zeros((m, k), dtype=torch.uint8, device="cuda")
    codes[-last:] = a.view(torch.uint8)
    scale = torch.ones((m, 1), device="cuda")
    scale[-last:] = sa
    y = fo.block_scaled_mm(codes.view(a.dtype), scale, b, sb, bias)
    assert torch.equal(y[-last:], fo.block_scaled_mm(a, sa, b, sb, bias))   # one block of K: one sum, whatever the tile
    for at in range(0, m - last, 50_000):
        assert torch.equal(y[at:min(at + 100, m - last)], bias.expand(min(100, m - last - at), n))
    assert torch.equal(y[m - last - 1], bias)


def test_gradient_of_the_gate():
    m, f, last = (1 << 17) + 5, 8192, 3
    x = torch.zeros((m, 2 * f), dtype=torch.bfloat16, device="cuda")
    gy = torch.zeros((m, f), dtype=torch.bfloat16, device="cuda")
    x[-last:], gy[-last:] = _randn(4, last, 2 * f), _randn(5, last, f)
    small = x[-last:].clone().requires_grad_()
    want = torch.autograd.grad(fo.silu_mul(small), small, gy[-last:].clone())[0]
    x.requires_grad_()
    got = torch.autograd.grad(fo.silu_mul(x), x, gy)[0]
    assert torch.equal(got[-last:], want) and not got[-last - 1].any() and not got[0].any()


@pytest.mark.parametrize("d", [1024, 4096, 20_000])
def test_gradient_of_the_norm(d):
    """Rows of one wave, of a workgroup and past a workgroup's registers."""
    m, last = (1 << 31) // d + 7, 3
    x = torch.ones((m, d), dtype=torch.bfloat16, device="cuda")
    gy = torch.zeros((m, d), dtype=torch.bfloat16, device="cuda")
    x[-last:], gy[-last:] = _randn(6, last, d), _randn(7, last, d)
    w = _randn(8, d).requires_grad_()
    small = x[-last:].clone().requires_grad_()
    want, want_w = torch.autograd.grad(fo.rms_norm(small, w), (small, w), gy[-last:].clone())
    x.requires_grad_()
    y = fo.rms_norm(x, w)
    got, got_w = torch.autograd.grad(y, (x, w), gy)
    assert torch.equal(got[-last:], want) and not got[-last - 1].any() and not got[0].any()
    # three rows' terms and zeros: two roundings of a bf16 result, and the fp32 sum's order (a few terms of 2^-24)
    exact = (gy[-last:].double() * (y[-last:].double() / w.detach().double())).abs().sum(0)
    assert ((got_w.double() - want_w.double()).abs() <= want_w.double().abs() * 2.0**-7 + exact * 2.0**-20 + 1e-30).all()
