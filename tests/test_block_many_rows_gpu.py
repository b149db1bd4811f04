"""Launches of 2^32 threads and more, which the runtime cuts off without an error: many short rows, and very long ones."""

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def memory(cuda_device):
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _rows(m, n, seed=0):
    """A few rows' values, over and over: what each row's result is does not depend on where it is."""
    few = torch.randn((1021, n), generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(BF16)
    return few, few.repeat(-(-m // 1021), 1)[:m]


def _repeats(got, few):
    """Whether all rows of got are those of few, over and over."""
    whole = len(got) // len(few) * len(few)
    assert got.dtype == few.dtype and got.shape[1:] == few.shape[1:]
    same = torch.equal(got[whole:], few[:len(got) - whole])
    for part in got[:whole].split(len(few) << 14):
        same = same and bool((part.reshape(-1, *few.shape) == few).all())
    return same


def test_norm():
    m, n = (1 << 26) + 5, 8
    few, x = _rows(m, n)
    few_res, res = _rows(m, n, 1)
    w = torch.randn(n, device="cuda").to(BF16)
    for got, want in zip(fo.rms_norm(x, w, res), fo.rms_norm(few, w, few_res)):
        assert _repeats(got, want)
        del got
    codes, scale, h = fo.rms_norm_quantized(x, w, res)
    del h
    want_codes, want_scale, _ = fo.rms_norm_quantized(few, w, few_res)
    assert _repeats(codes.view(torch.uint8), want_codes.view(torch.uint8)) and _repeats(scale, want_scale)


def test_norm_gradients():
    m, n = (1 << 26) + 5, 8
    few, x = _rows(m, n)
    w = torch.randn(n, device="cuda").to(BF16)
    _, gy = _rows(m, n, 2)
    for t in (few, x):
        t.requires_grad_()
    got, = torch.autograd.grad(fo.rms_norm(x, w), x, gy)
    want, = torch.autograd.grad(fo.rms_norm(few, w), few, gy[:1021])
    assert _repeats(got, want)


def test_gate():
    m = (1 << 28) + 5
    few, x = _rows(m, 2)
    assert _repeats(fo.silu_mul(x), fo.silu_mul(few))
    few_gy, gy = _rows(m, 1, 3)
    assert _repeats(torch.ops.feather_ops.silu_mul_backward(gy, x), torch.ops.feather_ops.silu_mul_backward(few_gy, few))
    del gy
    for call in (fo.silu_mul_quantized, fo.quantize_blocks):
        codes, scale = call(x)
        want_codes, want_scale = call(few)
        assert _repeats(scale, want_scale) and _repeats(codes.view(torch.uint8), want_codes.view(torch.uint8))
        del codes, scale


def test_column_sums_of_the_most_rows():
    m = (1 << 31) - 1
    x = torch.ones((m, 1), dtype=BF16, device="cuda")
    *_, sums = torch.ops.feather_ops.quantize_tiles(x, False, False, False, False, True)
    assert sums.shape == (1 << 24, 1) and (sums[:-1] == 128).all() and sums[-1].item() == 127


def test_sums_of_the_most_columns():
    n = (1 << 28) + 37
    part = torch.stack([torch.arange(n, device="cuda", dtype=torch.float32), torch.ones(n, device="cuda")])
    assert torch.equal(torch.ops.feather_ops.sum_rows(part, 2), part[0] + 1)
