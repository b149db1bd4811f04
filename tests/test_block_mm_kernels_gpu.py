"""Every kernel of the block-scaled product against 64 bits, by the shapes that reach it: both formats on either side, scales
by square and by row, with K ending inside a block and a piece."""

import pytest
import torch

import block_ref as ref
from block_mm_shapes import LAUNCHES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _uneven(m, k, seed):
    """Normal values, each row's blocks of 128 by another power of two, so that a scale of another row or block shows."""
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((m, k), generator=g, device="cuda")
    powers = torch.randint(-3, 4, (m, ref.blocks(k)), generator=g, device="cuda").float().exp2()
    return x * powers.repeat_interleave(128, 1)[:, :k]


@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("b", sorted(ref.FP8))
@pytest.mark.parametrize("a", sorted(ref.FP8))
@pytest.mark.parametrize("shape", LAUNCHES, ids=str)
def test_kernel(fo, shape, a, b, by_row):
    m, n, k = shape
    operands = (*fo.quantize_blocks(_uneven(m, k, 1), ref.FP8[a]),
                *fo.quantize_blocks(_uneven(n, k, 2), ref.FP8[b], square=not by_row))
    bias = _uneven(1, n, 3)[0]
    want, slack = ref.mm(*operands, bias)
    for dtype in (torch.float32, torch.bfloat16):
        if dtype != torch.float32:
            bias = bias.to(dtype)
            want, slack = ref.mm(*operands, bias)
        got = fo.block_scaled_mm(*operands, bias, dtype)
        ref.check_close(got, want, slack, shape)
        assert torch.equal(fo.block_scaled_mm(*operands, bias, dtype), got)   # the same bits again


@pytest.mark.parametrize("shape", LAUNCHES, ids=str)
def test_bytes_past_k_do_not_count(fo, shape):
    """Rows padded with NaN codes, which the kernels read up to the end of a piece."""
    m, n, k = shape
    a, sa = fo.quantize_blocks(_uneven(m, k, 4))
    b, sb = fo.quantize_blocks(_uneven(n, k, 5), square=True)
    want = fo.block_scaled_mm(a, sa, b, sb, None, torch.float32)
    nan = torch.full((m + n, ref.blocks(k) * 128 + 64), 0x7f, dtype=torch.uint8, device="cuda").view(a.dtype)
    nan[:m, :k], nan[m:, :k] = a, b
    assert torch.equal(fo.block_scaled_mm(nan[:m, :k], sa, nan[m:, :k], sb, None, torch.float32), want)
    assert want.isfinite().all()


@pytest.mark.parametrize("m", [1, 33, 200])
def test_zeros(fo, m):
    n, k = 300, 500
    weight = fo.quantize_blocks(_uneven(n, k, 6), square=True)
    zero = fo.quantize_blocks(torch.zeros((m, k), device="cuda"))
    assert (fo.block_scaled_mm(*zero, *weight, None, torch.float32) == 0).all()


@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("m,n", [(2, 300), (20, 9000), (50, 70), (100, 300), (1400, 300), (300, 3300), (1312, 5426), (5551, 646), (1411, 5383)])
def test_no_columns_to_sum_over(fo, m, n, by_row):
    """K = 0: the bias alone, on whatever kernel."""
    a, b = (torch.zeros((rows, 0), dtype=torch.float8_e4m3fn, device="cuda") for rows in (m, n))
    sa, sb = torch.ones((m, 0), device="cuda"), torch.ones((n if by_row else ref.blocks(n), 0), device="cuda")
    bias = _uneven(1, n, 7)[0].bfloat16()
    assert torch.equal(fo.block_scaled_mm(a, sa, b, sb, bias), bias.expand(m, n))
    assert (fo.block_scaled_mm(a, sa, b, sb) == 0).all()
