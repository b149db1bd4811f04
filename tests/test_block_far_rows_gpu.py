"""Rows of codes and scales that lie further apart than the product's kernels reach: slices of long batches."""

import pytest
import torch

import block_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _quantized(fo, m, k, seed, **kw):
    g = torch.Generator("cuda").manual_seed(seed)
    return fo.quantize_blocks(torch.randn((m, k), generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("m", [4, 80])
def test_last_token_of_a_long_batch(fo, m):
    """Codes [m, tokens, K] with each batch's rows 2^23 bytes apart, their scales 2^21 floats."""
    k, n, tokens = 1024, 200, 8192
    a, sa = _quantized(fo, m, k, 1)
    b, sb = _quantized(fo, n, k, 2, square=True)
    batch = torch.zeros((m, tokens, k), dtype=torch.uint8, device="cuda").view(a.dtype)
    batch[:, -1] = a
    scales = torch.full((m, 1 << 21), float("nan"), device="cuda")
    scales[:, :k // 128] = sa
    far, far_scale = batch[:, -1], scales[:, :k // 128]
    assert far.stride(0) > 1 << 22 and far_scale.stride(0) > 1 << 20
    want = fo.block_scaled_mm(a, sa, b, sb)
    ref.check_close(want, *ref.mm(a, sa, b, sb))
    assert torch.equal(fo.block_scaled_mm(far, sa, b, sb), want)
    assert torch.equal(fo.block_scaled_mm(a, far_scale, b, sb), want)
    assert torch.equal(fo.block_scaled_mm(far, far_scale, b, sb), want)
    # as the second operand, with scales by row; far as the weight's codes of a layer
    want = fo.block_scaled_mm(b, sb.repeat_interleave(128, 0)[:n], a, sa)
    assert torch.equal(fo.block_scaled_mm(b, sb.repeat_interleave(128, 0)[:n], far, far_scale), want)
    # a long batch whose scales are block by block, [K / 128, m, tokens]: the last token's are `tokens` apart from row to row
    by_block = torch.full((k // 128, m, tokens), float("nan"), device="cuda")
    by_block[:, :, -1] = sa.t()
    assert torch.equal(fo.block_scaled_mm(a, by_block[:, :, -1].t(), b, sb), fo.block_scaled_mm(a, sa, b, sb))
