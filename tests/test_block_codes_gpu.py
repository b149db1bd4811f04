"""Codes are the nearest ones of value / scale: the quotient is rounded once to fp32, whichever way the block lies."""

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


def _want(x, q, square=False):
    """By the 64-bit quotient, rounded to fp32 and then to the code (of 16-bit values no quotient lies between the two
    nearest fp32 ones' middle and a 64-bit rounding of it)."""
    x = x.double()
    scale = ref.largest(x, square).clamp(min=2.0**-100) / ref.LARGEST[q]
    return (x / ref.spread(scale, *x.shape)).float().to(q).view(torch.uint8)


@pytest.mark.parametrize("q", sorted(ref.FP8))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_code(fo, dtype, q):
    """Two million values of few bits, whose quotients are ties now and then."""
    q = ref.FP8[q]
    x = (torch.randn((1024, 2048), generator=torch.Generator("cuda").manual_seed(1), device="cuda") * 3).to(dtype)
    assert torch.equal(fo.quantize_blocks(x, q)[0].view(torch.uint8), _want(x, q))
    assert torch.equal(fo.quantize_blocks(x, q, square=True)[0].view(torch.uint8), _want(x, q, True))
    codes, _, codes_t, _, _ = torch.ops.feather_ops.quantize_tiles(x, q == torch.float8_e5m2, False, True, True, False)
    assert torch.equal(codes.view(torch.uint8), _want(x, q))
    assert torch.equal(codes_t.view(torch.uint8), _want(x.t(), q))


@pytest.mark.parametrize("q", sorted(ref.FP8))
@pytest.mark.parametrize("size", [1e-44, 1e-36, 1e-28, 1.0, 1e30, 3e38])
def test_values_of_any_size(fo, size, q):
    """fp32, down to where the scale's floor holds and up to the range's end: the same, but for quotients within 2^-40 of a
    tie, which 64 bits round either way."""
    q = ref.FP8[q]
    x = (torch.rand((256, 512), generator=torch.Generator("cuda").manual_seed(2), device="cuda", dtype=torch.float64) * 2 - 1) * size
    x = x.float()
    codes, scale = fo.quantize_blocks(x, q)
    ref.check_quantized(x, codes, scale)
    off = codes.view(torch.uint8) != _want(x, q)
    assert off.sum() <= 1, off.sum()


@pytest.mark.parametrize("q", sorted(ref.FP8))
def test_infinity_and_nan(fo, q):
    q = ref.FP8[q]
    x = torch.randn((4, 256), device="cuda")
    x[0, 5], x[1, 200], x[2, 7] = float("inf"), float("-inf"), float("nan")
    for codes, scale in (fo.quantize_blocks(x, q), fo.quantize_blocks(x.t().contiguous().t(), q)):
        values = codes.float()
        assert scale[0, 0] == scale[1, 1] == float("inf") and scale[2, 0].isnan() and scale.isfinite().sum() == 5
        assert values[0, 5].isnan() and values[1, 200].isnan() and values[2, :128].isnan().all()
        values[0, 5] = values[1, 200] = 0
        assert (values[0, :128] == 0).all() and (values[1, 128:] == 0).all() and values[3].isfinite().all()
