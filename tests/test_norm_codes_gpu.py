"""The codes of a normed row: its norm is a factor of values and scale alike, so codes do not depend on how it was rounded."""

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


def _want(x, w, residual, q, eps):
    y, _, _ = ref.rms_norm(x, w, residual, eps)
    scale = ref.largest(y).clamp(min=2.0**-100) / ref.LARGEST[q]
    return (y / ref.spread(scale, *y.shape)).float().to(q).view(torch.uint8)


@pytest.mark.parametrize("q", sorted(ref.FP8))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n", [(700, 128), (300, 1000), (40, 4096), (200, 5120), (3, 11352), (5, 20000)])
def test_every_code(fo, m, n, dtype, q):
    """16-bit rows and weights, whose products are exact in fp32: every code is the 64-bit definition's."""
    g = torch.Generator("cuda").manual_seed(m)
    x, res = (torch.randn((m, n), generator=g, device="cuda").to(dtype) for _ in range(2))
    w = (1 + torch.randn(n, generator=g, device="cuda") * 0.1).to(dtype)
    q = ref.FP8[q]
    for residual in (None, res):
        codes = fo.rms_norm_quantized(x, w, residual, 1e-6, q)[0]
        assert torch.equal(codes.view(torch.uint8), _want(x, w, residual, q, 1e-6))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_blocks_under_the_floor(fo, dtype):
    """Scales at their floor: codes are value over 2^-100 / L, near zero."""
    x = torch.ones((3, 384), device="cuda")
    x[:, 128:256] = 2.0**-110
    x[1, 128:256] = 0
    x[2, 200] = 2.0**-90
    x = x.to(dtype)
    w = torch.ones(384, device="cuda", dtype=dtype)
    codes, scale = fo.rms_norm_quantized(x, w, None, 0.0)
    want, _, _ = ref.rms_norm(x, w, None, 0.0)
    exact = ref.largest(want).clamp(min=2.0**-100) / 448
    ref.check_close(scale, exact, ref.norm_slack(384) * exact)
    quotient = want / ref.spread(exact, 3, 384)
    low, high = ((quotient * (1 + d)).to(codes.dtype).float() for d in (-(2.0**-20), 2.0**-20))
    assert bool(((codes.float() == low) | (codes.float() == high)).all())
    assert scale[0, 1] == scale[1, 1] == 2.0**-100 / 448 and scale[2, 1] > scale[0, 1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_infinity_and_nan(fo, dtype):
    """A row with an infinity has a norm of zero: its own block is NaN, the others are zero; a NaN reaches the whole row."""
    x = torch.randn((3, 300), device="cuda")
    x[0, 5], x[1, 299] = float("inf"), float("nan")
    codes, scale = fo.rms_norm_quantized(x.to(dtype), torch.ones(300, device="cuda", dtype=dtype))
    assert scale[0, 0].isnan() and codes[0, :128].float().isnan().all()
    assert (scale[0, 1:] == 2.0**-100 / 448).all() and (codes[0, 128:].float() == 0).all()
    assert scale[1].isnan().all() and codes[1].float().isnan().all()
    assert scale[2].isfinite().all() and codes[2].float().isfinite().all()
