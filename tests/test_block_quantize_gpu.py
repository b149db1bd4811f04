"""Quantization to blocks of 128 against its definition in 64 bits: rows, squares and transposed blocks, every type, odd
sizes, strides, zeros, the smallest and the largest values, infinities and NaN."""

import pytest
import torch

import block_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(1, 1), (1, 128), (3, 129), (5, 7), (16, 256), (127, 130), (128, 128), (129, 300), (200, 1000)]


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _data(m, n, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn((m, n), generator=g, device="cuda") * torch.randn((m, 1), generator=g, device="cuda").exp()).to(dtype)


@pytest.mark.parametrize("q", sorted(ref.FP8))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_rows_and_squares(fo, m, n, dtype, q):
    x = _data(m, n, dtype)
    ref.check_quantized(x, *fo.quantize_blocks(x, ref.FP8[q]))
    ref.check_quantized(x, *fo.quantize_blocks(x, ref.FP8[q], square=True), square=True)


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_tiles(fo, m, n, dtype, square):
    """One reading for both directions and the column sums, and each alone: the same bits."""
    x = _data(m, n, dtype, 1)
    tiles = torch.ops.feather_ops.quantize_tiles.default
    both = tiles(x, False, square, True, True, True)
    ref.check_quantized(x, both[0], both[1], square)
    ref.check_quantized(x.t(), both[2], both[3], square)
    # 32 additions a lane, 3 across the waves
    parts = torch.stack([c.double().sum(0) for c in x.split(128)])
    sizes = torch.stack([c.double().abs().sum(0) for c in x.split(128)])
    ref.check_close(both[4], parts, 35 * 2.0**-24 * sizes)
    for k, wanted in enumerate([(True, False, False), (False, True, False), (False, False, True)]):
        one = tiles(x, False, square, *wanted)
        for i in ((0, 1), (2, 3), (4,))[k]:
            assert torch.equal(one[i].float(), both[i].float())
    ref.check_close(torch.ops.feather_ops.sum_rows.default(both[4], 2), x.double().sum(0),
                    (35 + parts.shape[0]) * 2.0**-23 * x.double().abs().sum(0))


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_batches(fo, dtype):
    wide = _data(40, 700, dtype, 2)
    for view in (wide[:, 3:300], wide[::2, :256], wide[:, 8:264], wide.t()[:300], wide[5:6, 1:], wide[:1].expand(9, 700)):
        for got in (fo.quantize_blocks(view), torch.ops.feather_ops.quantize_tiles.default(
                view if view.stride(1) == 1 and view.stride(0) else view.contiguous(), False, False, True, False, False)[:2]):
            ref.check_quantized(view, *got)
    x = _data(6, 200, dtype, 3).view(2, 3, 200)
    codes, scale = fo.quantize_blocks(x)
    assert codes.shape == x.shape and scale.shape == (2, 3, 2)
    ref.check_quantized(x.view(6, 200), codes.reshape(6, 200), scale.reshape(6, 2))


@pytest.mark.parametrize("q", sorted(ref.FP8))
def test_every_bf16_magnitude(fo, q):
    """Rows of one block each, whose largest value runs over every finite bf16 magnitude, subnormals among them."""
    bits = torch.arange(0x7f80, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.bfloat16)
    x = torch.zeros((bits.numel(), 8), dtype=torch.bfloat16, device="cuda")
    x[:, 3], x[:, 5] = bits, -bits * 0.3
    ref.check_quantized(x, *fo.quantize_blocks(x, ref.FP8[q]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("square", [False, True])
def test_not_finite(fo, dtype, square):
    """A NaN makes its block NaN, an infinity its scale infinite and its code NaN; other blocks keep their bits."""
    x = _data(300, 400, dtype, 4)
    clean = fo.quantize_blocks(x, square=square)
    x[7, 130], x[200, 5], x[299, 399] = float("nan"), float("inf"), float("-inf")
    codes, scale = fo.quantize_blocks(x, square=square)
    rows = [r // 128 if square else r for r in (7, 200, 299)]
    assert scale[rows[0], 1].isnan() and codes[7, 128:256].isnan().all()
    assert scale[rows[1], 0] == float("inf") and codes[200, 5].isnan() and (codes[200, :5].float() == 0).all()
    assert scale[rows[2], 3] == float("inf") and codes[299, 399].isnan()
    keep = torch.ones_like(scale, dtype=torch.bool)
    keep[rows, [1, 0, 3]] = False
    assert torch.equal(scale[keep], clean[1][keep])
    keep = ref.spread(keep, 300, 400)
    assert torch.equal(codes.float()[keep], clean[0].float()[keep])
    transposed = torch.ops.feather_ops.quantize_tiles.default(x, False, square, False, True, False)
    want = torch.ops.feather_ops.quantize_tiles.default(x.t().contiguous(), False, square, True, False, False)
    assert torch.equal(transposed[3].nan_to_num(-1.0), want[1].nan_to_num(-1.0))
    assert torch.equal(transposed[2].float().nan_to_num(-1.0), want[0].float().nan_to_num(-1.0))


def test_past_4_gib(fo):
    """Elements past 32-bit offsets: the last rows of a matrix of 2^32 + some bytes."""
    m, n = 1 << 15, (1 << 16) + 256
    x = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    x[-2:] = _data(2, n, torch.bfloat16, 5)
    codes, scale = fo.quantize_blocks(x)
    ref.check_quantized(x[-2:], codes[-2:], scale[-2:])
    assert (codes[-3].float() == 0).all()
    _, _, codes_t, scale_t, _ = torch.ops.feather_ops.quantize_tiles.default(x, False, False, False, True, False)
    ref.check_quantized(x[-128:].t(), codes_t[:, -128:], scale_t[:, -1:])


def test_refusals(fo):
    x = torch.zeros((4, 8), device="cuda")
    with pytest.raises(ValueError, match="fp8 dtype"):
        fo.quantize_blocks(x, torch.float16)
    with pytest.raises(RuntimeError, match="bfloat16, float16 or float32"):
        fo.quantize_blocks(x.double())
    with pytest.raises(ValueError, match="matrix"):
        fo.quantize_blocks(x[None], square=True)
    with pytest.raises(NotImplementedError):
        fo.quantize_blocks(x.cpu())


@pytest.mark.parametrize("shape", [(0, 128), (4, 0), (0, 0), (2, 0, 128)])
def test_empty(fo, shape):
    codes, scale = fo.quantize_blocks(torch.zeros(shape, device="cuda"))
    assert codes.shape == shape and scale.shape == (*shape[:-1], ref.blocks(shape[-1]))
