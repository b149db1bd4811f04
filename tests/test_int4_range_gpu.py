"""Few rows of 4-bit products at the ends of their types' ranges, and the sums of codes as they are: exact where fp32 holds them."""

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu
ROWS = [1, 9, 24, 50]   # of each kernel for few rows
GROUPS = [(32, True), (64, False), (64, True), (128, False), (128, True)]


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _weight(n, k, group, zeros, dtype, scale, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
    zero = torch.randint(0, 16, (groups, n), generator=g, device="cuda", dtype=torch.uint8).t() if zeros else None
    return codes, torch.full((groups, n), scale, dtype=dtype, device="cuda").t(), zero


def _same(got, want):
    """Infinities, their signs, and NaN where the definition has them."""
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.double().nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0) * got.isinf(),
                       want.nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0) * want.isinf())


@pytest.mark.parametrize("group,zeros", GROUPS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m", ROWS)
def test_infinite_inputs(fo, m, dtype, group, zeros):
    """An infinity gives infinities of its weights' signs, and NaN where those are zero."""
    weight = _weight(40, 300, group, zeros, dtype, 0.01)
    x = torch.randn(m, 300, device="cuda").to(dtype)
    for row in range(0, m, 2):
        x[row, (37 * row + 5) % 300] = float("inf") if row % 4 else float("-inf")
    want = x.double() @ ref.int4_values(*weight, 300).t()
    assert want.isinf().any() and want.isnan().any()
    _same(fo.int4_linear(x, *weight), want)
    gate, up = want.chunk(2, 1)
    plain = (gate > 20) & up.isfinite() & (up != 0)   # gates past the activation's bend, where it is the gate itself
    got = fo.int4_gated_linear(x, *weight)
    _same(got[plain & gate.isinf()], (gate * up)[plain & gate.isinf()])
    assert torch.equal((gate.isnan() | up.isnan()) & ~got.isnan(), torch.zeros_like(got, dtype=torch.bool))


@pytest.mark.parametrize("group,zeros", GROUPS)
@pytest.mark.parametrize("m", ROWS)
def test_largest_inputs(fo, m, group, zeros):
    """Rows of bfloat16's largest and lowest values: sums of them times codes pass fp32's range, results do not."""
    dtype, k = torch.bfloat16, 520
    weight = _weight(40, k, group, zeros, dtype, 2.0**-14)
    x = torch.full((m, k), torch.finfo(dtype).max, dtype=dtype, device="cuda")
    x[1::2] = torch.finfo(dtype).min
    want, bound = ref.int4(x, *weight, None)
    assert want.abs().max() < torch.finfo(dtype).max / 2
    ref.check(fo.int4_linear(x, *weight), want, bound)


@pytest.mark.parametrize("group,zeros", GROUPS)
@pytest.mark.parametrize("exponent", [-118, -124])
@pytest.mark.parametrize("m", ROWS)
def test_smallest_inputs(fo, m, exponent, group, zeros):
    """bfloat16's least values: no product of one with a code is lost where results have a place for it."""
    dtype, k = torch.bfloat16, 300
    weight = _weight(40, k, group, zeros, dtype, 1.0)
    x = (torch.randn(m, k, device="cuda") * 2.0**exponent).to(dtype)
    want, bound = ref.int4(x, *weight, None)
    # terms are multiples of fp32's least value, 2^-149, in the sums' unit of 2048: each may be off by half of one
    ref.check(fo.int4_linear(x, *weight), want, bound + k * 2.0**-150 * 2048)


@pytest.mark.parametrize("group,zeros", GROUPS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m", ROWS)
def test_sums_that_fp32_holds_are_exact(fo, m, dtype, group, zeros):
    """In every 32 columns large values that cancel, beside small ones: integers, whose partial sums are under 2^24 in any order. What is left is
    the small ones' sum, and only its rounding may be off."""
    g = torch.Generator("cuda").manual_seed(m)
    k, n, blocks = 512, 48, 16
    # up to 255 * 2^5 (fp16 holds them), 12 to a block and their opposites, times 2 at most in size
    large = torch.randint(128, 256, (m, blocks, 12), generator=g, device="cuda") * 2 ** torch.randint(0, 6, (m, blocks, 12), generator=g, device="cuda")
    large = large * (2 * torch.randint(0, 2, large.shape, generator=g, device="cuda") - 1)
    x = torch.cat((large, torch.randint(-3, 4, (m, blocks, 8), generator=g, device="cuda"), -large.flip(2)), 2).view(m, k).to(dtype)
    z = torch.randint(2, 14, (n, 1), generator=g, device="cuda") if zeros else 8
    q = torch.randint(-2, 3, (n, blocks, 16), generator=g, device="cuda")
    q = torch.cat((q, q.flip(2)), 2).view(n, k) + z   # the same codes for a value and its opposite
    codes = (q[:, ::2] | q[:, 1::2] << 4).to(torch.uint8)
    groups = k // group
    scale = torch.full((groups, n), 0.25, dtype=dtype, device="cuda").t()
    zero = z.to(torch.uint8).repeat(1, groups).t().contiguous().t() if zeros else None
    want = x.double() @ ref.int4_values(codes, scale, zero, k).t()
    assert 24 * 2 * 255 * 32 * (128 // 32) < 1 << 24 and want.abs().max() < 600
    assert torch.equal(fo.int4_linear(x, codes, scale, zero), want.to(dtype))
