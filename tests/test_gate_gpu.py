"""The gated activation, its fp8 output and its gradient against 64 bits."""

import pytest
import torch

import block_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(1, 1), (3, 5), (1, 128), (17, 129), (5, 1000), (64, 136), (2, 14336), (300, 777), (33, 2048)]
# exp in fp32 of an argument g: its own error and the argument's rounding before it, |g| <= 104 (past that s is 0 or 1);
# the division, the sum and two products. The definition's scale of errors is |g u| times the least representable part.
SLACK = 2.0**-24 * 16


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _data(m, n, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn((m, n), generator=g, device="cuda") * 2).to(dtype)


def _slack(x, want):
    """16 roundings, and exp's argument error of |g| 2^-23."""
    g = x.double().chunk(2, -1)[0]
    return (SLACK + g.abs() * 2.0**-22) * want.abs() + 2.0**-126 * (1 + x.double().abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_forward(fo, m, n, dtype):
    x = _data(m, 2 * n, dtype)
    y = fo.silu_mul(x)
    want = ref.silu(x)
    assert y.dtype == dtype
    ref.check_close(y, want, _slack(x, want))
    batch = fo.silu_mul(x.view(1, m, 2 * n))
    assert batch.shape == (1, m, n) and torch.equal(batch[0], y)


@pytest.mark.parametrize("q", sorted(ref.FP8))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_quantized(fo, m, n, dtype, q):
    x = _data(m, 2 * n, dtype, 3)
    codes, scale = fo.silu_mul_quantized(x, ref.FP8[q])
    want = ref.silu(x)
    slack = SLACK + 2.0**-22 * x.double().abs().max().item()
    exact = ref.largest(want).clamp(min=2.0**-100) / ref.LARGEST[ref.FP8[q]]
    ref.check_close(scale, exact, slack * exact)
    quotient = want / ref.spread(scale.double(), m, n)
    low, high = ((quotient * (1 + d)).to(codes.dtype).float() for d in (-2 * slack - 2.0**-22, 2 * slack + 2.0**-22))
    assert codes.dtype == ref.FP8[q] and bool(((codes.float() == low) | (codes.float() == high)).all())


def _grad(x, gy):
    """The gradient in 64 bits and its bound: sums of two terms, each with the forward's error."""
    g, u = x.double().chunk(2, -1)
    s, gy = torch.sigmoid(g), gy.double()
    grad = torch.cat([gy * u * s * (1 + g * (1 - s)), gy * g * s], -1)
    size = torch.cat([(gy * u * s).abs() * (1 + g.abs()), (gy * g * s).abs()], -1)
    return grad, (SLACK + torch.cat([g, g], -1).abs() * 2.0**-22) * size + 2.0**-126 * (1 + x.double().abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_gradient_against_the_formula(fo, m, n, dtype):
    x, gy = _data(m, 2 * n, dtype, 5).requires_grad_(), _data(m, n, dtype, 6)
    got, = torch.autograd.grad(fo.silu_mul(x), x, gy)
    ref.check_close(got, *_grad(x.detach(), gy))


def test_gradient_against_differences(fo):
    """Along a random direction in fp32: the step's own error from the 64-bit form, the outputs' rounding over the step."""
    m, n, step = 7, 300, 2.0**-6
    x, gy, along = _data(m, 2 * n, torch.float32, 7), _data(m, n, torch.float32, 8), _data(m, 2 * n, torch.float32, 9)
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(fo.silu_mul(leaf), leaf, gy)
    grad, slack = _grad(x, gy)
    up, down = (fo.silu_mul(x + s * along).double() for s in (step, -step))
    up64, down64 = (ref.silu(x + s * along) for s in (step, -step))
    own = abs(((up64 - down64) * gy).sum() / (2 * step) - (grad * along).sum())
    noise = (2 * _slack(x, up64) + 2.0**-23 * up64.abs()).mul(gy.abs()).sum() / step
    assert abs(((up - down) * gy).sum() / (2 * step) - (got.double() * along).sum()) <= own + noise + (slack * along.abs()).sum()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(fo, dtype):
    wide = _data(40, 1200, dtype, 11)
    for view in (wide[:, 3:603], wide[::2, :512], wide.t()[:200], wide[:1].expand(5, 1200), wide[:, 8:40]):
        want = ref.silu(view)
        ref.check_close(fo.silu_mul(view), want, _slack(view, want))
    leaf = wide.clone().requires_grad_()
    gy = _data(600, 40, dtype, 12).t()
    got, = torch.autograd.grad(fo.silu_mul(leaf), leaf, gy)
    ref.check_close(got, *_grad(wide, gy))


def test_large_and_not_finite_gates(fo):
    inf = float("inf")
    g = torch.tensor([-1e4, -200.0, -88.0, 0.0, 88.0, 1e4, inf, float("nan")], device="cuda")
    y = fo.silu_mul(torch.cat([g, torch.full_like(g, 2.0)])[None])[0]
    assert (y[:2] == 0).all() and y[3] == 0 and y[5] == 2e4 and y[6] == inf and y[7].isnan()
    assert y[2].item() == pytest.approx(2 * -88 * 6.0546e-39, rel=1e-3, abs=1.2e-38)
    _, scale = fo.silu_mul_quantized(torch.cat([g, torch.full_like(g, 2.0)])[None])
    assert scale.isnan().all()


def test_past_4_gib(fo):
    m, n = (1 << 17) + 5, 8192
    x = torch.zeros((m, 2 * n), dtype=torch.bfloat16, device="cuda")
    x[-2:] = _data(2, 2 * n, torch.bfloat16, 13)
    want = ref.silu(x[-2:])
    ref.check_close(fo.silu_mul(x)[-2:], want, _slack(x[-2:], want))


def test_refusals(fo):
    x = torch.zeros((4, 64), device="cuda")
    for call in (fo.silu_mul, fo.silu_mul_quantized):
        with pytest.raises(ValueError, match="x must be"):
            call(x.double())
        with pytest.raises(ValueError, match="even"):
            call(x[:, :63])
        with pytest.raises(NotImplementedError):
            call(x.cpu())
    with pytest.raises(ValueError, match="fp8 dtype"):
        fo.silu_mul_quantized(x, torch.uint8)


@pytest.mark.parametrize("shape", [(0, 64), (3, 0)])
def test_empty(fo, shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    y = fo.silu_mul(x)
    assert y.shape == (shape[0], shape[1] // 2)
    assert torch.autograd.grad(y.sum(), x)[0].shape == shape
    codes, scale = fo.silu_mul_quantized(x)
    assert codes.shape == y.shape and scale.shape == (shape[0], ref.blocks(y.shape[1]))
