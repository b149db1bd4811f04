"""The root-mean-square norm with the residual's addition, its fp8 output and its gradients against 64 bits."""

import pytest
import torch

import block_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# One value, less than a piece, one wave's rows, the workgroup's, and rows past its registers; odd lengths of each.
SHAPES = [(1, 1), (3, 5), (2, 128), (5, 500), (1, 512), (9, 1000), (7, 1024), (130, 2048), (4, 2050), (3, 4096), (600, 4100),
          (2, 6144), (5, 8192), (3, 12345), (2, 16384), (3, 16392), (70, 20001)]


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _randn(seed, *shape):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def _inputs(m, n, dtype, seed=0):
    x, res = _randn(seed, m, n).to(dtype), (_randn(seed + 1, m, n) * 3).to(dtype)
    return x, (1 + 0.3 * _randn(seed + 2, n)).to(dtype), res


def _check(y, x, w, res, eps):
    want, h, _ = ref.rms_norm(x, w, res, eps)
    ref.check_close(y, want, ref.norm_slack(x.shape[-1]) * want.abs())
    return h


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_forward(fo, m, n, dtype):
    x, w, res = _inputs(m, n, dtype)
    _check(fo.rms_norm(x, w), x, w, None, 1e-6)
    y, h = fo.rms_norm(x, w, res, 1e-2)
    assert torch.equal(h, _check(y, x, w, res, 1e-2))
    wide = w.float() * 1.001   # a weight kept in fp32
    y, _ = fo.rms_norm(x, wide, res)
    _check(y, x, wide, res, 1e-6)


@pytest.mark.parametrize("q", sorted(ref.FP8))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_quantized(fo, m, n, dtype, q):
    """The scale is within the norm's error of its definition, and each code the nearest of a value within it."""
    x, w, res = _inputs(m, n, dtype, 5)
    for residual in (None, res):
        got = fo.rms_norm_quantized(x, w, residual, 1e-6, ref.FP8[q])
        want, h, _ = ref.rms_norm(x, w, residual, 1e-6)
        codes, scale = got[:2]
        assert codes.dtype == ref.FP8[q] and (residual is None or torch.equal(got[2], h))
        slack = ref.norm_slack(n)
        exact = ref.largest(want).clamp(min=2.0**-100) / ref.LARGEST[ref.FP8[q]]
        ref.check_close(scale, exact, slack * exact)
        quotient = want / ref.spread(scale.double(), m, n)
        low, high = ((quotient * (1 + d)).to(codes.dtype).float() for d in (-2 * slack - 2.0**-22, 2 * slack + 2.0**-22))
        assert bool(((codes.float() == low) | (codes.float() == high)).all())


def _grad_reference(x, w, res, gy, gh, eps):
    """Gradients in 64 bits and the bounds of their fp32 kernels: the mean is a sum like the norm's, each of the other steps
    a rounding; the weight's gradient a sum over rows."""
    n = x.shape[-1]
    _, h, r = ref.rms_norm(x, w, res, eps)
    normed, g = h.double() * r, gy.double() * w.double()
    mean, mean_size = (g * normed).mean(-1, keepdim=True), (g * normed).abs().mean(-1, keepdim=True)
    grad = r * (g - normed * mean)
    size = r * (g.abs() + normed.abs() * mean_size)
    if gh is not None:
        grad, size = grad + gh.double(), size + gh.double().abs()
    slack = 4 * ref.norm_slack(n) * size
    gw, gw_size = (gy.double() * normed).sum(0), (gy.double() * normed).abs().sum(0)
    return grad, slack, gw, (x.shape[0] * 2.0**-23 + 2 * ref.norm_slack(n)) * gw_size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_gradients_against_the_formula(fo, m, n, dtype):
    x, w, res = _inputs(m, n, dtype, 10)
    gy, gh = _randn(20, m, n).to(dtype), _randn(21, m, n).to(dtype)
    for residual, gh_in, weight in ((None, None, w), (res, gh, w), (res, None, w.float())):
        leaves = [t.clone().requires_grad_() for t in (x, weight)] + ([residual.clone().requires_grad_()] if residual is not None
                                                                       else [])
        out = fo.rms_norm(leaves[0], leaves[1], leaves[2] if residual is not None else None, 1e-3)
        outs, grads = ([out], [gy]) if residual is None else (list(out), [gy, gh_in])
        if gh_in is None:
            outs, grads = outs[:1], grads[:1]
        got = torch.autograd.grad(outs, leaves, grads)
        grad, slack, gw, gw_slack = _grad_reference(x, weight, residual, gy, gh_in, 1e-3)
        ref.check_close(got[0], grad, slack, "x")
        ref.check_close(got[1], gw, gw_slack, "weight")
        assert got[1].dtype == weight.dtype
        if residual is not None:
            assert torch.equal(got[2], got[0])


@pytest.mark.parametrize("n", [40, 3000])
def test_gradients_against_differences(fo, n):
    """Along a random direction in fp32. The quotient of central differences has the step's own error, which the 64-bit
    formula gives, and the outputs' rounding: the norm's error of each over the step."""
    m, step, eps = 6, 2.0**-6, 1e-3
    x, w, res = _inputs(m, n, torch.float32, 30)
    gy, gh = _randn(40, m, n), _randn(41, m, n)
    along = [_randn(50 + i, *t.shape) for i, t in enumerate((x, w, res))]
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    got = torch.autograd.grad(fo.rms_norm(*leaves, eps), leaves, (gy, gh))
    slope = sum((g.double() * d.double()).sum() for g, d in zip(got, along))

    def moved(f, s):
        y, h = f(*(t + s * d for t, d in zip((x, w, res), along)))
        return (y.double() * gy.double()).sum() + (h.double() * gh.double()).sum(), \
            (y.double() * gy.double()).abs().sum() + (h.double() * gh.double()).abs().sum()

    def plain(x, w, res):
        y, h, _ = ref.rms_norm(x, w, res, eps)
        return y, h

    up, size = moved(lambda *t: fo.rms_norm(*t, eps), step)
    down, _ = moved(lambda *t: fo.rms_norm(*t, eps), -step)
    up64, _ = moved(plain, step)
    down64, _ = moved(plain, -step)
    grad, slack, gw, gw_slack = _grad_reference(x, w, res, gy, gh, eps)
    slope64 = (grad * (along[0] + along[2]).double()).sum() + (gw * along[1].double()).sum()
    own = abs((up64 - down64) / (2 * step) - slope64)
    noise = 4 * ref.norm_slack(n) * size / step
    grads = (slack * (along[0].abs() + along[2].abs()).double()).sum() + (gw_slack * along[1].abs().double()).sum()
    assert abs((up - down) / (2 * step) - slope) <= own + noise + grads


def test_only_what_is_asked_for(fo):
    m, n = 40, 300
    x, w, res = _inputs(m, n, torch.bfloat16, 60)
    gy, gh = _randn(61, m, n).bfloat16(), _randn(62, m, n).bfloat16()
    every = [t.clone().requires_grad_() for t in (x, w, res)]
    want = torch.autograd.grad(fo.rms_norm(*every), every, (gy, gh))
    for which in range(3):
        args = [x, w, res]
        args[which] = args[which].clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(fo.rms_norm(*args), args[which], (gy, gh))[0], want[which])
    args = [t.clone().requires_grad_() for t in (x, w, res)]
    gx, gw, gr = torch.autograd.grad(fo.rms_norm(*args)[1], args, gh, allow_unused=True)   # h alone
    assert torch.equal(gx, gh) and gw is None and torch.equal(gr, gh)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_batches(fo, dtype):
    wide, w, other = _inputs(50, 900, dtype, 70)
    for view, res in ((wide[:, 3:600], other[:, 5:602]), (wide[::3], other[1::3]), (wide.t()[:200], other.t()[1:201]),
                      (wide[:1].expand(6, 900), other[:6]), (wide[:, 8:520], other[:, :512])):
        ww = w[: view.shape[1]] if view.shape[1] <= 900 else None
        y, h = fo.rms_norm(view, ww, res)
        assert torch.equal(h, _check(y, view, ww, res, 1e-6))
    ww = torch.stack([w, w], 1)[:, 0]   # a weight apart
    _check(fo.rms_norm(wide, ww), wide, w, None, 1e-6)
    x = wide.view(5, 10, 900)
    y, h = fo.rms_norm(x, w, other.view(5, 10, 900))
    assert y.shape == h.shape == x.shape
    _check(y.view(50, 900), wide, w, other, 1e-6)
    leaf = x.clone().requires_grad_()
    gy = _randn(71, 900, 10, 5).to(dtype).permute(2, 1, 0)   # a gradient in another order
    got, = torch.autograd.grad(fo.rms_norm(leaf, w), leaf, gy)
    grad, slack, _, _ = _grad_reference(wide, w, None, gy.reshape(50, 900), None, 1e-6)
    ref.check_close(got.view(50, 900), grad, slack)


def test_zero_rows_and_values_that_are_not_finite(fo):
    x = _randn(80, 6, 700)
    w = torch.ones(700, device="cuda")
    x[1] = 0
    x[2, 650], x[3, 0] = float("nan"), float("inf")
    x[4] *= 1e-30
    y = fo.rms_norm(x, w)
    assert (y[1] == 0).all() and y[2].isnan().all() and y[3, 0].isnan() and (y[3, 1:] == 0).all()
    _check(y[[0, 4, 5]], x[[0, 4, 5]], w, None, 1e-6)
    codes, scale = fo.rms_norm_quantized(x, w)
    assert scale[2].isnan().all() and scale[[0, 1, 4, 5]].isfinite().all() and (codes[1].float() == 0).all()
    assert fo.rms_norm(x[1:2], w, None, 0.0).isnan().all()   # 0 / 0


def test_past_4_gib(fo):
    m, n = (1 << 19) + 3, 4096
    x = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    x[-2:] = _randn(90, 2, n).bfloat16()
    w = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = fo.rms_norm(x, w)
    _check(y[-2:], x[-2:], w, None, 1e-6)
    assert (y[-3] == 0).all()


def test_streams_and_graphs(fo):
    x, w, res = _inputs(64, 1024, torch.bfloat16, 95)
    graph = torch.cuda.CUDAGraph()
    fo.rms_norm_quantized(x, w, res)
    with torch.cuda.graph(graph):
        held = fo.rms_norm_quantized(x, w, res)
    for replay in range(4):
        new = _inputs(64, 1024, torch.bfloat16, 100 + replay)
        for mine, other in zip((x, w, res), new):
            mine.copy_(other)
        want = fo.rms_norm_quantized(*new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a.float(), b.float())


def test_refusals(fo):
    x, w, res = _inputs(4, 64, torch.bfloat16)
    for call in (fo.rms_norm, fo.rms_norm_quantized):
        with pytest.raises(ValueError, match="x must be"):
            call(x.double(), w)
        with pytest.raises(ValueError, match="weight must be"):
            call(x, w[:-1])
        with pytest.raises(ValueError, match="residual must have"):
            call(x, w, res.float())
        with pytest.raises(ValueError, match="residual must have"):
            call(x, w, res[:-1])
        with pytest.raises(RuntimeError, match="weight must have"):
            call(x, w.half())
        with pytest.raises(NotImplementedError):
            call(x.cpu(), w.cpu())
    with pytest.raises(ValueError, match="fp8 dtype"):
        fo.rms_norm_quantized(x, w, None, 1e-6, torch.bfloat16)


def test_empty(fo):
    x = torch.zeros((0, 64), device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, h = fo.rms_norm(x, w, x)
    assert y.shape == h.shape == (0, 64)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == (0, 64) and (gw == 0).all()
    codes, scale, h = fo.rms_norm_quantized(x, w, x)
    assert codes.shape == (0, 64) and scale.shape == (0, 1) and h.shape == (0, 64)
