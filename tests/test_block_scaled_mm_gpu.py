"""The block-scaled fp8 product and its layer against 64 bits: sizes around every tile, formats, strides, scales by square
and by row, zeros, infinities and NaN, streams and graphs; gradients against the formulas and against differences."""

import pytest
import torch

import block_ref as ref

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _randn(m, n, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn((m, n), generator=g, device="cuda")


def _operands(fo, m, n, k, a="e4m3", b="e4m3", by_row=False, seed=0):
    qa = fo.quantize_blocks(_randn(m, k, seed), ref.FP8[a])
    qb = fo.quantize_blocks(_randn(n, k, seed + 1) * 0.1, ref.FP8[b], square=not by_row)
    return *qa, *qb


def _check(fo, operands, bias=None, dtype=BF16):
    got = fo.block_scaled_mm(*operands, bias, dtype)
    assert got.dtype == dtype
    want, slack = ref.mm(*operands, bias)
    ref.check_close(got, want, slack, tuple(operands[0].shape) + tuple(operands[2].shape))
    return got


SIZES = [(1, 1, 1), (1, 128, 128), (1, 1000, 2560), (2, 15, 16), (5, 17, 100), (16, 16, 128), (17, 129, 129), (33, 64, 272),
         (31, 255, 1024), (63, 300, 640), (64, 256, 4096), (65, 127, 384), (100, 500, 2000), (128, 128, 128),
         (129, 130, 136), (255, 257, 512), (256, 256, 256), (257, 513, 1040), (300, 1000, 900), (512, 640, 128),
         (1000, 264, 768), (1, 5000, 72), (300, 2, 5000), (16, 4100, 16384), (128, 1024, 8192), (700, 700, 3001)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes(fo, m, n, k, by_row, dtype):
    operands = _operands(fo, m, n, k, by_row=by_row)
    _check(fo, operands, dtype=dtype)
    _check(fo, operands, _randn(1, n, 9)[0].to(dtype), dtype)


@pytest.mark.parametrize("a", sorted(ref.FP8))
@pytest.mark.parametrize("b", sorted(ref.FP8))
@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 300, 700), (20, 96, 512), (48, 200, 384), (130, 260, 640), (600, 1100, 1500)])
def test_formats(fo, m, n, k, a, b, by_row):
    _check(fo, _operands(fo, m, n, k, a, b, by_row, seed=3), dtype=FP32)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_layouts(fo, m):
    """Rows apart with NaN codes between them, scales in either order or strided, rows that start anywhere."""
    k, n = 200, 136
    a, sa, b, sb = _operands(fo, m, n, k, seed=5)
    want = _check(fo, (a, sa, b, sb))
    nan = torch.full((m + n, 512), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    wide_a, wide_b = nan[:m, 16:216], nan[m:, 32:232]
    wide_a.copy_(a)
    wide_b.copy_(b)
    far = torch.full((2, m, 4), float("nan"), device="cuda")
    far[1, :, ::2] = sa
    for aa in (a, a.contiguous(), wide_a, torch.cat([a[:, :1], a], 1)[:, 1:], a.t().contiguous().t()):
        for ss in (sa, sa.contiguous(), far[1, :, ::2]):
            assert torch.equal(fo.block_scaled_mm(aa, ss, wide_b, sb.contiguous()), want)


def test_sizes_agree_with_one_another(fo):
    """Rows do not depend on the rows beside them but for the order of their sums, and the same call gives the same bits."""
    a, sa, b, sb = _operands(fo, 700, 384, 2048, seed=7)
    whole = _check(fo, (a, sa, b, sb), dtype=FP32)
    for rows in (1, 16, 50, 200):
        part = _check(fo, (a[:rows], sa[:rows], b, sb), dtype=FP32)
        assert torch.equal(part, fo.block_scaled_mm(a[:rows], sa[:rows], b, sb, None, FP32))
        assert (part - whole[:rows]).abs().max() <= 2 * ref.mm(a[:rows], sa[:rows], b, sb)[1].max()


@pytest.mark.parametrize("m", [1, 33, 200])
def test_zero_infinite_and_nan_blocks(fo, m):
    """A row's NaN or infinity stays in its row, a weight's in the columns of its square; blocks of zeros add nothing."""
    n, k = 300, 500
    x, w = _randn(m, k, 11), _randn(n, k, 12)
    x[:, 128:256] = 0
    x[0, 300] = float("inf")
    x[m - 1, 20] = float("nan")
    w[128:256, 384:] = 0
    w[299, 0] = float("nan")
    y = fo.block_scaled_mm(*fo.quantize_blocks(x), *fo.quantize_blocks(w, square=True), None, FP32)
    bad_row = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad_row[0] = bad_row[m - 1] = True
    assert y[bad_row].isnan().all() and y[:, 256:].isnan().all()
    assert y[~bad_row][:, :256].isfinite().all()
    zero = fo.block_scaled_mm(*fo.quantize_blocks(x * 0 if m == 33 else torch.zeros_like(x)),
                              *fo.quantize_blocks(_randn(n, k, 13), square=True), None, FP32)
    if m != 33:
        assert (zero == 0).all()


@pytest.mark.parametrize("m,n,k", [(0, 5, 128), (4, 0, 128), (3, 5, 0), (0, 0, 0)])
def test_empty(fo, m, n, k):
    a = torch.zeros((m, k), dtype=torch.float8_e4m3fn, device="cuda")
    b = torch.zeros((n, k), dtype=torch.float8_e4m3fn, device="cuda")
    sa, sb = torch.ones((m, ref.blocks(k)), device="cuda"), torch.ones((ref.blocks(n), ref.blocks(k)), device="cuda")
    bias = torch.arange(n, device="cuda").to(BF16)
    assert torch.equal(fo.block_scaled_mm(a, sa, b, sb, bias), bias.expand(m, n))
    assert torch.equal(fo.block_scaled_mm(a, sa, b, sb), torch.zeros((m, n), dtype=BF16, device="cuda"))


def test_weight_past_4_gib(fo):
    """The last columns of a weight of more than 2^32 bytes."""
    n, k = (1 << 16) + 130, 1 << 16
    b = torch.zeros((n, k), dtype=torch.uint8, device="cuda")
    tail, tail_scale = fo.quantize_blocks(_randn(130, k, 20), square=True)
    b[-130:] = tail.view(torch.uint8)
    sb = torch.ones((ref.blocks(n), k // 128), device="cuda")
    sb[-2:] = tail_scale
    a, sa = fo.quantize_blocks(_randn(3, k, 21))
    for rows in (1, 3):
        y = fo.block_scaled_mm(a[:rows], sa[:rows], b.view(torch.float8_e4m3fn), sb, None, FP32)
        assert (y[:, :-130] == 0).all()
        want, slack = ref.mm(a[:rows], sa[:rows], tail, tail_scale)
        ref.check_close(y[:, -130:], want, slack)
    big, big_scale = b.view(torch.float8_e4m3fn), torch.ones((n, k // 128), device="cuda")
    big_scale[-130:] = tail_scale.repeat_interleave(128, 0)[:130]
    y = fo.block_scaled_mm(big, big_scale, a, sa, None, FP32)   # as the first operand, with scales by row on both
    want, slack = ref.mm(tail, big_scale[-130:], a, sa)
    assert (y[:-130] == 0).all()
    ref.check_close(y[-130:], want, slack)


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (100, 384, 8192), (512, 512, 512)])
def test_other_streams_and_graphs(fo, m, n, k):
    """On a stream of its own, and captured: replays with new inputs and eager calls between them."""
    operands = _operands(fo, m, n, k, seed=30)
    want = fo.block_scaled_mm(*operands)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fo.block_scaled_mm(*operands)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = fo.block_scaled_mm(*operands)
    for replay in range(4):
        fresh = _operands(fo, m, n, k, seed=40 + replay)
        for mine, new in zip(operands, fresh):
            mine.copy_(new)
        eager = fo.block_scaled_mm(*fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager)


def test_refusals(fo):
    a, sa, b, sb = _operands(fo, 20, 140, 256)
    mm = fo.block_scaled_mm
    for bad, message in [((a.float(), sa, b, sb), "float8"), ((a, sa.double(), b, sb), "float32"),
                         ((a, sa[:, :1], b, sb), "a_scale must be"), ((a[:7], sa, b, sb), "a_scale must be"),
                         ((a, sa, b, sb[:1]), "b_scale must be"), ((a, sa, b[:, :128], sb[:, :1]), "same number of columns"),
                         ((a, sa, b, sb, torch.zeros(140, device="cuda")), "bias must have"),
                         ((a, sa, b, sb, torch.zeros(139, device="cuda", dtype=BF16)), "bias must be"),
                         ((a, sa.cpu(), b, sb), "CUDA tensors")]:
        with pytest.raises(RuntimeError, match=message):
            mm(*bad)
    with pytest.raises(ValueError, match="output dtype"):
        mm(a, sa, b, sb, None, torch.float64)
    with pytest.raises(ValueError, match="matrix"):
        mm(a[None], sa, b, sb)
    with pytest.raises(NotImplementedError):
        mm(a.cpu(), sa.cpu(), b.cpu(), sb.cpu())
    with pytest.raises(ValueError, match="x must be"):
        fo.block_scaled_linear(torch.zeros((2, 3), device="cuda"), torch.zeros((4, 5), device="cuda"))
    with pytest.raises(ValueError, match="output dtype"):
        fo.block_scaled_linear(torch.zeros((2, 3), device="cuda").double(), torch.zeros((4, 3), device="cuda"))


# ---- the layer ----


def _whole(m, n, seed):
    """Integers of at most 14 with a 14 in every block of 128 of rows, columns and squares: exact in e4m3 after scaling (a
    scale of 2^-5, codes of 4 significant bits), so products and sums are whole numbers."""
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randint(-14, 15, (m, n), generator=g, device="cuda").float()
    x[::128], x[:, ::128] = 14, 14
    return x


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (3, 130, 40), (130, 140, 260), (257, 384, 128)])
def test_layer_is_exact_on_whole_numbers(fo, m, n, k, bias):
    """Outputs and gradients equal the formulas', and the gradients the differences of outputs: with whole numbers nothing
    is rounded (sums stay under 2^24)."""
    x, w, gy = _whole(m, k, 1).requires_grad_(), _whole(n, k, 2).requires_grad_(), _whole(m, n, 3)
    b = _whole(1, n, 4)[0].requires_grad_() if bias else None
    y = fo.block_scaled_linear(x, w, b)
    want = x.detach().double() @ w.detach().double().t() + (b.detach().double() if bias else 0)
    assert torch.equal(y.double(), want)
    grads = torch.autograd.grad(y, (x, w) + ((b,) if bias else ()), gy)
    assert torch.equal(grads[0].double(), gy.double() @ w.detach().double())
    assert torch.equal(grads[1].double(), gy.double().t() @ x.detach().double())
    if bias:
        assert torch.equal(grads[2].double(), gy.double().sum(0))

    def total(x, w, b):
        with torch.no_grad():
            return (fo.block_scaled_linear(x, w, b).double() * gy.double()).sum()

    # off the rows and columns of 14s, which keep the scales
    i, j, c = (m - 1) if m > 1 else 0, k - 1, n - 1
    for which, (at, grad) in enumerate([((i, j), grads[0]), ((c, j), grads[1])]):
        if at[0] % 128 == 0:
            continue
        moved = []
        for d in (1, -1):
            args = [x.detach().clone(), w.detach().clone()]
            args[which][at] = 3 + d
            moved.append(total(*args, b))
        assert (moved[0] - moved[1]) / 2 == grad[at].double()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("q", sorted(ref.FP8))
def test_layer_against_the_formulas(fo, dtype, q):
    """Outputs and gradients are the 64-bit products of the quantized operands."""
    m, n, k = 150, 200, 300
    x, w = _randn(m, k, 51).to(dtype).requires_grad_(), _randn(n, k, 52).to(dtype).requires_grad_()
    b, gy = _randn(1, n, 53)[0].to(dtype).requires_grad_(), (_randn(m, n, 54) * 1e-2).to(dtype)
    y = fo.block_scaled_linear(x[None], w, b, ref.FP8[q])
    assert y.shape == (1, m, n) and y.dtype == dtype
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy[None])
    quant = lambda t, **kw: fo.quantize_blocks(t.detach(), ref.FP8[q], **kw)  # noqa: E731
    wq = quant(w, square=True)
    ref.check_close(y[0].detach(), *ref.mm(*quant(x), *wq, b.detach()))
    wt = (wq[0].t(), wq[1].t())
    ref.check_close(gx, *ref.mm(*quant(gy), *wt))
    ref.check_close(gw, *ref.mm(*quant(gy.t().contiguous()), *quant(x.t().contiguous())))
    ref.check_close(gb, gy.double().sum(0), (m + 8) * 2.0**-23 * gy.double().abs().sum(0))
    assert gx.dtype == gw.dtype == gb.dtype == dtype


def test_layer_gradients_one_at_a_time(fo):
    """Each gradient by itself has the bits it has with the others; the frozen layer's input gradient too."""
    m, n, k = 70, 130, 190
    x, w, b = (_randn(m, k, 61).to(BF16), _randn(n, k, 62).to(BF16), _randn(1, n, 63)[0].to(BF16))
    gy = _randn(m, n, 64).to(BF16)
    all_three = [t.clone().requires_grad_() for t in (x, w, b)]
    y = fo.block_scaled_linear(*all_three)
    want = torch.autograd.grad(y, all_three, gy)
    for which in range(3):
        args = [t.clone() for t in (x, w, b)]
        args[which].requires_grad_()
        got = fo.block_scaled_linear(*args)
        assert torch.equal(got, y)
        assert torch.equal(torch.autograd.grad(got, args[which], gy)[0], want[which])
    layer = torch.nn.Linear(k, n, device="cuda", dtype=BF16)
    with torch.no_grad():
        layer.weight.copy_(w)
        layer.bias.copy_(b)
    layer.requires_grad_(False)
    assert fo.to_block_scaled_linear(layer) == 1 and fo.to_block_scaled_linear(layer) == 0
    assert layer.weight_fp8.dtype == torch.float8_e4m3fn and set(layer.state_dict()) == {"weight", "bias"}
    assert torch.equal(layer(x), y)
    xg = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(layer(xg), xg, gy)[0], want[0])


def test_trained_layer_is_quantized_on_every_pass(fo):
    layer = torch.nn.Linear(256, 128, device="cuda", dtype=BF16)
    fo.to_block_scaled_linear(layer)
    x = _randn(9, 256, 70).to(BF16)
    assert not hasattr(layer, "weight_fp8")
    layer(x).sum().backward()
    assert layer.weight.grad.shape == (128, 256) and layer.bias.grad.shape == (128,)
    before = layer(x).detach()
    with torch.no_grad():
        layer.weight.mul_(2)
        layer.bias.zero_()
        assert not torch.equal(layer(x), before)
        assert torch.equal(layer(x), fo.block_scaled_linear(x, layer.weight))


def test_empty_layer(fo):
    x = torch.zeros((0, 64), device="cuda", requires_grad=True)
    w = _randn(32, 64, 80).requires_grad_()
    y = fo.block_scaled_linear(x, w)
    assert y.shape == (0, 32)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == (0, 64) and (gw == 0).all()
