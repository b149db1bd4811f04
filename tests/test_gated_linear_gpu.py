"""The gated block in 16 bits and its gradients against 64 bits."""

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu
# (rows, K, F): single values; few rows and each kernel for them; lengths of no whole tile, piece or stage; K of no multiple of 8;
# products whose K is split; every tile.
SHAPES = [(1, 1, 1), (1, 8, 3), (2, 7, 5), (1, 4096, 40), (5, 72, 33), (16, 520, 129), (17, 136, 64), (33, 200, 257), (64, 1032, 96),
          (65, 64, 64), (100, 333, 50), (130, 520, 1001), (257, 2576, 129), (300, 128, 2048), (700, 72, 700), (1000, 264, 1400)]


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _data(m, k, f, dtype, bias, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    return ((randn(m, k) * 2).to(dtype), (randn(2 * f, k) * k**-0.5).to(dtype), randn(2 * f).to(dtype) if bias else None,
            (randn(m, f) * 0.1).to(dtype))


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m,k,f", SHAPES)
def test_forward(fo, m, k, f, dtype, act):
    x, w, b, _ = _data(m, k, f, dtype, bias=m % 2 == 0)
    y = fo.gated_linear(x, w, b, act)
    assert y.dtype == dtype and y.shape == (m, f)
    ref.check(y, *ref.gated(x, w, b, act))


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m,k,f", SHAPES)
def test_gradients(fo, m, k, f, dtype, act):
    x, w, b, gy = _data(m, k, f, dtype, bias=f % 2 == 1, seed=1)
    wanted = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = fo.gated_linear(x, w, b, act)
    plain = fo.gated_linear(x.detach(), w.detach(), None if b is None else b.detach(), act)
    assert torch.equal(y, plain)   # what is kept for the backward changes nothing
    grads = torch.autograd.grad(y, wanted, gy)
    detached = [None if t is None else t.detach() for t in (x, w, b)]
    for got, t, (want, bound) in zip(grads, wanted, ref.gated_gradients(*detached, act, gy)):
        assert got.dtype == t.dtype
        ref.check(got, want, bound)


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
def test_gradients_are_the_differences_of_the_definition(act):
    """The slopes of the reference itself, by central differences in 64 bits."""
    g = torch.linspace(-9, 9, 4001, dtype=torch.float64)
    step = 1e-5
    slope = (ref.activation(g + step, act)[0] - ref.activation(g - step, act)[0]) / (2 * step)
    assert (slope - ref.activation(g, act)[1]).abs().max() < 1e-9


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("m", [3, 90])
def test_layouts(fo, m, act):
    """Batches, rows apart, off 16-byte boundaries, columns first, and one row for all."""
    x, w, b, gy = _data(m, 72, 40, torch.bfloat16, True)
    want = fo.gated_linear(x, w, b, act)
    assert torch.equal(fo.gated_linear(x.view(1, m, 1, 72), w, b, act).view(m, 40), want)
    apart = torch.full((m, 200), float("nan"), dtype=x.dtype, device="cuda")
    for at in (0, 8, 3):
        apart[:, at:at + 72] = x
        assert torch.equal(fo.gated_linear(apart[:, at:at + 72], w, b, act), want)
        apart.fill_(float("nan"))
    assert torch.equal(fo.gated_linear(x.t().contiguous().t(), w.t().contiguous().t(), b, act), want)
    assert torch.equal(fo.gated_linear(x[:1].expand(m, 72), w, b, act), fo.gated_linear(x[:1].repeat(m, 1), w, b, act))
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    expected = torch.autograd.grad(fo.gated_linear(xs, ws, b, act), (xs, ws), gy)
    got = torch.autograd.grad(fo.gated_linear(xs, ws, b, act), (xs, ws), gy.t().contiguous().t())
    assert all(torch.equal(p, q) for p, q in zip(got, expected))
    one = torch.autograd.grad(fo.gated_linear(xs, ws, b, act).sum(), (xs, ws))   # an expanded gradient
    ones = torch.autograd.grad(fo.gated_linear(xs, ws, b, act), (xs, ws), torch.ones_like(gy))
    assert all(torch.equal(p, q) for p, q in zip(one, ones))


@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True), (True, True, False)])
def test_single_gradients(fo, needs):
    x, w, b, gy = _data(40, 64, 24, torch.float16, True)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    expected = torch.autograd.grad(fo.gated_linear(*full), full, gy)
    some = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), needs)]
    fo.gated_linear(*some).backward(gy)
    for t, n, want in zip(some, needs, expected):
        assert (torch.equal(t.grad, want) if n else t.grad is None)


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m", [2, 70])
def test_extreme_gates(fo, m, dtype, act):
    """Gates of the type's lowest and largest values, infinities and NaN; a masked row's gradients are zero, not NaN."""
    low, large = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.zeros(m, 8, dtype=dtype, device="cuda")
    x[:, 0] = 1
    w = torch.zeros(2 * 6, 8, dtype=dtype, device="cuda")
    w[:6, 0] = torch.tensor([low, large, float("-inf"), float("nan"), 0.0, -200.0])
    w[6:, 0] = torch.tensor([large, 0.5, 2.0, 1.0, float("inf"), 1.0])
    x[:, 1:] = 0
    w[:, 1:] = 0
    xs = x.clone().requires_grad_()
    y = fo.gated_linear(xs, w, None, act)
    got = y[0].float().cpu()
    assert got[0] == 0 and got[1] == torch.tensor(large, dtype=torch.float64).mul(0.5).to(dtype).float()
    assert got[2] == 0 and got[3].isnan() and got[4].isnan() and got[5].abs() < 1e-6
    assert all(torch.equal(row, y[0]) or (row.isnan() == y[0].isnan()).all() for row in y)
    masked = torch.zeros_like(w)
    masked[0, 0], masked[6, 0] = low, large
    ms = masked.clone().requires_grad_()
    for g in torch.autograd.grad(fo.gated_linear(xs, ms, None, act), (xs, ms), torch.ones_like(y)):
        assert (g == 0).all()


def test_empty(fo):
    for m, k, f in ((0, 16, 8), (3, 0, 8), (3, 16, 0)):
        x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.randn(2 * f, k, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = fo.gated_linear(x, w)
        assert y.shape == (m, f) and (y == 0).all()
        y.sum().backward()
        assert (x.grad == 0).all() and (w.grad == 0).all()


def test_refusals(fo):
    x, w, b, _ = _data(4, 16, 8, torch.bfloat16, True)
    for bad in (dict(x=x.float()), dict(weight=w.half()), dict(weight=w[:3]), dict(weight=w[:, :8]), dict(bias=b[:3]),
                dict(activation="relu"), dict(x=x[0, 0])):
        with pytest.raises((ValueError, RuntimeError)):
            fo.gated_linear(**(dict(x=x, weight=w, bias=b, activation="silu") | bad))
    with pytest.raises((RuntimeError, NotImplementedError)):
        fo.gated_linear(x.cpu(), w.cpu())
    xs = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(fo.gated_linear(xs, w).sum(), xs, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        fo.gated_linear(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), w)


def test_deterministic(fo):
    x, w, _, gy = _data(200, 1024, 100, torch.bfloat16, False)
    xs, ws = x.requires_grad_(), w.requires_grad_()
    first = None
    for _ in range(4):
        y = fo.gated_linear(xs, ws)
        got = [y, *torch.autograd.grad(y, (xs, ws), gy)]
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(got, first))


@pytest.mark.parametrize("m", [1, 40, 200])
def test_memory_past_the_operands_is_not_read(fo, m):
    """Operands and outputs at the end of what was allocated, beside values that would show."""
    k, f = 264, 70
    x, w, b, gy = _data(m, k, f, torch.bfloat16, True)
    want = fo.gated_linear(x, w, b)

    def framed(t):
        whole = torch.full((t.numel() + 512,), float("nan"), dtype=t.dtype, device="cuda")
        whole[256:256 + t.numel()] = t.reshape(-1)
        return whole[256:256 + t.numel()].view(t.shape)

    assert torch.equal(fo.gated_linear(framed(x), framed(w), framed(b)), want)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    expected = torch.autograd.grad(fo.gated_linear(*leaves), leaves, gy)
    framed_leaves = [framed(t).requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(fo.gated_linear(*framed_leaves), framed_leaves, framed(gy))
    assert all(torch.equal(p, q) for p, q in zip(got, expected))


@pytest.mark.parametrize("m", [2, 96])
def test_another_stream_and_graphs(fo, m):
    """A captured step follows its operands, with the program's own work between the replays; two graphs do not disturb each other."""
    x, w, b, gy = _data(m, 1024, 40, torch.bfloat16, True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        elsewhere = fo.gated_linear(x, w, b)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(elsewhere, fo.gated_linear(x, w, b))

    def step(xs, ws, bs):
        y = fo.gated_linear(xs, ws, bs)
        return [y, *torch.autograd.grad(y, (xs, ws, bs), gy)]

    graphs = []
    for _ in range(2):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        with torch.cuda.stream(stream):
            step(*leaves)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(*leaves)
        graphs.append((graph, leaves, out))
    for turn in range(3):
        for graph, leaves, out in graphs:
            with torch.no_grad():
                leaves[0].copy_(x * (turn + 1))
                leaves[1].copy_(w * 0.5 ** turn)
            graph.replay()
            torch.cuda.synchronize()
            want = step(*[t.detach().clone().requires_grad_() for t in leaves])
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_compiled(fo):
    x, w, b, gy = _data(24, 40, 16, torch.bfloat16, True)

    def step(xs, ws, bs):
        return fo.gated_linear(xs * 2, ws, bs, "gelu")

    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = step(*leaves)
    expected = torch.autograd.grad(want, leaves, gy)
    y = torch.compile(step, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(y, want)
    for got, grad in zip(torch.autograd.grad(y, leaves, gy), expected):
        assert torch.equal(got, grad)
