"""Products with 4-bit weights and group scales, their quantization and the layer, against 64 bits."""

import copy

import pytest
import torch
from torch import nn

import linear_ref as ref

pytestmark = pytest.mark.gpu
# (rows, K, N): single values, K of no whole group, byte or piece, columns of no multiple of 4, each kernel for few rows, split K,
# and more rows.
SHAPES = [(1, 1, 1), (1, 4096, 64), (1, 130, 5), (2, 33, 3), (3, 384, 20), (7, 1000, 77), (16, 4096, 33), (17, 520, 48), (24, 200, 130),
          (40, 264, 63), (64, 640, 100), (65, 136, 40), (200, 1031, 70), (300, 640, 520)]
GROUPS = [(32, False), (64, True), (128, False), (128, True)]


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


def _weight(n, k, group, zeros, dtype, seed=0):
    """Codes of every value, as a checkpoint may hold them."""
    g = torch.Generator("cuda").manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
    scale = (torch.rand((groups, n), generator=g, device="cuda") * 0.1 + 0.01).to(dtype).t()
    zero = torch.randint(0, 16, (groups, n), generator=g, device="cuda", dtype=torch.uint8).t() if zeros else None
    return codes, scale, zero


def _rows(m, k, dtype, seed=1):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn((m, k), generator=g, device="cuda") + 0.3).to(dtype)


def _bound(x, weight, bias, rounded):
    want, bound = ref.int4(x, *weight, bias)
    if rounded:   # the weight is rounded to x's dtype first
        w = ref.int4_values(*weight, x.shape[1])
        bound = bound + x.double().abs() @ ref.half_step(x.dtype, w).t()
    return want, bound


@pytest.mark.parametrize("group,zeros", GROUPS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(fo, m, k, n, dtype, group, zeros):
    weight, x = _weight(n, k, group, zeros, dtype), _rows(m, k, dtype)
    bias = _rows(1, n, dtype, 2)[0] if m % 2 else None
    y = fo.int4_linear(x, *weight, bias)
    assert y.dtype == dtype and y.shape == (m, n)
    ref.check(y, *_bound(x, weight, bias, m > 64))


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("group,zeros", GROUPS)
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m,k,f", [(1, 8, 1), (1, 130, 5), (1, 4096, 50), (4, 33, 3), (9, 264, 70), (24, 520, 17), (50, 640, 33), (90, 200, 66)])
def test_gated_is_the_block_of_the_two_halves(fo, m, k, f, dtype, group, zeros, act):
    weight, x = _weight(2 * f, k, group, zeros, dtype), _rows(m, k, dtype)
    bias = _rows(1, 2 * f, dtype, 2)[0] if m % 2 else None
    y = fo.int4_gated_linear(x, *weight, bias, act)
    h, bound = _bound(x, weight, bias, m > 64)
    gate, up = h.chunk(2, 1)
    d_gate, d_up = bound.chunk(2, 1)
    value, slope = ref.activation(gate, act)
    off = (slope.abs() + 2 * d_gate) * d_gate * up.abs() + value.abs() * d_up + d_gate * d_up
    ref.check(y, value * up, off + ref.ACT * (value * up).abs())


@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 8), (5, 130, 21), (40, 264, 64), (70, 1031, 100)])
def test_gradients(fo, m, k, n, dtype):
    weight, x = _weight(n, k, 64, True, dtype), _rows(m, k, dtype).requires_grad_()
    bias = torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
    gy = _rows(m, n, dtype, 3)
    y = fo.int4_linear(x, *weight, bias)
    gx, gb = torch.autograd.grad(y, (x, bias), gy)
    w = ref.int4_values(*weight, k)
    size = gy.double().abs() @ w.abs()
    ref.check(gx, gy.double() @ w, gy.double().abs() @ ref.half_step(dtype, w) + ref.sum_error(n, size))
    ref.check(gb, gy.double().sum(0), (m + 34) * ref.ULP * gy.double().abs().sum(0))
    (alone,) = torch.autograd.grad(fo.int4_linear(x, *weight), x, gy)
    assert torch.equal(alone, gx)
    (of_bias,) = torch.autograd.grad(fo.int4_linear(x.detach(), *weight, bias), bias, gy)
    assert torch.equal(of_bias, gb)


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
def test_gated_with_gradients_is_its_parts(fo, act):
    weight, x = _weight(48, 64, 32, True, torch.bfloat16), _rows(5, 64, torch.bfloat16).requires_grad_()
    y = fo.int4_gated_linear(x, *weight, None, act)
    h = fo.int4_linear(x, *weight)
    gate, up = h.double().chunk(2, 1)
    value = ref.activation(gate, act)[0]
    assert ((y.double() - value * up).abs() <= 2 * ref.half_step(torch.bfloat16, (value * up).abs()) +
            ref.half_step(torch.bfloat16, value.abs()) * up.abs() + ref.ACT).all()
    y.sum().backward()
    assert x.grad.isfinite().all() and x.grad.abs().sum() > 0


@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("group,zeros", GROUPS)
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (5, 128), (64, 1000), (129, 4097)])
def test_quantize(fo, n, k, group, zeros, dtype):
    w = _rows(n, k, dtype, 5) * torch.linspace(0.01, 3, n, device="cuda")[:, None].to(dtype)
    w[0] = 0
    codes, scale, zero = fo.quantize_int4(w, group, zeros=zeros)
    groups = -(-k // group)
    assert codes.shape == (n, -(-k // 2)) and scale.shape == (n, groups) and scale.dtype == dtype
    assert (zero is None) if not zeros else (zero.shape == scale.shape and zero.dtype == torch.uint8 and zero.max() <= 15)
    blocks = torch.zeros(n, groups * group, dtype=torch.float32, device="cuda")
    blocks[:, :k] = w.float()
    blocks = blocks.view(n, groups, group)
    # the definition's own operations, in fp32
    if zeros:
        low, high = blocks.amin(2).clamp(max=0), blocks.amax(2).clamp(min=0)
        s = ((high - low) / 15).to(dtype)
        z = torch.where(s > 0, (-low / s.float()).round().clamp(0, 15), 8.0)
    else:
        s = (blocks.abs().amax(2) / 7).to(dtype)
        z = torch.full_like(s, 8).float()
    assert torch.equal(scale, s)
    if zeros:
        assert torch.equal(zero.float(), z)
    q = torch.where(s[:, :, None] > 0, ((blocks / s.float()[:, :, None]).round() + z[:, :, None]).clamp(0, 15), z[:, :, None])
    q = q.view(n, -1)[:, :k]
    got = torch.stack((codes & 15, codes >> 4), 2).flatten(1)[:, :k]
    assert torch.equal(got.float(), q)
    values = fo.dequantize_int4(codes, scale, zero, k)
    assert values.dtype == dtype and torch.equal(values, ref.int4_values(codes, scale, zero, k).to(dtype))
    # symmetric: every value within half a step and the scale's rounding; with zero points within a step, which rounding them costs
    step = scale.double().repeat_interleave(group, 1)[:, :k]
    eps = torch.finfo(dtype).eps
    assert ((ref.int4_values(codes, scale, zero, k) - w.double()).abs() <= step * (1.0 if zeros else 0.5) * (1 + 16 * eps) + 8 * eps * step).all()


def test_quantize_values_that_are_not_numbers(fo):
    w = _rows(4, 256, torch.bfloat16)
    w[1, 3], w[2, 200] = float("nan"), float("inf")
    for zeros in (False, True):
        weight = fo.quantize_int4(w, 128, zeros=zeros)
        v = fo.dequantize_int4(*weight)
        assert v[1, :128].isnan().all() and v[1, 128:].isfinite().all()
        assert v[2, 128:].isnan().all() and v[2, :128].isfinite().all() and v[[0, 3]].isfinite().all()
        y = fo.int4_linear(_rows(2, 256, torch.bfloat16), *weight)
        assert y[:, [1, 2]].isnan().all() and y[:, [0, 3]].isfinite().all()


@pytest.mark.parametrize("m", [2, 80])
def test_layouts(fo, m):
    """Codes, scales and rows of x wherever they lie give the same bits."""
    weight, x = _weight(37, 200, 32, True, torch.float16), _rows(m, 200, torch.float16)
    codes, scale, zero = weight
    want = fo.int4_linear(x, *weight)
    assert torch.equal(fo.int4_linear(x.view(m, 1, 200), *weight).view(m, 37), want)
    assert torch.equal(fo.int4_linear(x, codes, scale.contiguous(), zero.contiguous()), want)
    wide = torch.zeros(37, 131, dtype=torch.uint8, device="cuda")
    for at in (0, 4, 1):
        wide[:, at:at + 100] = codes
        assert torch.equal(fo.int4_linear(x, wide[:, at:at + 100], scale, zero), want)
    apart = torch.zeros(m, 333, dtype=x.dtype, device="cuda")
    apart[:, 5:205] = x
    assert torch.equal(fo.int4_linear(apart[:, 5:205], *weight), want)
    padded = torch.full((7, 50), float("nan"), dtype=scale.dtype, device="cuda")
    padded[:, 3:40] = scale.t()
    assert torch.equal(fo.int4_linear(x, codes, padded[:, 3:40].t(), zero), want)
    # scales in the other type are rounded to x's
    assert torch.equal(fo.int4_linear(x, codes, scale.float(), zero), want)


def test_memory_past_the_operands_is_not_read(fo):
    """Codes and scales that end with their memory, beside values that would show."""
    for n, k in ((21, 130), (3, 70), (16, 256)):
        codes, scale, zero = _weight(n, k, 64, True, torch.bfloat16)
        x = _rows(3, k, torch.bfloat16)
        want = fo.int4_linear(x, codes, scale, zero)
        tail = torch.full((scale.numel() + 64,), float("nan"), dtype=scale.dtype, device="cuda")
        tail[: scale.numel()] = scale.t().reshape(-1)
        framed = tail[: scale.numel()].view(-1, n).t()
        assert torch.equal(fo.int4_linear(x, codes, framed, zero), want)
        rows = torch.full((x.numel() + 64,), float("nan"), dtype=x.dtype, device="cuda")
        rows[: x.numel()] = x.reshape(-1)
        assert torch.equal(fo.int4_linear(rows[: x.numel()].view(3, k), codes, scale, zero), want)


def test_empty(fo):
    weight = _weight(8, 64, 32, True, torch.bfloat16)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    assert fo.int4_linear(x, *weight).shape == (0, 8)
    fo.int4_linear(x, *weight).sum().backward()
    assert x.grad.shape == (0, 64)
    assert fo.int4_gated_linear(x.detach(), *weight).shape == (0, 4)
    none = fo.quantize_int4(torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda"), 64)
    assert fo.int4_linear(torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda"), *none).shape == (2, 0)


def test_refusals(fo):
    codes, scale, zero = _weight(8, 64, 32, True, torch.bfloat16)
    x = _rows(2, 64, torch.bfloat16)
    good = dict(x=x, codes=codes, scale=scale, zero=zero)
    for bad in (dict(x=x.float()), dict(x=x[:, :32]), dict(codes=codes.int()), dict(codes=codes[:4]), dict(scale=scale[:, :1].repeat(1, 5)),
                dict(zero=zero.float()), dict(zero=zero[:, :1]), dict(bias=x[0, :3]), dict(scale=scale.int()),
                dict(scale=scale.clone().requires_grad_())):
        with pytest.raises(ValueError):
            fo.int4_linear(**(good | bad))
    with pytest.raises(ValueError):
        fo.int4_gated_linear(x, codes[:7], scale[:7], zero[:7])
    with pytest.raises(ValueError):
        fo.quantize_int4(torch.zeros(4, 4, device="cuda"))
    with pytest.raises(ValueError):
        fo.quantize_int4(x, 48)
    with pytest.raises((RuntimeError, NotImplementedError)):
        fo.int4_linear(x.cpu(), codes.cpu(), scale.cpu())
    xs = x.clone().requires_grad_()
    gy = torch.ones(2, 8, dtype=x.dtype, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(fo.int4_linear(xs, codes, scale, zero), xs, gy, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()


@pytest.mark.parametrize("m", [1, 30, 100])
def test_graphs(fo, m):
    """A captured forward and backward, replayed between other work."""
    weight = _weight(40, 2048, 128, False, torch.bfloat16)
    x, gy = _rows(m, 2048, torch.bfloat16), _rows(m, 40, torch.bfloat16, 4)
    leaf = x.clone().requires_grad_()

    def step(t):
        y = fo.int4_linear(t, *weight)
        return [y, *torch.autograd.grad(y, (t,), gy), fo.int4_gated_linear(t.detach(), *weight)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(leaf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(leaf)
    for turn in range(3):
        with torch.no_grad():
            leaf.copy_(x * (turn + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = step(leaf.detach().clone().requires_grad_())
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_layer(fo):
    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(72, 40), nn.GELU(), nn.Linear(40, 9, bias=False)).cuda().bfloat16()
    keys = list(model.state_dict())
    original = copy.deepcopy(model)
    assert fo.to_int4_linear(model, 32, zeros=True) == 2 and isinstance(model[0], fo.Int4Linear)
    assert list(model.state_dict()) == keys
    x = _rows(6, 72, torch.bfloat16)
    for layer, plain in ((model[0], original[0]),):
        codes, scale, zero = fo.quantize_int4(plain.weight, 32, zeros=True)
        assert torch.equal(layer(x), fo.int4_linear(x, codes, scale, zero, plain.bias))
    xs = x.clone().requires_grad_()
    model(xs).sum().backward()
    assert xs.grad.isfinite().all() and model[0].bias.grad is not None and model[0].weight.grad is None
    with torch.no_grad():
        assert torch.equal(torch.compile(model, backend="aot_eager", fullgraph=True)(x), model(x))
    assert fo.to_int4_linear(nn.Sequential(nn.Linear(8, 8))) == 0   # fp32 weights stay as they are


def test_compiled_gradients(fo):
    weight, x = _weight(24, 70, 32, True, torch.bfloat16), _rows(5, 70, torch.bfloat16)
    bias = _rows(1, 24, torch.bfloat16)[0]

    def step(t, b):
        return fo.int4_linear(t * 2, *weight, b)

    leaves = [x.clone().requires_grad_(), bias.clone().requires_grad_()]
    want = step(*leaves)
    expected = torch.autograd.grad(want.float().square().sum(), leaves)
    y = torch.compile(step, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(y, want)
    got = torch.autograd.grad(y.float().square().sum(), leaves)
    assert torch.equal(got[0], expected[0])
    assert (got[1].double() - expected[1].double()).abs().max() <= ref.half_step(torch.bfloat16, expected[1].double()).max() * 4
