"""The feed-forward operators as they are used together: the example's layer, trained in 16 bits and with 4-bit weights; long
batches; and tensors past 4 GiB."""

import importlib.util
import pathlib
import subprocess
import sys

import pytest
import torch
from torch import nn

import linear_ref as ref

pytestmark = pytest.mark.gpu
PATH = pathlib.Path(__file__).resolve().parents[1] / "feather-ops_amd" / "examples" / "gated_mlp.py"


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


@pytest.fixture(scope="module")
def example(fo):
    spec = importlib.util.spec_from_file_location("gated_mlp", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _reference(norm, wide, narrow, act, eps, x, residual):
    """The layer in 64 bits from the given weights."""
    h = (x + residual).double()
    y = h * (h.square().mean(-1, keepdim=True) + eps).rsqrt() * norm
    gate, up = (y @ wide.t()).chunk(2, -1)
    return (ref.activation(gate, act)[0] * up) @ narrow.t()


# Each of the layer's three 16-bit intermediates (the norm's output, the block's, and the layer's) is rounded to 8 bits, off by 2^-8 at
# most and 2^-9.8 in the mean square; the gated product doubles the norm's. In gradients as many again, of the two sums' gradients
# and of each product's result: together, as squares, under 5 such steps of 2^-8 in norm.
OFF = 5 * 2.0**-8


@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_training(example, tokens, act):
    torch.manual_seed(tokens)
    mlp = example.GatedMLP(640, 1000, act)
    x, residual = (torch.randn(tokens, 640, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    y, h = mlp(x, residual)
    gy = torch.randn_like(y)
    inputs = (x, mlp.norm, mlp.gate_up.weight, mlp.down.weight)
    got = torch.autograd.grad(y, inputs, gy)
    leaves = [t.detach().double().requires_grad_() for t in inputs]
    stream = (leaves[0] + residual.detach().double())
    rounded = stream + ((x + residual).detach().double() - stream).detach()   # the residual stream is rounded before the norm
    h64 = rounded
    n = h64 * (h64.square().mean(-1, keepdim=True) + mlp.eps).rsqrt() * leaves[1]
    gate, up = (n @ leaves[2].t()).chunk(2, -1)
    if act == "silu":
        value = nn.functional.silu(gate)
    else:
        value = nn.functional.gelu(gate, approximate="tanh" if act == "gelu_tanh" else "none")
    want_y = (value * up) @ leaves[3].t()
    want = torch.autograd.grad(want_y, leaves, gy.double())
    for a, b in [(y, want_y), *zip(got, want)]:
        assert ((a.double() - b).norm() / b.norm()).item() < OFF
    assert torch.equal(h, x + residual)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("tokens", [1, 24, 200])
def test_decoding_and_an_adapter(fo, example, tokens, zeros):
    torch.manual_seed(tokens)
    mlp = example.GatedMLP(640, 1000)
    x, residual = (torch.randn(tokens, 640, device="cuda").bfloat16() for _ in range(2))
    keys = list(mlp.state_dict())
    mlp.quantize_(64, zeros)
    assert list(mlp.state_dict()) == keys
    wide, narrow = (ref.int4_values(layer.weight_int4, layer.weight_scale, layer.weight_zero, k)
                    for layer, k in ((mlp.gate_up, 640), (mlp.down, 1000)))
    want = _reference(mlp.norm.detach().double(), wide, narrow, "silu", mlp.eps, x, residual)
    with torch.no_grad():
        y, h = mlp(x, residual)
    assert ((y.double() - want).norm() / want.norm()).item() < OFF and torch.equal(h, x + residual)
    # an adapter before the frozen layer: its gradients, and those of the norm, against differences of the layer itself in 64 bits
    a = (torch.randn(640, 640, device="cuda") * 0.02).bfloat16().requires_grad_()
    gy = torch.randn_like(y)
    got = torch.autograd.grad(mlp(x @ a, residual)[0], (a, mlp.norm), gy)
    direction = torch.randn_like(a).double()
    norm64, a64 = mlp.norm.detach().double(), a.detach().double()

    def loss(step):
        h = (x.double() @ (a64 + step * direction) + residual.double())
        n = h * (h.square().mean(-1, keepdim=True) + mlp.eps).rsqrt() * norm64
        gate, up = (n @ wide.t()).chunk(2, -1)
        return ((ref.activation(gate, "silu")[0] * up) @ narrow.t() * gy.double()).sum()

    slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
    mine = (got[0].double() * direction).sum()
    # a random direction sees the error of the gradient's norm, by its own size and a few times over by chance
    assert (mine - slope).abs() <= 4 * OFF * got[0].double().norm() and got[1].isfinite().all()


def test_steps_in_a_graph(fo, example):
    """Two layers of 4-bit weights, captured, replayed between eager work of the same layers."""
    torch.manual_seed(3)
    layers = [example.GatedMLP(512, 704).quantize_(128, False) for _ in range(2)]
    x, residual = (torch.randn(5, 512, device="cuda").bfloat16() for _ in range(2))

    def step():
        y, h = layers[0](x, residual)
        return layers[1](y, h)

    with torch.no_grad():
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for turn in range(3):
            x.copy_(torch.randn_like(x))
            want = [t.clone() for t in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.parametrize("k", [2048, 2045])
@pytest.mark.parametrize("kind", ["gated", "int4"])
def test_forward_and_backward_in_two_graphs(fo, kind, k):
    """They share their memory; products are split. Replays with new inputs, eager passes of the same leaves between them. While an
    eager graph of the leaves lives on another stream, a captured backward is refused."""
    m, f = 96, 64
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.randn((m, k), generator=g, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn((2 * f, k), generator=g, device="cuda") * k**-0.5).bfloat16().requires_grad_()
    codes = fo.quantize_int4(w.detach(), 32)
    leaves = (x, w) if kind == "gated" else (x,)

    def forward():
        return fo.gated_linear(x, w, None, "gelu") if kind == "gated" else fo.int4_linear(x, *codes)

    gy = torch.randn((m, f if kind == "gated" else 2 * f), generator=g, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(forward(), leaves, gy)
    torch.cuda.synchronize()
    alive = forward()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused, stream=side):
        y = forward()
        with pytest.raises(RuntimeError, match="lives on another stream"):
            torch.autograd.grad(y, leaves, gy)
    torch.autograd.grad(alive, leaves, gy)
    del alive, y
    pool, graphs = torch.cuda.graph_pool_handle(), [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0], pool=pool, stream=side):
        y = forward()
    with torch.cuda.graph(graphs[1], pool=pool, stream=side):
        grads = torch.autograd.grad(y, leaves, gy)
    for _ in range(4):
        with torch.no_grad():
            x.copy_(x * 0.5)
        eager = forward()
        want = (eager.detach(), *torch.autograd.grad(eager, leaves, gy))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip((y.detach(), *grads), want))


def test_vectors_batches_and_inference_mode(fo):
    x, w = torch.randn(2, 3, 72, device="cuda").half(), torch.randn(80, 72, device="cuda").half() * 0.1
    int4 = fo.quantize_int4(w, 32, zeros=True)
    for call in (lambda t: fo.gated_linear(t, w), lambda t: fo.int4_linear(t, *int4), lambda t: fo.int4_gated_linear(t, *int4)):
        rows = call(x.view(6, 72))
        assert torch.equal(call(x), rows.view(2, 3, -1)) and torch.equal(call(x[1, 2]), call(x[1, 2:])[0])
        with torch.inference_mode():
            assert torch.equal(call(x.clone()), rows.view(2, 3, -1))
        assert not call(x).requires_grad
    vector = x[0, 0].clone().requires_grad_()
    for call in (lambda t: fo.gated_linear(t, w), lambda t: fo.int4_linear(t, *int4)):
        (grad,) = torch.autograd.grad(call(vector).sum(), vector)
        (want,) = torch.autograd.grad(call(vector[None]).sum(), vector)
        assert torch.equal(grad, want)


def test_calls_on_two_streams_and_threads_at_once(fo):
    """Split products, whose workspaces are their stream's."""
    import threading

    x = [torch.randn(64, 4096, device="cuda").bfloat16() for _ in range(4)]
    w = torch.randn(128, 4096, device="cuda").bfloat16() * 0.02
    int4 = fo.quantize_int4(w)
    want = [(fo.gated_linear(t, w), fo.int4_linear(t, *int4)) for t in x]
    streams, got = [torch.cuda.Stream() for _ in x], [[] for _ in x]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i] = [fo.gated_linear(x[i], w), fo.int4_linear(x[i], *int4)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(x))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for mine, yours in zip(got, want) for p, q in zip(mine, yours))


def test_command():
    run = subprocess.run([sys.executable, str(PATH), "--tokens", "3", "--width", "256", "--hidden", "384"],
                         capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr[-2000:]
    assert "training:" in run.stdout and "inference:" in run.stdout


@pytest.mark.parametrize("m", [4, 80])
def test_last_token_of_a_long_batch(fo, m):
    """Rows further apart than the products reach."""
    k, f, tokens = 512, 72, 8192
    w, last = torch.randn(2 * f, k, device="cuda").half() * 0.05, torch.randn(m, k, device="cuda").half()
    batch = torch.zeros(m, tokens, k, device="cuda", dtype=torch.half)
    batch[:, -1] = last
    assert batch[:, -1].stride(0) > 1 << 21
    assert torch.equal(fo.gated_linear(batch[:, -1], w), fo.gated_linear(last, w))
    int4 = fo.quantize_int4(w)
    assert torch.equal(fo.int4_linear(batch[:, -1], *int4), fo.int4_linear(last, *int4))
    gy = torch.zeros(m, tokens, f, device="cuda", dtype=torch.half)
    gy[:, -1] = torch.randn(m, f, device="cuda").half()
    leaf = last.requires_grad_()
    got = [torch.autograd.grad(fo.gated_linear(leaf, w), leaf, g)[0] for g in (gy[:, -1], gy[:, -1].contiguous())]
    assert torch.equal(*got)


def test_gated_past_4_gib(fo):
    """Outputs of 5 GiB, and what is kept and the sums' gradients beyond."""
    m, k, f = 160000, 64, 16400
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn((m, k), generator=g, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn((2 * f, k), generator=g, device="cuda") * k**-0.5).bfloat16().requires_grad_()
    y = fo.gated_linear(x, w)
    assert y.numel() * 2 > 1 << 32
    gy = torch.randn((m, f), generator=g, device="cuda", dtype=torch.bfloat16)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    rows = torch.tensor([0, 1, m // 2 + 1, m - 40, m - 1], device="cuda")
    ref.check(y[rows], *ref.gated(x[rows].detach(), w.detach(), None, "silu"))
    want, bound = ref.gated_gradients(x[rows].detach(), w.detach(), None, "silu", gy[rows])[0]
    ref.check(gx[rows], want, bound)
    cols = torch.tensor([0, 7, f // 2, f - 1], device="cuda")
    some = torch.cat((w[cols], w[f + cols])).detach()
    want, bound = ref.gated_gradients(x.detach(), some, None, "silu", gy[:, cols])[1]
    ref.check(gw[torch.cat((cols, f + cols))], want, bound)


@pytest.mark.parametrize("m", [1, 24, 130])
def test_codes_past_4_gib(fo, m):
    n, k = 140000, 65536
    g = torch.Generator("cuda").manual_seed(0)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    assert codes.numel() > 1 << 32
    scale = (torch.rand((k // 128, n), generator=g, device="cuda") * 1e-3 + 1e-4).bfloat16().t()
    x = torch.randn((m, k), generator=g, device="cuda").bfloat16()
    y = fo.int4_linear(x, codes, scale)
    half = fo.int4_gated_linear(x, codes, scale)
    rows = torch.tensor([0, 1, n // 2 - 1, n // 2, n - 33, n - 1], device="cuda")
    want, bound = ref.int4(x, codes[rows], scale[rows], None, None)
    rounding = ref.half_step(x.dtype, ref.int4_values(codes[rows], scale[rows], None, k)).t()
    if m > 64:
        bound = bound + x.double().abs() @ rounding
    ref.check(y[:, rows], want, bound)
    pairs = torch.tensor([0, n // 2 - 1, n // 2, n - 1], device="cuda")
    want, bound = ref.int4(x, codes[pairs], scale[pairs], None, None)
    if m > 64:
        bound = bound + x.double().abs() @ ref.half_step(x.dtype, ref.int4_values(codes[pairs], scale[pairs], None, k)).t()
    (gate, up), (d_gate, d_up) = (want[:, :2], want[:, 2:]), (bound[:, :2], bound[:, 2:])
    value, slope = ref.activation(gate, "silu")
    off = (slope.abs() + 2 * d_gate) * d_gate * up.abs() + value.abs() * d_up + d_gate * d_up + ref.ACT * (value * up).abs()
    ref.check(half[:, [0, n // 2 - 1]], value * up, off)


@pytest.mark.parametrize("m", [1, 24, 50, 80])
def test_weights_past_4_gib(fo, m):
    """Read along their rows by the kernels for few rows and by tiles, and across them by dx."""
    k, f, chunks = 16384, 70000, 4
    g = torch.Generator("cuda").manual_seed(0)
    w = torch.empty((2 * f, k), dtype=torch.bfloat16, device="cuda")
    for part in w.chunk(8):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * k**-0.5)
    assert w.numel() * 2 > 1 << 32
    x = torch.randn((m, k), generator=g, device="cuda").bfloat16().requires_grad_()
    y = fo.gated_linear(x, w)
    cols = torch.tensor([0, 1, f // 2, f - 33, f - 1], device="cuda")
    ref.check(y[:, cols], *ref.gated(x.detach(), torch.cat((w[cols], w[f + cols])), None, "silu"))
    if m < 80:
        return
    gy = torch.randn((m, f), generator=g, device="cuda").bfloat16()
    (gx,) = torch.autograd.grad(y, x, gy)
    want, bound = 0, 0
    for at in torch.arange(f, device="cuda").chunk(chunks):   # in parts, for the 64-bit weight's sake
        part = ref.gated_gradients(x.detach(), torch.cat((w[at], w[f + at])), None, "silu", gy[:, at])[0]
        want, bound = want + part[0], bound + part[1]
    ref.check(gx, want, chunks * bound)   # a sum over all of them is off by at most as many times its parts' bounds
