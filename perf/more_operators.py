"""A decoder's feed-forward block in 16 bits and with 4-bit weights, as timed cases: the gated block (both projections, the
activation and the product) with its gradients, and products with 4-bit weights and group scales.

A case is a dict of plain values; `kind` says which public entry points it goes through:

- "gated": `gated_linear`, inference;
- "gated-train": `gated_linear`, forward and backward: gradients for the input, the weight and the bias;
- "int4": one `int4_linear` call;
- "int4-ffn": a decoding step through `layers` feed-forward blocks with 4-bit weights, `int4_gated_linear` and `int4_linear` each
  on the same few rows. The weights together are larger than the GPU's 256 MB last-level cache, so each call reads its own
  from HBM;
- "int4-train": forward and backward of `int4_linear` with its frozen weight: the input's gradient, for adapters before it.

Sizes are `m` rows and `k` inputs; `f` outputs of a gated block (its weight has 2 f rows, the gates' first) or `n` of a product.
`a` is the type of activations, outputs, 16-bit weights and scales, `group` the values to a scale and `zeros` whether groups have
a zero point of their own (else it is 8).
"""

import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = 2  # bytes of either
DEVICE = "cuda"


def listed():
    return [
        # One decoded token through a block's first half.
        dict(name="gated-1", kind="gated", m=1, k=4096, f=14336, a="bf16", act="silu", bias=False),
        # A decoding step of 24 sequences.
        dict(name="gated-24", kind="gated", m=24, k=5120, f=13824, a="fp16", act="silu", bias=False),
        # A prompt of 512 tokens.
        dict(name="gated-512", kind="gated", m=512, k=4096, f=14336, a="bf16", act="silu", bias=False),
        # No dimension is a whole number of tiles.
        dict(name="gated-4097", kind="gated", m=4097, k=2576, f=5000, a="fp16", act="gelu", bias=True),
        # A training step on a ragged batch.
        dict(name="gated-train-1000", kind="gated-train", m=1000, k=5120, f=13824, a="bf16", act="gelu_tanh", bias=True),
        # A training step.
        dict(name="gated-train-4096", kind="gated-train", m=4096, k=4096, f=12288, a="bf16", act="silu", bias=False),
        # One decoded token through an attention projection: launch latency.
        dict(name="int4-1", kind="int4", m=1, k=4096, n=4096, a="fp16", group=128, zeros=False, bias=False),
        # One decoded token through four blocks.
        dict(name="int4-ffn-1", kind="int4-ffn", m=1, k=4096, f=14336, layers=4, a="bf16", act="silu", group=128,
             zeros=False),
        # A decoding step of 24 sequences.
        dict(name="int4-ffn-24", kind="int4-ffn", m=24, k=5120, f=13824, layers=4, a="fp16", act="silu", group=64,
             zeros=True),
        # A prompt of 512 tokens through a projection.
        dict(name="int4-512", kind="int4", m=512, k=5120, n=13824, a="bf16", group=128, zeros=False, bias=True),
        # A long ragged prompt; a row's last group is half full.
        dict(name="int4-4097", kind="int4", m=4097, k=2576, n=5000, a="fp16", group=32, zeros=True, bias=False),
        # An adapter's training step through a frozen layer.
        dict(name="int4-train-1000", kind="int4-train", m=1000, k=4096, n=14336, a="bf16", group=128, zeros=True, bias=False),
    ]


# No drawn case costs more than the largest listed ones.
MAX_MKF = 4096 * 4096 * 12288
MAX_WEIGHT = 5120 * 2 * 13824
MAX_LAYER = 5120 * 13824


def draw(rng):
    def size(low, high, step=1):
        """A multiple of `step`, evenly spread over the logarithm."""
        value = low * (high / low) ** rng.random()
        return min(high, max(low, round(value / step) * step))

    kind = rng.choice(["gated", "gated", "gated", "gated-train", "gated-train", "int4", "int4", "int4", "int4-ffn", "int4-train"])
    case = dict(kind=kind, a=rng.choice(["bf16", "fp16"]))
    step = rng.choice([1, 8, 16, 64])
    gated = kind.startswith("gated")
    if gated or kind == "int4-ffn":
        case["act"] = rng.choice(["silu", "silu", "gelu", "gelu_tanh"])
    if not gated:
        case["group"], case["zeros"] = rng.choice([32, 64, 128, 128]), rng.random() < 0.5
    if kind == "int4-ffn":
        while True:
            k, f = size(2048, 16384, 32), size(2048, 16384, 32)
            if 0.5 * MAX_LAYER < k * f <= MAX_LAYER:
                return case | dict(m=size(1, 64), k=k, f=f, layers=4)
    case["bias"] = rng.random() < 0.3
    while True:
        m, k, n = size(1, 8192), size(128, 16384, step), size(128, 16384, step)
        if m * k * n <= MAX_MKF / (1 if gated else 2) and k * n * (2 if gated else 1) <= MAX_WEIGHT:
            return case | dict(m=m, k=k) | ({"f": n} if gated else {"n": n})


# ---- inputs ----


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def _stream(g, m, n):
    """Normed activations: channels of different sizes, a few of them large."""
    x = _randn(g, m, n) * (_randn(g, n) * 0.5).exp()
    x[:, ::97] *= 8
    return x


def _grad(g, m, n):
    """A gradient: small next to the activations, with a few larger values."""
    grad = _randn(g, m, n)
    return grad * grad.abs() * 1e-3


def _int4(g, n, k, case):
    """A weight as a checkpoint holds it: codes, two to a byte with the even column in the low half, scales and zero points of
    groups, stored group by group."""
    group, dtype = case["group"], DTYPES[case["a"]]
    groups = -(-k // group)
    w = torch.zeros(n, groups * group, device=DEVICE)
    w[:, :k] = _randn(g, n, k) * k**-0.5
    blocks = w.view(n, groups, group)
    if case["zeros"]:
        low, high = blocks.amin(2).clamp(max=0), blocks.amax(2).clamp(min=0)
        scale = ((high - low) / 15).to(dtype)
        zero = (-low / scale.float()).round().clamp(0, 15)
    else:
        scale = (blocks.abs().amax(2) / 7).to(dtype)
        zero = torch.full_like(scale, 8).float()
    q = (blocks / scale.float()[:, :, None]).round().add(zero[:, :, None]).clamp(0, 15).to(torch.uint8).view(n, -1)
    q = q[:, : 2 * -(-k // 2)]
    codes = (q[:, ::2] | q[:, 1::2] << 4).contiguous()
    return codes, scale.t().contiguous().t(), zero.to(torch.uint8).t().contiguous().t() if case["zeros"] else None


def _inputs(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    kind, m, k, dtype = case["kind"], case["m"], case["k"], DTYPES[case["a"]]
    if kind == "int4-ffn":
        f = case["f"]
        return {"blocks": [(_stream(g, m, k).to(dtype), _int4(g, 2 * f, k, case), _stream(g, m, f).to(dtype), _int4(g, k, f, case))
                           for _ in range(case["layers"])]}
    rows, n = (2 * case["f"], case["f"]) if kind.startswith("gated") else (case["n"], case["n"])
    got = {"x": _stream(g, m, k).to(dtype), "bias": (_randn(g, rows) * 0.3).to(dtype) if case["bias"] else None}
    if kind.startswith("gated"):
        got["w"] = (_randn(g, rows, k) * k**-0.5).to(dtype)
    else:
        got["w"] = _int4(g, rows, k, case)
    if kind.endswith("train"):
        got["gy"] = _grad(g, m, n).to(dtype)
    return got


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["kind"].endswith("train"):
        state["x"].requires_grad_()
        if case["kind"] == "gated-train":
            state["w"].requires_grad_()
            if case["bias"]:
                state["bias"].requires_grad_()
    return state


# ---- the framework's calls ----

_feather = None


def _package():
    global _feather
    if _feather is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "feather-ops_amd"))
        import feather_ops

        _feather = feather_ops
    return _feather


def _run_own(state):
    fo, case = _package(), state["case"]
    kind, act = case["kind"], case.get("act")
    if kind == "int4-ffn":
        return [y for x, up, h, down in state["blocks"]
                for y in (fo.int4_gated_linear(x, *up, activation=act), fo.int4_linear(h, *down))]
    x, w, bias = state["x"], state["w"], state["bias"]
    if kind == "gated":
        return fo.gated_linear(x, w, bias, act)
    if kind == "int4":
        return fo.int4_linear(x, *w, bias)
    if kind == "int4-train":
        y = fo.int4_linear(x, *w, bias)
        return [y.detach(), *torch.autograd.grad(y, [x], state["gy"])]
    y = fo.gated_linear(x, w, bias, act)
    return [y.detach(), *torch.autograd.grad(y, [x, w] if bias is None else [x, w, bias], state["gy"])]


# ---- the plain forms, in 32 bits ----

ROOT_HALF = 0.5**0.5
TANH_SLOPE = (8 / 3.141592653589793) ** 0.5
CUBE = 0.044715


def _activation(g, act):
    """(activation, slope) at g."""
    if act == "gelu":
        below = 0.5 * (1 + torch.erf(g * ROOT_HALF))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (2 * 3.141592653589793) ** -0.5
    z = g if act == "silu" else TANH_SLOPE * (g + CUBE * g * g * g)
    slope = 1 if act == "silu" else TANH_SLOPE * (1 + 3 * CUBE * g * g)
    s = torch.sigmoid(z)
    return g * s, s + g * s * torch.sigmoid(-z) * slope


def _values(codes, scale, zero, k):
    """What 4-bit codes stand for."""
    q = torch.stack((codes & 15, codes >> 4), 2).flatten(1)[:, :k].float()
    group = next(size for size in (32, 64, 128) if -(-k // size) == scale.shape[1])
    spread = (lambda t: t.float().repeat_interleave(group, 1)[:, :k])
    return (q - (8 if zero is None else spread(zero))) * spread(scale)


def _project(x, w, bias):
    y = x.float() @ w.float().t()
    return y if bias is None else y + bias.float()


def _gate(h, act):
    gate, up = h.chunk(2, 1)
    return _activation(gate, act)[0] * up


def _run_plain(state):
    case = state["case"]
    kind, dtype, act = case["kind"], DTYPES[case["a"]], case.get("act")
    if kind == "int4-ffn":
        return [y for x, up, h, down in state["blocks"]
                for y in (_gate(_project(x, _values(*up, x.shape[1]), None), act).to(dtype),
                          _project(h, _values(*down, h.shape[1]), None).to(dtype))]
    x, bias = state["x"].detach(), None if state["bias"] is None else state["bias"].detach()
    if kind.startswith("int4"):
        w = _values(*state["w"], case["k"])
        y = _project(x, w, bias).to(dtype)
        return y if kind == "int4" else [y, (state["gy"].float() @ w).to(dtype)]
    w = state["w"].detach()
    h = _project(x, w, bias)
    if kind == "gated":
        return _gate(h, act).to(dtype)
    gate, up = h.chunk(2, 1)
    value, slope = _activation(gate, act)
    gy = state["gy"].float()
    gh = torch.cat((gy * up * slope, gy * value), 1)
    got = [(value * up).to(dtype), (gh @ w.float()).to(dtype), (gh.t() @ x.float()).to(dtype)]
    return got if bias is None else [*got, gh.sum(0).to(dtype)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----


def work(case):
    kind, m, k = case["kind"], case["m"], case["k"]

    def weight(n, k):
        return n * -(-k // 2) + n * -(-k // case["group"]) * (SIZE + case["zeros"])

    if kind == "int4-ffn":
        f = case["f"]
        one = weight(2 * f, k) + weight(k, f) + 2 * SIZE * m * (k + f)
        return {"bytes": case["layers"] * one, "flops": case["layers"] * 6 * m * f * k}
    if kind.startswith("gated"):
        f = case["f"]
        one = SIZE * (m * k + 2 * f * k + m * f + (2 * f if case["bias"] else 0))
        return {"bytes": one, "flops": 4 * m * f * k} if kind == "gated" else {"bytes": 2 * one, "flops": 12 * m * f * k}
    n = case["n"]
    bias = SIZE * n if case["bias"] else 0
    if kind == "int4":
        return {"bytes": weight(n, k) + SIZE * m * (k + n) + bias, "flops": 2 * m * n * k}
    return {"bytes": weight(n, k) + 2 * SIZE * m * (k + n) + bias, "flops": 4 * m * n * k}


# ---- the definitions, in 64 bits ----


def _exact_weight(codes, scale, zero, k):
    n = codes.shape[0]
    j = torch.arange(k, device=codes.device)
    q = codes.int()[:, j // 2].bitwise_right_shift(4 * (j % 2).int()).bitwise_and(15).double()
    group = [size for size in (128, 64, 32) if (k + size - 1) // size == scale.shape[1]][0]
    z = torch.full((n, k), 8.0, dtype=torch.float64, device=codes.device) if zero is None else zero.double()[:, j // group]
    return (q - z) * scale.double()[:, j // group]


def _exact_gate(g, act):
    """The activation and its slope, from exponentials of |g| and the normal distribution's function."""
    if act == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g.square() / 2) / (2 * torch.pi) ** 0.5
    if act == "silu":
        e = torch.exp(-g.abs())
        s = torch.where(g < 0, e, torch.ones_like(e)) / (1 + e)
        return g * s, s * (1 + g * (1 - s))
    t = torch.tanh((2 / torch.pi) ** 0.5 * (g + 0.044715 * g.pow(3)))
    return g * (1 + t) / 2, (1 + t) / 2 + g / 2 * (1 - t.square()) * (2 / torch.pi) ** 0.5 * (1 + 0.134145 * g.square())


def exact(case, seed):
    inputs = _inputs(case, seed)
    kind, k, act = case["kind"], case["k"], case.get("act")
    if kind == "int4-ffn":
        got = []
        for x, up, h, down in inputs["blocks"]:
            both = x.double() @ _exact_weight(*up, k).t()
            got += [_exact_gate(both[:, : case["f"]], act)[0] * both[:, case["f"] :],
                    h.double() @ _exact_weight(*down, case["f"]).t()]
        return got
    x = inputs["x"].double()
    w = inputs["w"].double() if kind.startswith("gated") else _exact_weight(*inputs["w"], k)
    y = torch.mm(x, w.t())
    if inputs["bias"] is not None:
        y += inputs["bias"].double()
    if kind == "int4":
        return y
    if kind == "int4-train":
        return [y, torch.mm(inputs["gy"].double(), w)]
    value, slope = _exact_gate(y[:, : case["f"]], act)
    up = y[:, case["f"] :]
    if kind == "gated":
        return value * up
    gy = inputs["gy"].double()
    gg, gu = gy * slope * up, gy * value
    got = [value * up, gg @ w[: case["f"]] + gu @ w[case["f"] :], torch.cat((gg.t() @ x, gu.t() @ x))]
    return got if inputs["bias"] is None else [*got, torch.cat((gg.sum(0), gu.sum(0)))]
