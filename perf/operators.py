"""The operators of fp8 models with a scale for each block of 128 values, as timed cases: the block-scaled product and its
gradients, the root-mean-square norm with the residual's addition, and the gated activation.

A case is a dict of plain values; `kind` says which public entry point it goes through:

- "norm": `rms_norm_quantized`, a decoder layer's residual addition and norm ahead of an fp8 product;
- "norm-train": `rms_norm`, forward and backward;
- "mm": one `block_scaled_mm` call on quantized operands;
- "decode": the feed-forward weights of `layers` decoder layers, one product each on the same few rows. The weights
  together are larger than the GPU's 256 MB last-level cache, so each call reads its own from HBM;
- "linear": inference through an `nn.Linear` relabelled by `to_block_scaled_linear`: 16-bit activations in and out;
- "train": forward and backward of `block_scaled_linear`: gradients for the input, the weight and the bias;
- "gate": `silu_mul_quantized`, the gated activation ahead of an MLP's down projection;
- "gate-train": `silu_mul`, forward and backward.

Sizes are `m` rows, `n` output columns and `k` inputs (the norm's and the gate's width is `n`). `a` is the type of the
16-bit (or fp32) inputs and outputs, `q` the fp8 format.
"""

import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
BLOCK = 128
LEAST = 2.0**-100  # blocks whose values are all smaller are scaled as if their largest were this
EPS = 1e-6
DEVICE = "cuda"


def listed():
    return [
        # One decoded token between two layers: launch latency.
        dict(name="norm-1", kind="norm", m=1, n=4096, a="bf16", q="e4m3", residual=True),
        # The norm of 4096 image and 16 text tokens: a stream through memory.
        dict(name="norm-4112", kind="norm", m=4112, n=5120, a="fp16", q="e4m3", residual=True),
        # A training step's norm.
        dict(name="norm-train-4096", kind="norm-train", m=4096, n=4096, a="bf16", residual=True),
        # One decoded token through the feed-forward weights of four layers.
        dict(name="decode-1", kind="decode", m=1, n=14336, k=4096, layers=4, a="bf16", q="e4m3"),
        # A decoding step of 24 sequences.
        dict(name="decode-24", kind="decode", m=24, n=14336, k=4096, layers=4, a="fp16", q="e4m3"),
        # A prompt of 512 tokens through an up projection.
        dict(name="mm-512", kind="mm", m=512, n=13824, k=5120, a="fp16", q="e4m3", bias=False, by_row=False),
        # No dimension is a whole number of tiles.
        dict(name="mm-4097", kind="mm", m=4097, n=5000, k=2576, a="bf16", q="e4m3", bias=True, by_row=False),
        # A long prompt through a whole layer, from 16-bit activations to 16-bit outputs.
        dict(name="linear-4096", kind="linear", m=4096, n=14336, k=4096, a="bf16", q="e4m3", bias=False),
        # A training step of an up projection.
        dict(name="train-4096", kind="train", m=4096, n=12288, k=4096, a="bf16", q="e4m3", bias=True),
        # The gate of a decoding step of 16 sequences.
        dict(name="gate-16", kind="gate", m=16, n=14336, a="bf16", q="e4m3"),
        # The gate of a long prompt.
        dict(name="gate-4096", kind="gate", m=4096, n=12288, a="fp16", q="e4m3"),
        # A training step's gate on a ragged batch.
        dict(name="gate-train-1000", kind="gate-train", m=1000, n=13824, a="bf16"),
    ]


# No drawn case costs more than the largest listed ones.
MAX_MNK = 4096 * 14336 * 4096
MAX_TRAIN = 4096 * 12288 * 4096
MAX_DECODE_WEIGHT = 14336 * 4096
MAX_STREAM = 4096 * 12288


def draw(rng):
    def size(low, high, step=1):
        """A multiple of `step`, evenly spread over the logarithm."""
        value = low * (high / low) ** rng.random()
        return min(high, max(low, round(value / step) * step))

    kind = rng.choice(["norm", "norm", "norm-train", "mm", "mm", "mm", "decode", "linear", "train", "gate", "gate",
                       "gate-train"])
    a, q = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "e4m3", "e5m2"])
    step = rng.choice([1, 8, 16, 64])
    while True:
        m = size(1, 8192)
        if kind in ("norm", "norm-train", "gate", "gate-train"):
            n = size(128, 16384, step)
            if m * n > MAX_STREAM:
                continue
            if kind.startswith("norm"):
                a = rng.choice(["bf16", "fp16", "fp32"])
            case = dict(kind=kind, m=m, n=n, a=a)
            if kind.startswith("norm"):
                case["residual"] = rng.random() < 0.7
            if not kind.endswith("train"):
                case["q"] = q
            return case
        n, k = size(128, 16384, step), size(128, 16384, max(step, 16))
        if kind == "decode":
            n, k = size(2048, 16384, 16), size(2048, 16384, 16)
            if not 0.5 * MAX_DECODE_WEIGHT < n * k <= MAX_DECODE_WEIGHT:
                continue
            return dict(kind=kind, m=size(1, 128), n=n, k=k, layers=4, a=a, q=q)
        if m * n * k > (MAX_TRAIN if kind == "train" else MAX_MNK):
            continue
        if kind == "mm":
            return dict(kind=kind, m=m, n=n, k=k, a=a, q=q, bias=rng.random() < 0.3, by_row=rng.random() < 0.3)
        return dict(kind=kind, m=m, n=n, k=k, a=a, q="e4m3" if kind == "train" else q, bias=rng.random() < 0.5)


# ---- inputs ----


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def _quantized(x, q, rows=1):
    """fp8 codes and scales of random data. Scales of rows are stored block by block, as the framework's quantized outputs
    hold them."""
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // BLOCK)
    padded = torch.zeros(mb * rows, kb * BLOCK, device=DEVICE)
    padded[:m, :k] = x
    scale = padded.view(mb, rows, kb, BLOCK).abs().amax((1, 3)) / LARGEST[q]
    codes = x / scale.repeat_interleave(rows, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]
    return codes.to(DTYPES[q]), scale.t().contiguous().t() if rows == 1 else scale


def _weight(g, n, k, q, by_row=False):
    return _quantized(_randn(g, n, k) * k**-0.5, q, 1 if by_row else BLOCK)


def _stream(g, m, n):
    """Activations of a residual stream: channels of different sizes, a few of them large."""
    x = _randn(g, m, n) * (_randn(g, n) * 0.5).exp()
    x[:, ::97] *= 8
    return x


def _inputs(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    kind, m, n, dtype = case["kind"], case["m"], case["n"], DTYPES[case["a"]]
    if kind in ("norm", "norm-train"):
        got = {"x": _stream(g, m, n).to(dtype), "w": (1 + 0.2 * _randn(g, n)).to(dtype),
               "residual": _stream(g, m, n).to(dtype) if case["residual"] else None}
        if kind == "norm-train":
            got["gy"] = (_randn(g, m, n) * 1e-3).to(dtype)
            got["gh"] = (_randn(g, m, n) * 1e-3).to(dtype) if case["residual"] else None
        return got
    if kind in ("gate", "gate-train"):
        got = {"x": (_randn(g, m, 2 * n) * 1.5).to(dtype)}
        if kind == "gate-train":
            got["gy"] = (_randn(g, m, n) * 1e-3).to(dtype)
        return got
    k, q = case["k"], case["q"]
    if kind == "decode":
        return {"pairs": [(*_quantized(_stream(g, m, kk), q), *_weight(g, nn, kk, q))
                          for _ in range(case["layers"]) for nn, kk in ((n, k), (k, n))]}
    bias = _randn(g, n).to(dtype) if case["bias"] else None
    if kind == "mm":
        return {"a": _quantized(_stream(g, m, k), q), "b": _weight(g, n, k, q, case["by_row"]), "bias": bias}
    got = {"x": _stream(g, m, k).to(dtype), "w": (_randn(g, n, k) * k**-0.5).to(dtype), "bias": bias}
    if kind == "train":  # gradients are small next to the activations, with a few larger ones
        grad = _randn(g, m, n)
        got["gy"] = (grad * grad.abs() * 1e-3).to(dtype)
    return got


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["kind"] in ("norm-train", "gate-train", "train"):
        for name in ("x", "residual", "w", "bias"):
            if state.get(name) is not None:
                state[name].requires_grad_()
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


def _layer(state, fo):
    """The quantized layer that a user's program keeps: its weight is laid out once."""
    if "layer" not in state:
        case = state["case"]
        layer = torch.nn.Linear(case["k"], case["n"], bias=case["bias"], device="meta", dtype=DTYPES[case["a"]])
        layer.weight = torch.nn.Parameter(state["w"], requires_grad=False)
        if case["bias"]:
            layer.bias = torch.nn.Parameter(state["bias"], requires_grad=False)
        fo.to_block_scaled_linear(layer, DTYPES[case["q"]])
        state["layer"] = layer
    return state["layer"]


def _run_own(state):
    fo, case = _package(), state["case"]
    kind = case["kind"]
    if kind == "mm":
        return fo.block_scaled_mm(*state["a"], *state["b"], state["bias"], DTYPES[case["a"]])
    if kind == "decode":
        return [fo.block_scaled_mm(*pair, None, DTYPES[case["a"]]) for pair in state["pairs"]]
    if kind == "linear":
        with torch.no_grad():
            return _layer(state, fo)(state["x"])
    if kind == "train":
        y = fo.block_scaled_linear(state["x"], state["w"], state["bias"])
        wanted = [state[n] for n in ("x", "w", "bias") if state[n] is not None]
        return [y.detach(), *torch.autograd.grad(y, wanted, state["gy"])]
    if kind == "norm":
        return fo.rms_norm_quantized(state["x"], state["w"], state["residual"], EPS, DTYPES[case["q"]])
    if kind == "norm-train":
        if state["residual"] is None:
            y = fo.rms_norm(state["x"], state["w"], None, EPS)
            return [y.detach(), *torch.autograd.grad(y, (state["x"], state["w"]), state["gy"])]
        y, h = fo.rms_norm(state["x"], state["w"], state["residual"], EPS)
        grads = torch.autograd.grad((y, h), (state["x"], state["residual"], state["w"]), (state["gy"], state["gh"]))
        return [y.detach(), h.detach(), *grads]
    if kind == "gate":
        return fo.silu_mul_quantized(state["x"], DTYPES[case["q"]])
    y = fo.silu_mul(state["x"])
    return [y.detach(), *torch.autograd.grad(y, state["x"], state["gy"])]


# ---- the plain forms, in 32 bits ----


def _quantize(x, q, rows=1):
    m, k = x.shape
    padded = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -m % rows))
    blocks = padded.view(padded.shape[0] // rows, rows, -1, BLOCK)
    scale = blocks.abs().amax((1, 3), keepdim=True).clamp(min=LEAST) / LARGEST[q]
    codes = (blocks / scale).view(padded.shape)[:m, :k].to(DTYPES[q])
    return codes, scale[:, 0, :, 0]


def _values(codes, scale):
    """What codes [R, K] and scales [R or ceil(R / 128), ceil(K / 128)] stand for."""
    r, k = codes.shape
    if scale.shape[0] != r:
        scale = scale.repeat_interleave(BLOCK, 0)[:r]
    return codes.float() * scale.repeat_interleave(BLOCK, 1)[:, :k]


def _mm(a, a_scale, b, b_scale, bias, dtype):
    y = _values(a, a_scale) @ _values(b, b_scale).t()
    return (y if bias is None else y + bias.float()).to(dtype)


def _run_plain(state):
    case = state["case"]
    kind, dtype, q = case["kind"], DTYPES[case["a"]], case.get("q")
    if kind == "mm":
        return _mm(*state["a"], *state["b"], state["bias"], dtype)
    if kind == "decode":
        return [_mm(*pair, None, dtype) for pair in state["pairs"]]
    if kind == "linear":
        if "layer" not in state:  # the weight is quantized once, as a user's program does
            state["layer"] = _quantize(state["w"].float(), q, BLOCK)
        return _mm(*_quantize(state["x"].float(), q), *state["layer"], state["bias"], dtype)
    x = state["x"].detach().float()
    if kind == "train":
        w, gy = _quantize(state["w"].detach().float(), q, BLOCK), state["gy"].float()
        bias = None if state["bias"] is None else state["bias"].detach()
        y = _mm(*_quantize(x, q), *w, bias, dtype)
        gx = (_values(*_quantize(gy, q)) @ _values(*w)).to(dtype)
        gw = (_values(*_quantize(gy.t(), q)) @ _values(*_quantize(x.t(), q)).t()).to(dtype)
        return [y, gx, gw] if bias is None else [y, gx, gw, gy.sum(0).to(dtype)]
    if kind in ("norm", "norm-train"):
        w = state["w"].detach().float()
        h = state["x"].detach()
        if state["residual"] is not None:
            h = (x + state["residual"].detach().float()).to(dtype)
        r = torch.rsqrt(h.float().square().mean(1, keepdim=True) + EPS)
        normed = h.float() * r
        if kind == "norm":
            codes, scale = _quantize(normed * w, q)
            return (codes, scale) if state["residual"] is None else (codes, scale, h)
        gy = state["gy"].float()
        g = gy * w
        gh = r * (g - normed * (g * normed).mean(1, keepdim=True))
        gw = (gy * normed).sum(0).to(dtype)
        y = (normed * w).to(dtype)
        if state["residual"] is None:
            return [y, gh.to(dtype), gw]
        gh = (gh + state["gh"].float()).to(dtype)
        return [y, h, gh, gh, gw]
    gate, up = x[:, : case["n"]], x[:, case["n"] :]
    s = torch.sigmoid(gate)
    y = gate * s * up
    if kind == "gate":
        return _quantize(y, q)
    gy = state["gy"].float()
    return [y.to(dtype), torch.cat([gy * up * s * (1 + gate * (1 - s)), gy * gate * s], 1).to(dtype)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----


def work(case):
    kind, m, n, size = case["kind"], case["m"], case["n"], BYTES[case["a"]]
    nb = -(-n // BLOCK)
    if kind == "norm":
        streams = 3 if case["residual"] else 1  # x, the residual in and out
        return {"bytes": streams * size * m * n + size * n + m * (n + 4 * nb), "flops": 6 * m * n}
    if kind == "norm-train":  # x, y; the stream, dy, dx; with a residual it, its sum and its gradient
        streams = (2 + 3) + (3 if case["residual"] else 0)
        return {"bytes": streams * size * m * n + 3 * size * n, "flops": 16 * m * n}
    if kind == "gate":
        return {"bytes": 2 * size * m * n + m * (n + 4 * nb), "flops": 8 * m * n}
    if kind == "gate-train":
        return {"bytes": (3 + 5) * size * m * n, "flops": 20 * m * n}
    k = case["k"]
    kb = -(-k // BLOCK)
    if kind == "decode":
        one = n * k + (m + size * m) * (n + k) / 2 + 4 * (m + nb) * kb
        return {"bytes": 2 * case["layers"] * one, "flops": 4 * case["layers"] * m * n * k}
    bias = size * n if case["bias"] else 0
    if kind == "mm":
        b_scales = (n if case["by_row"] else nb) * kb
        return {"bytes": m * k + n * k + size * m * n + 4 * (m * kb + b_scales) + bias, "flops": 2 * m * n * k}
    if kind == "linear":
        return {"bytes": size * m * k + n * k + size * m * n + 4 * nb * kb + bias, "flops": 2 * m * n * k}
    # train: x, w and dy in; y, dx and dw out
    return {"bytes": 2 * size * (m * k + n * k + m * n) + 2 * bias, "flops": 6 * m * n * k}


# ---- the definitions, in 64 bits ----


def _exact_blocks(x, q, axis, square=False):
    """(codes, scales) of a 64-bit matrix with blocks of 128 along `axis`, or of 128 x 128; scales spread to x's shape."""
    r, c = x.shape
    rows, cols = (BLOCK if square or axis == 0 else 1), (BLOCK if square or axis == 1 else 1)
    spread = x.new_empty(r, c)
    amax = torch.zeros(-(-r // rows), -(-c // cols), dtype=torch.float64, device=x.device)
    i, j = torch.arange(r, device=x.device) // rows, torch.arange(c, device=x.device) // cols
    by_rows = torch.zeros(amax.shape[0], c, dtype=torch.float64, device=x.device).index_reduce_(0, i, x.abs(), "amax")
    amax.index_reduce_(1, j, by_rows, "amax")
    scales = torch.where(amax > LEAST, amax, torch.full_like(amax, LEAST)) / LARGEST[q]
    spread = scales[i][:, j]
    return (x / spread).to(DTYPES[q]), scales, spread


def _exact_values(x, q, axis, square=False):
    codes, _, spread = _exact_blocks(x, q, axis, square)
    return codes.double() * spread


def _spread(codes, scale):
    r, c = codes.shape
    rows = 1 if scale.shape[0] == r else BLOCK
    i, j = torch.arange(r, device=codes.device) // rows, torch.arange(c, device=codes.device) // BLOCK
    return codes.double() * scale.double()[i][:, j]


def exact(case, seed):
    inputs = _inputs(case, seed)
    kind, n, q = case["kind"], case["n"], case.get("q")
    if kind == "decode":
        return [_spread(a, sa) @ _spread(b, sb).t() for a, sa, b, sb in inputs["pairs"]]
    if kind == "mm":
        y = _spread(*inputs["a"]) @ _spread(*inputs["b"]).t()
        return y if inputs["bias"] is None else y + inputs["bias"].double()
    x = inputs["x"].double()
    if kind in ("linear", "train"):
        w = _exact_values(inputs["w"].double(), q, 1, square=True)
        y = _exact_values(x, q, 1) @ w.t()
        if inputs["bias"] is not None:
            y = y + inputs["bias"].double()
        if kind == "linear":
            return y
        gy = inputs["gy"].double()
        got = [y, _exact_values(gy, q, 1) @ w, _exact_values(gy, q, 0).t() @ _exact_values(x, q, 0)]
        return got if inputs["bias"] is None else [*got, gy.sum(0)]
    if kind in ("norm", "norm-train"):
        w, residual = inputs["w"].double(), inputs["residual"]
        if residual is not None:  # the stream is held in its type, and normed as held
            x = (x + residual.double()).to(DTYPES[case["a"]]).double()
        r = (x.pow(2).sum(1, keepdim=True) / n + EPS).pow(-0.5)
        y = x * r * w
        if kind == "norm":
            codes, scales, _ = _exact_blocks(y, q, 1)
            got = (codes.double(), scales)
            return got if residual is None else (*got, x)
        gy = inputs["gy"].double()
        gx = r * w * gy - x * r.pow(3) * (w * gy * x).sum(1, keepdim=True) / n
        gw = (gy * x * r).sum(0)
        if residual is None:
            return [y, gx, gw]
        gx = gx + inputs["gh"].double()
        return [y, x, gx, gx, gw]
    g, u = x.split(n, 1)
    e = torch.exp(-g)
    y = g * u / (1 + e)
    if kind == "gate":
        codes, scales, _ = _exact_blocks(y, q, 1)
        return codes.double(), scales
    gy = inputs["gy"].double()
    return [y, torch.cat([gy * u * (1 + e + g * e) / (1 + e).pow(2), gy * g / (1 + e)], 1)]
