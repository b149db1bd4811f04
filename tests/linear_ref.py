"""The gated block and 4-bit products in 64 bits, with a bound of what an fp32 computation that rounds its result once may be off.

Sums: a matrix instruction adds 32 products to a running fp32 sum, each addition off by at most one part in 2^24 of what is
there, so a sum of K is within (K / 32 + 32) 2^-24 of the sum of its terms' magnitudes. A rounding is off by half a step."""

import math

import torch

ULP = 2.0**-24
HALVES = [torch.bfloat16, torch.float16]
ACTIVATIONS = ["silu", "gelu", "gelu_tanh"]


def half_step(dtype, value):
    """What rounding to dtype may change of a value (of subnormal ones, half their common step)."""
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return torch.finfo(dtype).eps / 2 * value.abs() + least


def sum_error(k, magnitude):
    return (k / 32 + 34) * ULP * magnitude


def activation(g, act):
    """(value, slope)."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g)
    if act == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)
    t = torch.tanh(u)
    return g * torch.sigmoid(2 * u), torch.sigmoid(2 * u) + g / 2 * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g)


# The activations' own error: the argument of the exponential is off by its rounding, |z| <= 100 where the result counts, and a
# few operations more.
ACT = 2.0**-16


def gated(x, w, bias, act):
    """(value, bound) of y but for its rounding."""
    return _gated(x, w, bias, act)[:2]


def _gated(x, w, bias, act):
    x, w = x.double(), w.double()
    f, k = w.shape[0] // 2, w.shape[1]
    b = torch.zeros(2 * f, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    h, size = x @ w.t() + b, x.abs() @ w.abs().t() + b.abs()
    gate, up = h.chunk(2, 1)
    d_gate, d_up = sum_error(k, size).chunk(2, 1)
    value, slope = activation(gate, act)
    y = value * up
    return y, (slope.abs() + 2 * d_gate) * d_gate * up.abs() + value.abs() * d_up + d_gate * d_up + ACT * y.abs(), (
        gate, up, value, slope, d_gate, d_up)


def gated_gradients(x, w, bias, act, gy):
    """[(value, bound)] of the gradients of x, w and bias (but for their rounding; the sums' gradients are rounded to the type)."""
    dtype, k = x.dtype, x.shape[1]
    gate, up, value, slope, d_gate, d_up = _gated(x, w, bias, act)[2]
    x, w, gy = x.double(), w.double(), gy.double()
    gh = torch.cat((gy * up * slope, gy * value), 1)
    # a slope changes by at most 1.1 times its argument's change
    off = torch.cat((gy.abs() * (up.abs() * 1.1 * d_gate + slope.abs() * d_up + 1.1 * d_gate * d_up),
                     gy.abs() * 1.1 * d_gate), 1) + ACT * (gh.abs() + (gy * up).abs().repeat(1, 2) * 2.0**-6)
    rounded = off + half_step(dtype, gh.abs() + off)
    got = [(gh @ w, rounded @ w.abs() + sum_error(w.shape[0], gh.abs() @ w.abs())),
           (gh.t() @ x, rounded.t() @ x.abs() + sum_error(x.shape[0], gh.abs().t() @ x.abs()))]
    if bias is not None:
        got.append((gh.sum(0), off.sum(0) + (x.shape[0] + 34) * ULP * gh.abs().sum(0)))
    return got


def int4_values(codes, scale, zero, k):
    """The weight that codes stand for, in 64 bits."""
    q = torch.stack((codes & 15, codes >> 4), 2).flatten(1)[:, :k].double()
    group = next(size for size in (32, 64, 128) if -(-k // size) == scale.shape[1])
    z = 8.0 if zero is None else zero.double().repeat_interleave(group, 1)[:, :k]
    return (q - z) * scale.double().repeat_interleave(group, 1)[:, :k]


def int4(x, codes, scale, zero, bias):
    """(value, bound) of y from the codes as they are. In bf16 a group's sums are of codes + 128, in fp16 of codes - 8, and of x
    for the zero points: magnitudes of up to 143 + 143 for 15."""
    k = x.shape[1]
    w = int4_values(codes, scale, zero, k)
    group = next(size for size in (32, 64, 128) if -(-k // size) == scale.shape[1])
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if bias is None else bias.double()
    spread = scale.double().abs().repeat_interleave(group, 1)[:, :k]
    widest = 286.0 if x.dtype == torch.bfloat16 else 22.0
    inner = (min(k, 128) / 32 + 34) * ULP * (x.double().abs() @ (spread * widest).t())
    outer = sum_error(k, x.double().abs() @ w.abs().t() + b.abs())
    return x.double() @ w.t() + b, inner + outer


def check(got, want, bound):
    """got is want within bound and its own rounding."""
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    allowed = bound + half_step(got.dtype, want.abs() + bound)
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times what the computation may be off"
