"""The gated feed-forward block's first half in one kernel, `act(x Wg^T + bg) * (x Wu^T + bu)`, in 16 bits, with gradients; not in
the reference. Kernels: `csrc/linear_tile.h` (and the products of the backward), `csrc/linear_few.h` (few rows),
`csrc/linear_ops.hip`; autograd node: `csrc/linear_autograd.cpp`. C ABI: `include/feather_linear_ops.h`.

The weight holds both projections, `[2 F, K]`: the gates' rows first, as `silu_mul` takes their outputs.
"""

import functools

import torch
from torch import nn

from . import _lib
from .block_scaled import _workspace, as_rows

_ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
HALVES = (torch.bfloat16, torch.float16)

# The C ABI's limit of the stride from row to row, and of K.
_FAR = 1 << 21


def activation_number(activation: str) -> int:
    try:
        return _ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}") from None


def activate(gate: torch.Tensor, activation: int) -> torch.Tensor:
    if activation == 0:
        return nn.functional.silu(gate)
    return nn.functional.gelu(gate, approximate="tanh" if activation == 2 else "none")


def operand(x: torch.Tensor) -> torch.Tensor:
    """The matrix x as the products read it: rows on 16-byte boundaries, of whole pieces of 8 values, with zeros behind the last
    (copied where they are not)."""
    rows, cols = x.shape
    if cols % 8:
        return nn.functional.pad(x, (0, -cols % 8))
    if x.storage_offset() % 8 or (rows > 1 and (x.stride(0) % 8 or x.stride(0) > _FAR)):
        return x.clone(memory_format=torch.contiguous_format)
    return x


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(M: int, F: int, K: int, need_x: bool, need_weight: bool) -> int:
    """For the block, and for the products of the gradients that are needed."""
    lib = _lib.c_library()
    need = [lib.feather_gated_linear_workspace_bytes(M, F, K)]
    if need_x:
        need.append(lib.feather_product_workspace_bytes(M, K, 2 * F))
    if need_weight:
        need.append(lib.feather_product_workspace_bytes(2 * F, K, M))
    if min(need) < 0:
        raise ValueError(f"sizes are out of range: x [{M}, {K}], weight [{2 * F}, {K}]")
    return max(need)


def check_depth(of: str, depth: int, what: str) -> None:
    """A gradient's sum is no longer than a product's."""
    if depth > _FAR:
        raise ValueError(f"the gradient of {of} is a sum over {what}, at most {_FAR} of them, got {depth}")


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 activation: str = "silu") -> torch.Tensor:
    """`act(x @ Wg^T + bg) * (x @ Wu^T + bu)`: x `[..., K]`, weight `[2 F, K]` (Wg's rows, then Wu's), bias `[2 F]`, the result
    `[..., F]`. x and weight are both bfloat16 or both float16; bias is taken in their dtype. activation: "silu", "gelu" or
    "gelu_tanh" (its approximation). Sums, activation and product are fp32, rounded once.

    Differentiable once, in reverse mode, in x, weight and bias; for that both sums are kept in fp32 (8 F bytes a row), and their
    gradients rounded to x's dtype. Rows of x and weight that do not start on 16-byte boundaries, or whose length is no multiple
    of 8, are copied on every call. K is at most 2**21, and so are 2 F where x takes a gradient and x's rows where the weight does."""
    act = activation_number(activation)
    if x.dtype not in HALVES or weight.dtype != x.dtype:
        raise ValueError(f"x and weight must both be bfloat16 or both float16, got {x.dtype} and {weight.dtype}")
    if weight.dim() != 2 or weight.shape[0] % 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., K] and weight [2 F, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None:
        if bias.shape != weight.shape[:1]:
            raise ValueError(f"bias must have {weight.shape[0]} values, got {tuple(bias.shape)}")
        bias = bias.to(x.dtype).contiguous()
    if x.numel() == 0 or weight.numel() == 0:
        gate, up = nn.functional.linear(x, weight, bias).chunk(2, -1)
        return activate(gate, act) * up
    if (x.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        if x.requires_grad:
            check_depth("x", weight.shape[0], "the weight's rows")
        if weight.requires_grad:
            check_depth("the weight", x.numel() // x.shape[-1], "the rows of x")
    if torch.compiler.is_compiling():
        return _gated_linear_auto(x, weight, bias, act)
    return _gated(x, weight, bias, act)


def _gated(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, act: int) -> torch.Tensor:
    rows, weight = operand(as_rows(x)), operand(as_rows(weight))
    need_x, need_weight = rows.requires_grad, weight.requires_grad
    if not torch.is_grad_enabled():
        need_x = need_weight = False
    need = _workspace_bytes(int(rows.shape[0]), int(weight.shape[0]) // 2, int(rows.shape[1]), need_x, need_weight)
    y = torch.ops.feather_ops.gated_linear.default(rows, weight, bias, act, _workspace(rows, need) if need else None)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


# ---- one node under torch.compile ----


@torch.library.custom_op("feather_ops::gated_linear_auto", mutates_args=())
def _gated_linear_auto(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, act: int) -> torch.Tensor:
    """gated_linear as one opaque op."""
    return _gated(x, weight, bias, act)


@_gated_linear_auto.register_fake
def _(x, weight, bias, act):
    return x.new_empty((*x.shape[:-1], weight.shape[0] // 2))


@torch.library.custom_op("feather_ops::gated_linear_auto_backward", mutates_args=())
def _gated_linear_auto_backward(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, act: int,
                                need_x: bool, need_weight: bool,
                                need_bias: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of x, weight and bias, each empty where it is not asked for. What they need of the forward is computed
    again: x and the weight a traced program holds anyway."""
    ops = torch.ops.feather_ops
    k = x.shape[-1]
    rows, padded = operand(as_rows(x)), operand(as_rows(weight))
    need = _workspace_bytes(rows.shape[0], weight.shape[0] // 2, rows.shape[1], need_x, need_weight)
    workspace = _workspace(rows, need) if need else None
    kept = ops.gated_forward.default(rows, padded, bias, act, True, workspace)[1]
    grad_x, grad_weight, grad_bias = ops.gated_backward.default(as_rows(grad), kept, rows, padded, act, need_x, need_weight,
                                                                need_bias, workspace)
    if need_x:
        grad_x = grad_x[:, :k].contiguous().reshape(x.shape)
    if need_weight:
        grad_weight = grad_weight[:, :k].contiguous()
    return grad_x, grad_weight, grad_bias


@_gated_linear_auto_backward.register_fake
def _(grad, x, weight, bias, act, need_x, need_weight, need_bias):
    return (x.new_empty(x.shape if need_x else (0, 0)), weight.new_empty(weight.shape if need_weight else (0, 0)),
            x.new_empty((weight.shape[0],) if need_bias else (0,)))


def _auto_context(ctx, inputs, output) -> None:
    x, weight, bias, ctx.act = inputs
    ctx.save_for_backward(x, weight, bias)


def _auto_backward(ctx, grad: torch.Tensor) -> tuple:
    needs = ctx.needs_input_grad[:3]
    grads = _gated_linear_auto_backward(grad, *ctx.saved_tensors, ctx.act, *needs)
    return (*(g if need else None for g, need in zip(grads, needs)), None)


_gated_linear_auto.register_autograd(_auto_backward, setup_context=_auto_context)


# ---- shapes, for tracing ----


@torch.library.register_fake("feather_ops::gated_forward")
def _(x, weight, bias, activation, keep, workspace):
    f = weight.shape[0] // 2
    kept = (x.shape[0], 2 * ((f + 7) // 8 * 8)) if keep else (0, 0)
    return x.new_empty((x.shape[0], f)), x.new_empty(kept, dtype=torch.float32)


@torch.library.register_fake("feather_ops::gated_backward")
def _(grad_y, kept, x, weight, activation, need_x, need_weight, need_bias, workspace):
    return (x.new_empty(x.shape if need_x else (0, 0)), x.new_empty(weight.shape if need_weight else (0, 0)),
            x.new_empty((weight.shape[0],) if need_bias else (0,)))
