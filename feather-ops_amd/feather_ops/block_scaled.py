"""Products of two fp8 matrices with one scale for each block of 128 values, and the layers on them; not in the
reference, whose weights have one scale per tensor or column.

A quantized matrix is a pair (codes, scale): fp8 codes `[rows, K]` and fp32 scales `[rows, ceil(K / 128)]`, one for each
row and 128 columns, or `[ceil(rows / 128), ceil(K / 128)]`, one for each 128 x 128 square (weights). Codes times scales
are the values; a block's scale is its largest magnitude (at least 2**-100) over the format's largest value. The functions
here store rows of codes padded to 64 bytes and scales block by block (`scale.t()` is contiguous), which is what the
product reads fastest; it takes any strides.

Kernels: `csrc/block_scaled_mm.hip`, `csrc/quantize_tiles.hip`, `csrc/silu_mul.hip`; the layer and its
autograd node: `csrc/block_autograd.cpp`. C ABI: `include/feather_block_ops.h`.
"""

import functools
from collections.abc import Callable

import torch
from torch import nn
from torch._subclasses.fake_tensor import FakeTensor

from . import _lib
from .modules import relabel_modules
from .scaled_mm import _workspace_for

BLOCK = 128

# The C ABI's numbers of the value types.
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_FP8 = {torch.float8_e4m3fn: False, torch.float8_e5m2: True}   # dtype -> e5m2


def _is_e5m2(dtype: torch.dtype) -> bool:
    try:
        return _FP8[dtype]
    except KeyError:
        raise ValueError(f"the fp8 dtype must be torch.float8_e4m3fn or torch.float8_e5m2, got {dtype}") from None


def _type_number(dtype: torch.dtype) -> int:
    try:
        return _TYPES[dtype]
    except KeyError:
        raise ValueError(f"the output dtype must be bfloat16, float16 or float32, got {dtype}") from None


def as_rows(x: torch.Tensor) -> torch.Tensor:
    """x as a matrix of its last dimension's rows, with each row's values side by side (copied only where they are not)."""
    if x.dim() != 2:
        if x.dim() == 0:
            raise ValueError("x must have at least one dimension")
        x = x.reshape(x.numel() // x.shape[-1] if x.shape[-1] else 0, x.shape[-1])
    if not x.is_contiguous() and (x.stride(1) != 1 or x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _plain(x: torch.Tensor) -> torch.Tensor:
    """x out of autograd: the quantized results have no gradients."""
    return x.detach() if x.requires_grad else x


def quantize_blocks(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn, *, square: bool = False,
                    ) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of x `[..., K]` (bfloat16, float16 or float32): one scale for each row and 128 columns, or, with
    `square`, for each 128 x 128 square of a matrix (weights). Not differentiable."""
    e5m2 = _is_e5m2(dtype)
    rows = as_rows(_plain(x))
    if square:
        if x.dim() != 2:
            raise ValueError(f"square blocks need a matrix, got {x.dim()} dimensions")
        if rows.numel() == 0:
            return rows.new_empty(rows.shape, dtype=dtype), rows.new_empty(_square_shape(rows.shape), dtype=torch.float32)
        return torch.ops.feather_ops.quantize_tiles.default(rows, e5m2, True, True, False, False)[:2]
    codes, scale = torch.ops.feather_ops.quantize_blocks.default(rows, e5m2)
    if x.dim() != 2:
        return codes.reshape(x.shape), scale.reshape(*x.shape[:-1], scale.shape[-1])
    return codes, scale


def _square_shape(shape: torch.Size) -> tuple[int, int]:
    return -(-shape[0] // BLOCK), -(-shape[1] // BLOCK)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(M: int, N: int, K: int) -> int:
    return max(0, _lib.c_library().feather_block_scaled_mm_workspace_bytes(M, N, K))


# The arrival counters at a workspace's start, the only part of it that has to be zero.
_COUNTER_BYTES = 64 * 1024


def _workspace(a: torch.Tensor, nbytes: int) -> torch.Tensor:
    """A workspace for a product of a, shared with the other split launches of its stream; in a captured graph or a traced
    program one of its own, whose counters each run clears (all of it, as those launches do, is 33 MB at 512 x 14336 ->
    4096: 62 us a replay against 47)."""
    if isinstance(a, FakeTensor) or (a.is_cuda and torch.cuda.is_current_stream_capturing()):
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=a.device)
        workspace[:_COUNTER_BYTES].zero_()
        return workspace
    return _workspace_for(a, nbytes)


# The C ABI's limit of the stride from row to row.
_FAR_CODES = 1 << 22


def _codes(t: torch.Tensor, name: str) -> torch.Tensor:
    """Codes as the product reads them: rows on 16-byte boundaries, at most _FAR_CODES apart (copied where they are not)."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix, got {t.dim()} dimensions")
    rows, cols = t.shape
    pitch, step = t.stride()
    if (step == 1 or cols <= 1) and t.storage_offset() % 16 == 0 and (
            (pitch % 16 == 0 and cols <= pitch <= _FAR_CODES) or rows <= 1):
        return t
    out = torch.empty_strided((rows, cols), (-(-cols // 64) * 64, 1), dtype=t.dtype, device=t.device)
    return out.copy_(t)


def block_scaled_mm(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                    bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """`(a * a_scale) @ (b * b_scale)^T + bias` for quantized a `[M, K]` and b `[N, K]`: `[M, N]` in out_dtype.

    a_scale is `[M, ceil(K / 128)]`; b_scale `[ceil(N / 128), ceil(K / 128)]` or, one for each row of b,
    `[N, ceil(K / 128)]`. Each operand has its own fp8 format. bias: `[N]` in out_dtype. Sums are fp32 (each block's on the
    matrix cores, then times its scales), the result is rounded once. Codes whose rows do not start on 16-byte boundaries,
    or are over 4 MiB apart, and scales whose rows are over 2**20 apart are copied first: keep weights as `quantize_blocks`
    lays them out. K is at most 2**22. Not differentiable (`block_scaled_linear` is)."""
    out_type = _type_number(out_dtype)
    if torch.compiler.is_compiling():
        return _block_scaled_mm_auto(a, a_scale, b, b_scale, bias, out_type)
    return _product(a, a_scale, b, b_scale, bias, out_type)


def _product(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, bias: torch.Tensor | None,
             out_type: int) -> torch.Tensor:
    a, b = _codes(a, "a"), _codes(b, "b")
    m, k = a.shape
    n = b.shape[0]
    need = _workspace_bytes(int(m), int(n), int(k))   # int: the plan of a traced call fixes its sizes
    return torch.ops.feather_ops.block_scaled_mm.default(a, a_scale, b, b_scale, bias, out_type,
                                                         _workspace(a, need) if need else None)


@functools.lru_cache(maxsize=4096)
def _train_workspace_bytes(M: int, N: int, K: int) -> int:
    """For a layer's product and those of its gradients."""
    return max(_workspace_bytes(M, N, K), _workspace_bytes(M, K, N), _workspace_bytes(N, K, M))


def block_scaled_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                        dtype: torch.dtype = torch.float8_e4m3fn, *,
                        quantized_weight: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
    """`x @ weight^T + bias` in fp8 with a scale for each block of 128: x `[..., K]`, weight `[N, K]`, y `[..., N]` in x's
    dtype (bfloat16, float16 or float32).

    Differentiable once, in reverse mode, in x, weight and bias: the gradients are products of fp8 operands too, each
    quantized along the axis it is summed over (dx and dw are the exact gradients of the product but for that rounding, with
    the quantization itself taken as the identity; dw over at most 2**22 rows of x). Weight and activations are quantized on
    every call; `quantized_weight`, the result of `quantize_blocks(weight, dtype, square=True)`, saves that for a weight that
    does not change. bias is taken in x's dtype."""
    return _checked_linear(x, weight, bias, dtype, quantized_weight, _UNKNOWN)


def _checked_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, dtype: torch.dtype,
                    quantized_weight: tuple[torch.Tensor, torch.Tensor] | None, source: tuple[int, int]) -> torch.Tensor:
    """block_scaled_linear; source: which state of the weight the codes are of (_Source), for a traced program's passes to
    see for themselves."""
    _type_number(x.dtype)
    _is_e5m2(dtype)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None and bias.dtype != x.dtype:
        bias = bias.to(x.dtype)
    if x.numel() == 0 or weight.numel() == 0:
        return nn.functional.linear(x, weight.to(x.dtype), bias)
    trains = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))
    codes, scale = quantized_weight if quantized_weight is not None else (None, None)
    if codes is not None:
        # the backward takes the weight itself, in squares of dtype
        if (codes.shape != weight.shape or codes.dtype != dtype
                or (trains and scale.shape != _square_shape(weight.shape))):
            raise ValueError(f"quantized_weight must be the weight's {tuple(weight.shape)} in squares of {dtype}, got codes "
                             f"{tuple(codes.shape)} {codes.dtype} and scales {tuple(scale.shape)}")
    if torch.compiler.is_compiling():
        return _block_scaled_linear_auto(x, weight, bias, _FP8[dtype], codes, scale, *source)
    return _linear(x, weight, bias, _FP8[dtype], codes, scale, trains)


def _linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, e5m2: bool, codes: torch.Tensor | None,
            scale: torch.Tensor | None, trains: bool) -> torch.Tensor:
    rows, weight = as_rows(x), as_rows(weight)
    if codes is not None:
        codes = _codes(codes, "the weight's codes")
    need = (_train_workspace_bytes if trains else _workspace_bytes)(int(rows.shape[0]), *map(int, weight.shape))
    y = torch.ops.feather_ops.block_scaled_linear.default(rows, weight, bias, e5m2, codes, scale,
                                                          _workspace(rows, need) if need else None)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


# The state of a weight that is not known, or that has none: inference tensors do not count their changes.
_UNKNOWN = (0, -1)


def _state_of(weight: torch.Tensor) -> tuple[int, int]:
    """(address, version) of a weight: one of them is another after every change that torch sees."""
    return 0 if isinstance(weight, FakeTensor) else weight.data_ptr(), -1 if weight.is_inference() else weight._version


class _Source:
    """The weight that codes were taken of, and its state then."""

    def __init__(self, weight: torch.Tensor | None) -> None:
        self.weight = weight   # not a weak reference: torch swaps no tensor that has one
        self.state = _UNKNOWN if weight is None else _state_of(weight)

    def __reduce__(self) -> tuple:   # copied or stored: of no weight
        return _Source, (None,)


class BlockScaledLinear:
    """Mixin for `nn.Linear` (via `relabel_modules`): `forward` is `block_scaled_linear`, 16-bit (or fp32) in and out.

    A frozen weight (`requires_grad` False) is quantized once, by `quantize_weight_` (which `to_block_scaled_linear`
    calls), into two non-persistent buffers, `weight_fp8` and `weight_scale`. A pass that finds the weight changed
    (`load_state_dict`, a step of training, another parameter in its place) quantizes it into them again, so a captured
    graph follows when the layer is next called or `quantize_weight_` is; what a layer that is itself being captured or
    traced finds changed is quantized in that pass alone. Only writes through `weight.data`, which torch does not count,
    and those to a weight made in inference mode need a call of `quantize_weight_`. A weight that takes gradients is
    quantized on every pass. Parameters and `state_dict` stay as they were."""

    def quantize_weight_(self, fp8_dtype: torch.dtype | None = None) -> None:
        """Keep the weight's codes as it is now, in fp8_dtype (None: the format that the layer has, at first e4m3fn)."""
        if fp8_dtype is None:
            fp8_dtype = getattr(self, "_fp8_dtype", torch.float8_e4m3fn)
        codes, scale = quantize_blocks(self.weight, fp8_dtype, square=True)
        kept = self._buffers.get("weight_fp8")
        if (kept is not None and kept.dtype == codes.dtype and kept.shape == codes.shape and kept.device == codes.device
                and (torch.is_inference_mode_enabled() or not kept.is_inference())):
            kept.copy_(codes)   # in place, for graphs that read them
            self.weight_scale.copy_(scale)
        else:
            self.register_buffer("weight_fp8", codes, persistent=False)
            self.register_buffer("weight_scale", scale, persistent=False)
        self._fp8_dtype = fp8_dtype
        self._codes_of = _Source(self.weight)

    def register_parameter(self, name: str, param: nn.Parameter | None) -> None:
        super().register_parameter(name, param)
        if name == "weight":   # another one: what its codes were of is let go
            self._codes_of = _Source(None)

    def _apply(self, fn: Callable[[torch.Tensor], torch.Tensor], recurse: bool = True) -> nn.Module:
        """To another device or type (`to`, `half`, ...), which the weight takes, and codes and scales do not: they are taken
        of the weight as it is then, or (off the GPU, where they wait for the way back) moved."""
        kept = [self._buffers.pop(name, None) for name in ("weight_fp8", "weight_scale")]
        super()._apply(fn, recurse)
        if kept[0] is not None:
            if self.weight.is_cuda:
                self.quantize_weight_()
            else:
                for name, buffer in zip(("weight_fp8", "weight_scale"), kept):
                    self.register_buffer(name, buffer.to(self.weight.device), persistent=False)
                self._codes_of = _Source(None)
        return self

    def quantized_weight(self) -> tuple[torch.Tensor, torch.Tensor] | None:
        """The kept codes and scales of a frozen weight, brought up to date; None where every pass quantizes it. In a program
        that torch.compile traces they are not looked at: the layer's own node does that."""
        return self._kept_codes(self.weight)

    def _kept_codes(self, weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor] | None:
        if weight.requires_grad or self._buffers.get("weight_fp8") is None:
            return None
        source = self._codes_of
        if torch.compiler.is_compiling():
            if source.weight is None or not isinstance(weight, nn.Parameter):
                return None
        elif source.weight is not weight or source.state != _state_of(weight):
            if (not isinstance(weight, nn.Parameter) or torch._C._len_torch_dispatch_stack()
                    or (weight.is_cuda and torch.cuda.is_current_stream_capturing())):
                return None
            self.quantize_weight_()
        return self._buffers["weight_fp8"], self._buffers["weight_scale"]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        weight = self.weight
        codes = self._kept_codes(weight)
        return _checked_linear(x, weight, self.bias, self.__dict__.get("_fp8_dtype", torch.float8_e4m3fn), codes,
                               _UNKNOWN if codes is None else self._codes_of.state)


def to_block_scaled_linear(root: nn.Module, fp8_dtype: torch.dtype = torch.float8_e4m3fn,
                           accept: Callable[[nn.Module], bool] | None = None) -> int:
    """Relabel the `nn.Linear` modules under `root` (those `accept` approves, by default every one) as
    `BlockScaledLinear`, quantize the frozen ones' weights and return how many changed."""
    _is_e5m2(fp8_dtype)
    count = relabel_modules(root, BlockScaledLinear, accept or (lambda module: isinstance(module, nn.Linear)))
    for module in root.modules():
        if isinstance(module, BlockScaledLinear) and not hasattr(module, "_fp8_dtype"):
            module._fp8_dtype = fp8_dtype
            if not module.weight.requires_grad:
                module.quantize_weight_(fp8_dtype)
    return count


# ---- one node each under torch.compile ----


@torch.library.custom_op("feather_ops::block_scaled_mm_auto", mutates_args=())
def _block_scaled_mm_auto(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                          bias: torch.Tensor | None, out_type: int) -> torch.Tensor:
    """block_scaled_mm as one opaque op: neither the copies of what lies off the kernels' boundaries nor the workspace are
    traced."""
    return _product(a, a_scale, b, b_scale, bias, out_type)


@_block_scaled_mm_auto.register_fake
def _(a, a_scale, b, b_scale, bias, out_type):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=_DTYPE_OF[out_type])


@torch.library.custom_op("feather_ops::block_scaled_linear_auto", mutates_args=())
def _block_scaled_linear_auto(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, e5m2: bool,
                              codes: torch.Tensor | None, scale: torch.Tensor | None, address: int,
                              version: int) -> torch.Tensor:
    """block_scaled_linear as one opaque op. The weight's codes are taken if it is as they were taken of it, as far as that is
    known."""
    if codes is not None and (address, version) != _UNKNOWN and (address, version) != _state_of(weight):
        codes = scale = None
    return _linear(x, weight, bias, e5m2, codes, scale, False)


@_block_scaled_linear_auto.register_fake
def _(x, weight, bias, e5m2, codes, scale, address, version):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op("feather_ops::block_scaled_linear_auto_backward", mutates_args=())
def _block_scaled_linear_auto_backward(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, e5m2: bool, need_x: bool,
                                       need_weight: bool, need_bias: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of x, weight and bias, each empty where it is not asked for. x and the weight are kept as they are and
    quantized again: what the program's other nodes hold of them anyway."""
    ops = torch.ops.feather_ops
    gy, rows, weight = as_rows(grad), as_rows(x), as_rows(weight)
    m, (n, k) = gy.shape[0], weight.shape
    need = _train_workspace_bytes(m, n, k)
    workspace = _workspace(gy, need) if need else None
    grad_x, grad_weight, grad_bias = (t.new_empty(0) for t in (x, weight, x))
    codes, scale, codes_t, scale_t, sums = ops.quantize_tiles.default(gy, e5m2, False, need_x, need_weight, need_bias)
    if need_x:
        _, _, w, w_scale, _ = ops.quantize_tiles.default(weight, e5m2, True, False, True, False)
        grad_x = ops.block_scaled_mm.default(codes, scale, w, w_scale, None, _TYPES[x.dtype], workspace).reshape(x.shape)
    if need_weight:
        _, _, xt, xt_scale, _ = ops.quantize_tiles.default(rows, e5m2, False, False, True, False)
        grad_weight = ops.block_scaled_mm.default(codes_t, scale_t, xt, xt_scale, None, _TYPES[weight.dtype], workspace)
    if need_bias:
        grad_bias = ops.sum_rows.default(sums, _TYPES[x.dtype])
    return grad_x, grad_weight, grad_bias


@_block_scaled_linear_auto_backward.register_fake
def _(grad, x, weight, e5m2, need_x, need_weight, need_bias):
    return (x.new_empty(x.shape if need_x else (0,)), weight.new_empty(weight.shape if need_weight else (0,)),
            x.new_empty((weight.shape[0],) if need_bias else (0,)))


def _linear_auto_context(ctx, inputs, output) -> None:
    x, weight, bias, ctx.e5m2, *_ = inputs
    ctx.save_for_backward(x, weight)


def _linear_auto_backward(ctx, grad: torch.Tensor) -> tuple:
    x, weight = ctx.saved_tensors
    needs = ctx.needs_input_grad[:3]
    grads = _block_scaled_linear_auto_backward(grad, x, weight, ctx.e5m2, *needs)
    return (*(g if need else None for g, need in zip(grads, needs)), None, None, None, None, None)


_block_scaled_linear_auto.register_autograd(_linear_auto_backward, setup_context=_linear_auto_context)


# ---- shapes, for tracing ----


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _fake_codes(x: torch.Tensor, rows: int, cols: int, scale_rows: int, e5m2: bool) -> tuple[torch.Tensor, torch.Tensor]:
    dtype = torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn
    codes = torch.empty_strided((rows, cols), ((cols + 63) // 64 * 64, 1), dtype=dtype, device=x.device)
    scale = torch.empty_strided((scale_rows, _blocks(cols)), (1, scale_rows), dtype=torch.float32, device=x.device)
    return codes, scale


_DTYPE_OF = {number: dtype for dtype, number in _TYPES.items()}


@torch.library.register_fake("feather_ops::block_scaled_mm")
def _(a, a_scale, b, b_scale, bias, out_type, workspace):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=_DTYPE_OF[out_type])


@torch.library.register_fake("feather_ops::quantize_blocks")
def _(x, e5m2):
    return _fake_codes(x, x.shape[0], x.shape[1], x.shape[0], e5m2)


@torch.library.register_fake("feather_ops::quantize_tiles")
def _(x, e5m2, square, plain, transposed, sums):
    m, n = x.shape
    codes, scale = _fake_codes(x, m, n, _blocks(m) if square else m, e5m2) if plain else _fake_codes(x, 0, 0, 0, e5m2)
    codes_t, scale_t = (_fake_codes(x, n, m, _blocks(n) if square else n, e5m2) if transposed
                        else _fake_codes(x, 0, 0, 0, e5m2))
    return codes, scale, codes_t, scale_t, x.new_empty((_blocks(m), n) if sums else (0, 0), dtype=torch.float32)


@torch.library.register_fake("feather_ops::sum_rows")
def _(part, out_type):
    return part.new_empty(part.shape[1], dtype=_DTYPE_OF[out_type])
