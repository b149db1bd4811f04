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
    """A workspace for a product of a, shared with the other split launches of its stream; in a captured graph one of its
    own, whose counters each replay clears (all of it, as those launches do, is 33 MB at 512 x 14336 -> 4096: 62 us a replay
    against 47)."""
    if a.is_cuda and not isinstance(a, FakeTensor) and torch.cuda.is_current_stream_capturing():
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=a.device)
        workspace[:_COUNTER_BYTES].zero_()
        return workspace
    return _workspace_for(a, nbytes)


# The C ABI's limits of the strides from row to row (from square to square).
_FAR_CODES = 1 << 22
_FAR_SCALES = 1 << 20


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


def _scales(t: torch.Tensor) -> torch.Tensor:
    """Scales as the product reads them: rows at most _FAR_SCALES apart (copied where they are not)."""
    if t.dim() != 2 or t.shape[0] <= 1 or t.stride(0) <= _FAR_SCALES:
        return t
    return torch.empty_strided(t.shape, (1, t.shape[0]), dtype=t.dtype, device=t.device).copy_(t)


def block_scaled_mm(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                    bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """`(a * a_scale) @ (b * b_scale)^T + bias` for quantized a `[M, K]` and b `[N, K]`: `[M, N]` in out_dtype.

    a_scale is `[M, ceil(K / 128)]`; b_scale `[ceil(N / 128), ceil(K / 128)]` or, one for each row of b,
    `[N, ceil(K / 128)]`. Each operand has its own fp8 format. bias: `[N]` in out_dtype. Sums are fp32 (each block's on the
    matrix cores, then times its scales), the result is rounded once. Codes whose rows do not start on 16-byte boundaries,
    or are over 4 MiB apart, and scales whose rows are over 2**20 apart are copied first: keep weights as `quantize_blocks`
    lays them out. K is at most 2**22. Not differentiable (`block_scaled_linear` is)."""
    out_type = _type_number(out_dtype)
    a, b, a_scale, b_scale = _codes(a, "a"), _codes(b, "b"), _scales(a_scale), _scales(b_scale)
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

    Differentiable once, in reverse mode, in x, weight and bias: the gradients are products of fp8 operands too, each quantized along the axis it
    is summed over (dx and dw are the exact gradients of the product but for that rounding, with the quantization itself
    taken as the identity). Weight and activations are quantized on every call; `quantized_weight`, the result of
    `quantize_blocks(weight, dtype, square=True)`, saves that for a weight that does not change. bias is taken in x's
    dtype."""
    _type_number(x.dtype)
    _is_e5m2(dtype)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None and bias.dtype != x.dtype:
        bias = bias.to(x.dtype)
    if x.numel() == 0 or weight.numel() == 0:
        return nn.functional.linear(x, weight.to(x.dtype), bias)
    rows, weight = as_rows(x), as_rows(weight)
    trains = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))
    codes, scale = quantized_weight if quantized_weight is not None else (None, None)
    if codes is not None:
        # the backward takes the weight itself, in squares of dtype
        if (codes.shape != weight.shape or codes.dtype != dtype
                or (trains and scale.shape != _square_shape(weight.shape))):
            raise ValueError(f"quantized_weight must be the weight's {tuple(weight.shape)} in squares of {dtype}, got codes "
                             f"{tuple(codes.shape)} {codes.dtype} and scales {tuple(scale.shape)}")
        codes, scale = _codes(codes, "the weight's codes"), _scales(scale)
    need = (_train_workspace_bytes if trains else _workspace_bytes)(int(rows.shape[0]), *map(int, weight.shape))
    y = torch.ops.feather_ops.block_scaled_linear.default(rows, weight, bias, _FP8[dtype], codes, scale,
                                                          _workspace(rows, need) if need else None)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


class _Source:
    """The weight that codes were taken of, and its state then."""

    __slots__ = ("weight", "address", "version")

    def __init__(self, weight: torch.Tensor | None) -> None:
        self.weight = weight   # not a weak reference: torch swaps no tensor that has one
        self.address, self.version = (None, None) if weight is None else self._state(weight)

    @staticmethod
    def _state(weight: torch.Tensor) -> tuple[int, int | None]:
        address = 0 if isinstance(weight, FakeTensor) else weight.data_ptr()
        return address, None if weight.is_inference() else weight._version   # inference tensors do not count their changes

    def is_still(self, weight: torch.Tensor) -> bool:
        return self.weight is weight and (self.address, self.version) == self._state(weight)

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

    def quantize_weight_(self, fp8_dtype: torch.dtype = torch.float8_e4m3fn) -> None:
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
                self.quantize_weight_(self._fp8_dtype)
            else:
                for name, buffer in zip(("weight_fp8", "weight_scale"), kept):
                    self.register_buffer(name, buffer.to(self.weight.device), persistent=False)
                self._codes_of = _Source(None)
        return self

    def quantized_weight(self) -> tuple[torch.Tensor, torch.Tensor] | None:
        """The kept codes and scales of a frozen weight, brought up to date; None where every pass quantizes it."""
        weight = self.weight
        if weight.requires_grad or "weight_fp8" not in self._buffers:
            return None
        if not torch.compiler.is_compiling() and not self._codes_of.is_still(weight):
            if (not isinstance(weight, nn.Parameter) or torch._C._len_torch_dispatch_stack()
                    or (weight.is_cuda and torch.cuda.is_current_stream_capturing())):
                return None
            self.quantize_weight_(self._fp8_dtype)
        return self.weight_fp8, self.weight_scale

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return block_scaled_linear(x, self.weight, self.bias, getattr(self, "_fp8_dtype", torch.float8_e4m3fn),
                                   quantized_weight=self.quantized_weight())


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
