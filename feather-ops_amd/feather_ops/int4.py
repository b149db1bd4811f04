"""Products with 4-bit weights that have one scale for each group of columns, their quantization, and the layers on them; not in
the reference, whose weights have 8 bits. Kernels: `csrc/linear_few.h` (few rows), `csrc/int4_tile.h`, `csrc/linear_tile.h`,
`csrc/int4.hip`; autograd node: `csrc/linear_autograd.cpp`. C ABI: `include/feather_linear_ops.h`.

A quantized weight is `(codes, scale, zero)`: value (n, k) is `(q - zero) * scale` with the code q, 0 .. 15, and the scale and zero
point of its group of 32, 64 or 128 columns.

- codes: uint8 `[N, ceil(K / 2)]`, two columns to a byte, the even one in the low half;
- scale: `[N, ceil(K / group)]` in the activations' dtype, best stored group by group (`scale.t()` is contiguous);
- zero: uint8 like scale, 0 .. 15; or None: 8.
"""

import functools
from collections.abc import Callable

import torch
from torch import nn

from . import _lib
from .block_scaled import _UNKNOWN, _Source, _plain, _state_of, _workspace, as_rows
from .gate import silu_mul
from .gated import HALVES, _workspace_bytes as _gated_workspace_bytes, activate, activation_number, check_depth, operand
from .modules import relabel_modules

GROUPS = (32, 64, 128)
Int4Weight = tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]


def quantize_int4(weight: torch.Tensor, group: int = 128, *, zeros: bool = False) -> Int4Weight:
    """(codes, scale, zero) of a bfloat16 or float16 weight `[N, K]`. A group's scale is its largest magnitude / 7 (zero is then
    None) or, with `zeros`, its range (extended to 0) / 15, rounded to the weight's dtype; codes are the nearest. Not
    differentiable."""
    if weight.dim() != 2 or weight.dtype not in HALVES:
        raise ValueError(f"weight must be a bfloat16 or float16 matrix, got {tuple(weight.shape)} {weight.dtype}")
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    n, k = weight.shape
    w = as_rows(_plain(weight))
    if w.numel() == 0:
        shape = (n, -(-k // group))
        return (w.new_empty((n, -(-k // 2)), dtype=torch.uint8), w.new_empty(shape),
                w.new_empty(shape, dtype=torch.uint8) if zeros else None)
    codes, scale, zero = torch.ops.feather_ops.int4_quantize.default(w, group, zeros)
    return codes[:, : -(-k // 2)], scale[:, :n].t(), zero[:, :n].t() if zeros else None


@functools.lru_cache(maxsize=4096)
def _group_of(k: int, groups: int) -> int:
    for group in GROUPS:
        if -(-k // group) == groups:
            return group
    raise ValueError(f"scale must have one column for each group of 32, 64 or 128 columns of {k}, got {groups}")


def _grouped(t: torch.Tensor) -> torch.Tensor:
    """[N, groups] stored group by group, with memory for 4 values to a group at least (copied where it is not)."""
    n, groups = t.shape
    first, step = t.stride()
    if (n <= 1 or first == 1) and (max(n, step) if groups <= 1 else step) >= max(n, 4):
        end = (groups - 1) * step + 4
        if n >= 4 or (t.storage_offset() + end) * t.element_size() <= t.untyped_storage().nbytes():
            return t
    out = t.new_empty((groups, -(-n // 4) * 4))[:, :n].t()
    return out.copy_(t)


def _whole_bytes(codes: torch.Tensor) -> torch.Tensor:
    """Codes with rows on 4-byte boundaries that can be read to the next one (copied where they cannot)."""
    n, cols = codes.shape
    pitch, step = codes.stride()
    whole = -(-cols // 4) * 4
    if (step == 1 or cols <= 1) and codes.storage_offset() % 4 == 0 and ((pitch % 4 == 0 and whole <= pitch <= 1 << 22) or n <= 1):
        end = codes.storage_offset() + (n - 1) * pitch + whole
        if whole == cols or end <= codes.untyped_storage().nbytes():
            return codes
    out = codes.new_empty((n, -(-cols // 16) * 16))[:, :cols]
    return out.copy_(codes)


def _check(codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, k: int) -> None:
    size, groups = codes.shape, scale.shape
    if codes.dtype != torch.uint8 or len(size) != 2 or size[1] != -(-k // 2):
        raise ValueError(f"codes must be uint8 [N, {-(-k // 2)}], two columns to a byte, got {tuple(size)} {codes.dtype}")
    if len(groups) != 2 or groups[0] != size[0] or not scale.dtype.is_floating_point:
        raise ValueError(f"scale must be [{size[0]}, groups], got {tuple(groups)} {scale.dtype}")
    _group_of(int(k), int(groups[1]))   # int: the plan of a traced call fixes its sizes
    if scale.requires_grad:
        raise ValueError("a quantized weight takes no gradients")
    if zero is not None:
        if zero.dtype != torch.uint8 or zero.shape != groups:
            raise ValueError(f"zero must be uint8 {tuple(groups)}, got {tuple(zero.shape)} {zero.dtype}")


def _laid_out(codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, dtype: torch.dtype) -> Int4Weight:
    """A weight as the kernels read it, with scales in `dtype`: itself where it is."""
    return _whole_bytes(codes), _grouped(scale.to(dtype)), None if zero is None else _grouped(zero)


def dequantize_int4(codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None,
                    k: int | None = None) -> torch.Tensor:
    """The weight `[N, K]` that codes stand for, in scale's dtype (bfloat16 or float16), each value rounded once. k: the columns,
    where they are odd (None: twice the bytes of a row). Not differentiable."""
    if codes.dim() != 2:
        raise ValueError(f"codes must be a matrix, got {codes.dim()} dimensions")
    k = 2 * codes.shape[1] if k is None else k
    if scale.dtype not in HALVES:
        raise ValueError(f"scale must be bfloat16 or float16, got {scale.dtype}")
    if codes.shape[0] == 0 or k == 0:
        return scale.new_empty((codes.shape[0], k))
    scale = _plain(scale)
    _check(codes, scale, zero, k)
    return torch.ops.feather_ops.int4_dequantize.default(*_laid_out(codes, scale, zero, scale.dtype), k)[:, :k]


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(M: int, rows: int, K: int, gated: bool, trains: bool) -> int:
    lib = _lib.c_library()
    n, k8 = rows // 2 if gated else rows, -(-K // 8) * 8
    need = [lib.feather_int4_linear_workspace_bytes(M, n, K, gated)]
    if M > 64:   # some go through the product in 16 bits, by their sizes and the codes' alignment
        need.append(_gated_workspace_bytes(M, n, k8, False, False) if gated else lib.feather_product_workspace_bytes(M, n, k8))
    if trains:
        need.append(lib.feather_product_workspace_bytes(M, K, rows))
    if min(need) < 0:
        raise ValueError(f"sizes are out of range: x [{M}, {K}], weight [{rows}, {K}]")
    return max(need)


def _prepared(x: torch.Tensor, codes: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor | None:
    """Checks of x and bias; the bias as the kernels take it."""
    if x.dtype not in HALVES:
        raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    if bias is None:
        return None
    if bias.shape != codes.shape[:1]:
        raise ValueError(f"bias must have {codes.shape[0]} values, got {tuple(bias.shape)}")
    return bias.to(x.dtype).contiguous()


def int4_linear(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """`x @ W^T + bias` with a 4-bit weight W `[N, K]`: x `[..., K]`, the result `[..., N]`, both bfloat16 or float16; bias `[N]`.

    Up to 64 rows take the codes as they are, each group's sum times its scale in fp32. Of more rows most take W rounded to x's dtype
    (15 times a scale has to be within its range), and some, such as a batch's last ones, the codes: by the sizes alone. The
    result is rounded once. Differentiable once, in reverse mode, in x and bias (the weight is frozen): dx = dy @ W with W rounded
    to x's dtype. Scales in another dtype than x's, scales and zero points that are not stored group by group, codes whose rows do
    not start on 4-byte boundaries, and rows of x off 16-byte boundaries or of no multiple of 8 values are copied on every call.
    K is at most 2**21, and so is N where x takes a gradient."""
    return _checked_linear(x, codes, scale, zero, bias, None, _UNKNOWN)


def _checked_linear(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, bias: torch.Tensor | None,
                    weight: torch.Tensor | None, source: tuple[int, int]) -> torch.Tensor:
    """int4_linear; weight and source: what the codes were taken of, and its state then (_Source), for a traced program's passes to
    see for themselves."""
    bias = _prepared(x, codes, bias)
    k = x.shape[-1]
    _check(codes, scale, zero, k)
    if x.numel() == 0 or codes.numel() == 0:
        return nn.functional.linear(x, x.new_zeros((codes.shape[0], k)), bias)
    if x.requires_grad and torch.is_grad_enabled():
        check_depth("x", codes.shape[0], "the weight's rows")
    if torch.compiler.is_compiling():
        return _int4_linear_auto(x, codes, scale, zero, bias, weight, *source)
    return _linear(x, codes, scale, zero, bias)


def _linear(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None,
            bias: torch.Tensor | None) -> torch.Tensor:
    trains = x.requires_grad and torch.is_grad_enabled()
    k = x.shape[-1]
    rows = operand(as_rows(x))
    codes, scale, zero = _laid_out(codes, scale, zero, x.dtype)
    need = _workspace_bytes(int(rows.shape[0]), int(codes.shape[0]), int(k), False, trains)
    y = torch.ops.feather_ops.int4_linear.default(rows, codes, scale, zero, bias, k, _workspace(rows, need) if need else None)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


def int4_gated_linear(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None,
                      bias: torch.Tensor | None = None, activation: str = "silu") -> torch.Tensor:
    """`gated_linear` with a 4-bit weight of 2 F rows, the gates' first: x `[..., K]`, the result `[..., F]`, in one launch up to 64
    rows. Where x or bias takes gradients it is `int4_linear` and the activation of its outputs, in x's dtype: both sums are rounded
    before the activation, so a pass that records gradients and one that does not differ by that."""
    act = activation_number(activation)
    bias = _prepared(x, codes, bias)
    if codes.dim() != 2 or codes.shape[0] % 2:
        raise ValueError(f"codes must have an even number of rows, the gates' and the others', got {tuple(codes.shape)}")
    trains = torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad))
    if x.numel() == 0 or codes.numel() == 0 or trains:
        h = int4_linear(x, codes, scale, zero, bias)
        if act == 0:
            return silu_mul(h)
        gate, up = h.chunk(2, -1)
        return activate(gate, act) * up
    _check(codes, scale, zero, x.shape[-1])
    if torch.compiler.is_compiling():
        return _int4_gated_auto(x, codes, scale, zero, bias, act)
    return _gated(x, codes, scale, zero, bias, act)


def _gated(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, bias: torch.Tensor | None,
           act: int) -> torch.Tensor:
    k = x.shape[-1]
    rows = operand(as_rows(_plain(x)))
    codes, scale, zero = _laid_out(codes, scale, zero, x.dtype)
    need = _workspace_bytes(int(rows.shape[0]), int(codes.shape[0]), int(k), True, False)
    y = torch.ops.feather_ops.int4_forward.default(rows, codes, scale, zero, bias, k, True, act,
                                                   _workspace(rows, need) if need else None)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


# A state that no weight has: codes of another one.
_STALE = (-1, -1)


class Int4Linear:
    """Mixin for `nn.Linear` (via `relabel_modules`): `forward` is `int4_linear`, 16-bit in and out. The weight is frozen; gradients
    reach the input and the bias, so the layer can sit under trainable adapters.

    The weight is quantized by `quantize_weight_` (which `to_int4_linear` calls) into three non-persistent buffers, `weight_int4`,
    `weight_scale` and `weight_zero`. A pass that finds the weight changed (`load_state_dict`, another parameter in its place, another
    type) quantizes it into them again, so a captured graph follows when the layer is next called or `quantize_weight_` is; what a layer
    that is itself being captured or traced finds changed is quantized in that pass alone. Only writes through `weight.data`, which
    torch does not count, and those to a weight made in inference mode need a call of `quantize_weight_`. A weight that was let go
    (None, or of another shape) or moved to another device leaves the codes as they are. Parameters and `state_dict` stay as they
    were."""

    def quantize_weight_(self, group: int | None = None, zeros: bool | None = None) -> None:
        """Quantize the weight as it is now, in groups of `group` columns, with zero points or without (None: as the layer has them, at
        first 128 and without)."""
        before = self.__dict__.get("_int4_format", (128, False, None))
        group = before[0] if group is None else group
        zeros = before[1] if zeros is None else zeros
        dtype = self.weight.dtype if self.weight.dtype in HALVES else before[2]   # fp32: in the type that it had
        fresh = quantize_int4(self.weight if dtype is None else self.weight.to(dtype), group, zeros=zeros)
        kept = [self._buffers.get(name) for name in _BUFFERS]
        if all((old is None) == (new is None) and (old is None or _can_hold(old, new)) for old, new in zip(kept, fresh)):
            for old, new in zip(kept, fresh):   # in place, for graphs that read them
                if old is not None:
                    old.copy_(new)
        else:
            for name, new in zip(_BUFFERS, fresh):
                self.register_buffer(name, new, persistent=False)
        self._int4_format = (group, zeros, dtype)
        self._codes_of = _Source(self.weight)

    def register_parameter(self, name: str, param: nn.Parameter | None) -> None:
        super().register_parameter(name, param)
        if name == "weight":   # another one: what its codes were of is let go
            self._codes_of = _Source(None)

    def _apply(self, fn: Callable[[torch.Tensor], torch.Tensor], recurse: bool = True) -> nn.Module:
        """To another device or type (`to`, `half`, ...), which the weight takes. Codes, scales and zero points move with it to a
        device, and are taken of the weight as it is then on the GPU."""
        kept = [(name, self._buffers.pop(name)) for name in _BUFFERS if name in self._buffers]
        super()._apply(fn, recurse)
        if kept:
            device = fn(kept[0][1]).device
            for name, buffer in kept:
                if buffer is not None and buffer.device != device:
                    buffer = torch.empty_like(buffer, device=device) if buffer.is_meta else buffer.to(device)
                self.register_buffer(name, buffer, persistent=False)
            if self.weight is not None and not self._is_current(self.weight):
                self._codes_of = _Source(None)   # a later weight may lie where this one did
                if self._takes(self.weight) and self.weight.is_cuda:
                    self.quantize_weight_()
        return self

    def _takes(self, weight: torch.Tensor | None) -> bool:
        """Whether codes are to follow a weight: one of their shape and on their device."""
        codes = self._buffers["weight_int4"]
        return (weight is not None and weight.dim() == 2 and weight.shape[0] == codes.shape[0]
                and (weight.shape[1] + 1) // 2 == codes.shape[1] and weight.device == codes.device)

    def _is_current(self, weight: torch.Tensor | None) -> bool:
        source = self.__dict__.get("_codes_of")
        return source is not None and weight is not None and source.weight is weight and source.state == _state_of(weight)

    def quantized_weight(self) -> Int4Weight:
        """The codes, scales and zero points, brought up to date. In a program that torch.compile traces they are taken as they are: the
        layer's own node looks at them."""
        weight, buffers = self.weight, self._buffers
        kept = buffers["weight_int4"], buffers["weight_scale"], buffers["weight_zero"]
        if torch.compiler.is_compiling() or self._is_current(weight) or not self._takes(weight):
            return kept
        if (not isinstance(weight, nn.Parameter) or torch._C._len_torch_dispatch_stack()
                or (weight.is_cuda and torch.cuda.is_current_stream_capturing())):
            return _requantized(weight, *kept)
        self.quantize_weight_()
        return tuple(self._buffers[name] for name in _BUFFERS)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        codes, scale, zero = self.quantized_weight()
        if not torch.compiler.is_compiling() or not self._takes(self.weight):
            return int4_linear(x, codes, scale, zero, self.bias)
        weight, source = self.weight, getattr(self, "_codes_of", None)
        known = source is not None and source.weight is not None and isinstance(weight, nn.Parameter)
        return _checked_linear(x, codes, scale, zero, self.bias, _plain(weight), source.state if known else _STALE)


_BUFFERS = ("weight_int4", "weight_scale", "weight_zero")


def _can_hold(kept: torch.Tensor, new: torch.Tensor) -> bool:
    return (kept.dtype == new.dtype and kept.shape == new.shape and kept.stride() == new.stride() and kept.device == new.device
            and (torch.is_inference_mode_enabled() or not kept.is_inference()))


def _requantized(weight: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None) -> Int4Weight:
    """A weight in 4 bits as another one is."""
    if weight.dtype not in HALVES:
        weight = weight.to(scale.dtype)
    return quantize_int4(weight, _group_of(weight.shape[1], scale.shape[1]), zeros=zero is not None)


def to_int4_linear(root: nn.Module, group: int = 128, zeros: bool = False,
                   accept: Callable[[nn.Module], bool] | None = None) -> int:
    """Relabel the `nn.Linear` modules under `root` (those `accept` approves, by default every one with a bfloat16 or float16
    weight) as `Int4Linear`, quantize their weights and return how many changed."""
    def default_accept(module: nn.Module) -> bool:
        return isinstance(module, nn.Linear) and module.weight.dtype in HALVES

    count = relabel_modules(root, Int4Linear, accept or default_accept)
    for module in root.modules():
        if isinstance(module, Int4Linear) and not hasattr(module, "weight_int4"):
            module.quantize_weight_(group, zeros)
    return count


# ---- one node each under torch.compile ----


def _codes_now(weight: torch.Tensor | None, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, address: int,
               version: int) -> Int4Weight:
    """Codes if the weight is as it was when they were taken of it, as far as that is known, and else its own."""
    if weight is None or (address, version) in (_UNKNOWN, _state_of(weight)):
        return codes, scale, zero
    return _requantized(weight, codes, scale, zero)


@torch.library.custom_op("feather_ops::int4_linear_auto", mutates_args=())
def _int4_linear_auto(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None,
                      bias: torch.Tensor | None, weight: torch.Tensor | None = None, address: int = 0,
                      version: int = -1) -> torch.Tensor:
    """int4_linear as one opaque op."""
    return _linear(x, *_codes_now(weight, codes, scale, zero, address, version), bias)


@_int4_linear_auto.register_fake
def _(x, codes, scale, zero, bias, weight=None, address=0, version=-1):
    return x.new_empty((*x.shape[:-1], codes.shape[0]))


@torch.library.custom_op("feather_ops::int4_linear_auto_backward", mutates_args=())
def _int4_linear_auto_backward(grad: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None,
                               k: int, weight: torch.Tensor | None = None, address: int = 0, version: int = -1) -> torch.Tensor:
    codes, scale, zero = _codes_now(weight, codes, scale, zero, address, version)
    rows = operand(as_rows(grad))
    codes, scale, zero = _laid_out(codes, scale, zero, grad.dtype)
    need = max(0, _lib.c_library().feather_product_workspace_bytes(rows.shape[0], k, codes.shape[0]))
    dx = torch.ops.feather_ops.int4_backward.default(rows, codes, scale, zero, k, _workspace(rows, need) if need else None)
    return dx.reshape(*grad.shape[:-1], k)


@_int4_linear_auto_backward.register_fake
def _(grad, codes, scale, zero, k, weight=None, address=0, version=-1):
    return grad.new_empty((*grad.shape[:-1], k))


def _linear_auto_context(ctx, inputs, output) -> None:
    x, codes, scale, zero, _, weight, *ctx.source = inputs
    ctx.save_for_backward(codes, scale, zero, weight)
    ctx.k = x.shape[-1]


def _linear_auto_backward(ctx, grad: torch.Tensor) -> tuple:
    need_x, need_bias = ctx.needs_input_grad[0], ctx.needs_input_grad[4]
    dx = db = None
    if need_x:
        codes, scale, zero, weight = ctx.saved_tensors
        dx = _int4_linear_auto_backward(grad, codes, scale, zero, ctx.k, weight, *ctx.source)
    if need_bias:
        db = grad.reshape(-1, grad.shape[-1]).float().sum(0).to(grad.dtype)
    return dx, None, None, None, db, None, None, None


_int4_linear_auto.register_autograd(_linear_auto_backward, setup_context=_linear_auto_context)


@torch.library.custom_op("feather_ops::int4_gated_auto", mutates_args=())
def _int4_gated_auto(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None,
                     bias: torch.Tensor | None, act: int) -> torch.Tensor:
    """int4_gated_linear as one opaque op."""
    return _gated(x, codes, scale, zero, bias, act)


@_int4_gated_auto.register_fake
def _(x, codes, scale, zero, bias, act):
    return x.new_empty((*x.shape[:-1], codes.shape[0] // 2))


# ---- shapes, for tracing ----


@torch.library.register_fake("feather_ops::int4_forward")
def _(x, codes, scale, zero, bias, k, gated, activation, workspace):
    return x.new_empty((x.shape[0], codes.shape[0] // 2 if gated else codes.shape[0]))


@torch.library.register_fake("feather_ops::int4_backward")
def _(grad_y, codes, scale, zero, k, workspace):
    return grad_y.new_empty((grad_y.shape[0], k))


@torch.library.register_fake("feather_ops::int4_quantize")
def _(weight, group, zeros):
    n, k = weight.shape
    ld, groups = (n + 3) // 4 * 4, (k + group - 1) // group
    return (weight.new_empty((n, ((k + 1) // 2 + 15) // 16 * 16), dtype=torch.uint8), weight.new_empty((groups, ld)),
            weight.new_empty((groups, ld) if zeros else (0, 0), dtype=torch.uint8))


@torch.library.register_fake("feather_ops::int4_dequantize")
def _(codes, scale, zero, k):
    return scale.new_empty((codes.shape[0], (k + 7) // 8 * 8))
