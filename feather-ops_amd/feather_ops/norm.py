"""Root-mean-square norm with the residual's addition, in 16 bits, fp32 or fp8 with a scale for each block of 128; not in
the reference. Kernels: `csrc/rms_norm.hip`; autograd node: `csrc/block_autograd.cpp`.

    h = x + residual (in x's dtype)    y = h / sqrt(mean(h^2) + eps) * weight

The norm is of h as it is stored: the sum is rounded to the stream's dtype, which the next layer and the backward read,
and everything after it is fp32 until y is rounded once.
"""

import torch

from .block_scaled import _TYPES, _fake_codes, _is_e5m2, _plain, as_rows


def _checked(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None) -> None:
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must be a vector of x's last dimension, got {tuple(weight.shape)} for {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have x's shape and dtype, got {tuple(residual.shape)} {residual.dtype} for "
                         f"{tuple(x.shape)} {x.dtype}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
             eps: float = 1e-6) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """y in x's dtype, or (y, h) with a residual; x `[..., D]` in bfloat16, float16 or float32, weight `[D]` in x's dtype
    or float32. Differentiable once, in reverse mode, in x, weight and residual, through y and h."""
    _checked(x, weight, residual)
    if x.numel() == 0:
        h = x if residual is None else x + residual
        y = (h * weight).to(x.dtype)
        return y if residual is None else (y, h)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    y, h, _ = torch.ops.feather_ops.rms_norm.default(as_rows(x), weight,
                                                     None if residual is None else as_rows(residual), eps, False)
    if x.dim() != 2:   # a view costs a few microseconds of host time, with small tensors as much as a kernel
        y = y.reshape(x.shape)
        h = h if residual is None else h.reshape(x.shape)
    return y if residual is None else (y, h)


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                       dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, ...]:
    """`rms_norm` with y quantized as `quantize_blocks` does, from its unrounded values: (codes, scale), or
    (codes, scale, h) with a residual. What `block_scaled_mm` takes. Not differentiable."""
    _checked(x, weight, residual)
    e5m2 = _is_e5m2(dtype)
    x, weight = _plain(x), _plain(weight)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    residual = None if residual is None else _plain(residual)
    if x.numel() == 0:
        h = x if residual is None else x + residual
        out = (x.new_empty(x.shape, dtype=dtype), x.new_empty((*x.shape[:-1], -(-x.shape[-1] // 128)), dtype=torch.float32))
        return out if residual is None else (*out, h)
    codes, scale, h = torch.ops.feather_ops.rms_norm_quantized.default(
        as_rows(x), weight, None if residual is None else as_rows(residual), eps, e5m2)
    if x.dim() != 2:
        codes, scale = codes.reshape(x.shape), scale.reshape(*x.shape[:-1], scale.shape[-1])
        h = h if residual is None else h.reshape(x.shape)
    return (codes, scale) if residual is None else (codes, scale, h)


@torch.library.register_fake("feather_ops::rms_norm")
def _(x, weight, residual, eps, need_rstd):
    return (x.new_empty(x.shape), x.new_empty(x.shape if residual is not None else (0, 0)),
            x.new_empty(x.shape[0] if need_rstd else 0, dtype=torch.float32))


@torch.library.register_fake("feather_ops::rms_norm_quantized")
def _(x, weight, residual, eps, e5m2):
    return (*_fake_codes(x, x.shape[0], x.shape[1], x.shape[0], e5m2),
            x.new_empty(x.shape if residual is not None else (0, 0)))


@torch.library.register_fake("feather_ops::rms_norm_backward")
def _(grad_y, grad_h, h, weight, rstd, need_weight):
    return h.new_empty(h.shape), weight.new_empty(h.shape[1] if need_weight else 0)
