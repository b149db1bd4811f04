"""Gated activation `silu(gate) * up`, in 16 bits, fp32 or fp8 with a scale for each block of 128; not in the reference.
Kernels: `csrc/silu_mul.hip`; autograd node: `csrc/block_autograd.cpp`.

x holds gate and up side by side, `[..., 2 F]`, as one projection of both gives them.
"""

import torch

from .block_scaled import _TYPES, _fake_codes, _is_e5m2, _plain, as_rows


def _checked(x: torch.Tensor) -> None:
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] % 2:
        raise ValueError(f"x must have an even last dimension (gate and up side by side), got {tuple(x.shape)}")


def silu_mul(x: torch.Tensor) -> torch.Tensor:
    """`silu(x[..., :F]) * x[..., F:]` in x's dtype (bfloat16, float16 or float32), computed in fp32 and rounded once.
    Differentiable once, in reverse mode."""
    _checked(x)
    if x.numel() == 0:
        return x[..., : x.shape[-1] // 2] * 1
    y = torch.ops.feather_ops.silu_mul.default(as_rows(x))
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


def silu_mul_quantized(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of `silu_mul(x)`, quantized as `quantize_blocks` does, from its unrounded values: what
    `block_scaled_mm` takes. Not differentiable."""
    _checked(x)
    e5m2 = _is_e5m2(dtype)
    x = _plain(x)
    half = x.shape[-1] // 2
    if x.numel() == 0:
        return (x.new_empty((*x.shape[:-1], half), dtype=dtype),
                x.new_empty((*x.shape[:-1], -(-half // 128)), dtype=torch.float32))
    codes, scale = torch.ops.feather_ops.silu_mul_quantized.default(as_rows(x), e5m2)
    if x.dim() != 2:
        codes, scale = codes.reshape(*x.shape[:-1], half), scale.reshape(*x.shape[:-1], scale.shape[-1])
    return codes, scale


@torch.library.register_fake("feather_ops::silu_mul")
def _(x):
    return x.new_empty((x.shape[0], x.shape[1] // 2))


@torch.library.register_fake("feather_ops::silu_mul_quantized")
def _(x, e5m2):
    return _fake_codes(x, x.shape[0], x.shape[1] // 2, x.shape[0], e5m2)


@torch.library.register_fake("feather_ops::silu_mul_backward")
def _(grad_y, x):
    return x.new_empty(x.shape)
