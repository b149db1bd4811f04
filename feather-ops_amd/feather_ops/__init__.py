"""feather_ops for MI355X (gfx950): fp16/bf16 x fp8 scaled matmul on hand-written CDNA4 kernels.

Import order mirrors the reference's `feather_ops/__init__.py:1-3`: torch first, then the native
extension, which registers `torch.ops.feather_ops.*`.
"""

import torch  # noqa: F401  torch's libraries must be loaded before the extension

from . import _lib

_lib.load()

from .block_scaled import (  # noqa: E402
    BlockScaledLinear,
    block_scaled_linear,
    block_scaled_mm,
    quantize_blocks,
    to_block_scaled_linear,
)
from .convert import bf16_to_fp16  # noqa: E402
from .gate import silu_mul, silu_mul_quantized  # noqa: E402
from .gated import gated_linear  # noqa: E402
from .int4 import (  # noqa: E402
    Int4Linear,
    dequantize_int4,
    int4_gated_linear,
    int4_linear,
    quantize_int4,
    to_int4_linear,
)
from .modules import ScaledMMLinear, relabel_modules, relabelled_class, to_scaled_mm_linear  # noqa: E402
from .norm import rms_norm, rms_norm_quantized  # noqa: E402
from .scaled_mm import (  # noqa: E402
    prepack_b_for_scaled_mm,
    prepack_transpose,
    scaled_mm_hip,
    select_scaled_mm_config,
    select_scaled_mm_splits,
    set_weight_streaming,
    tile_shape,
)

__all__ = [
    "BlockScaledLinear",
    "Int4Linear",
    "ScaledMMLinear",
    "bf16_to_fp16",
    "block_scaled_linear",
    "block_scaled_mm",
    "dequantize_int4",
    "gated_linear",
    "int4_gated_linear",
    "int4_linear",
    "prepack_b_for_scaled_mm",
    "prepack_transpose",
    "quantize_blocks",
    "quantize_int4",
    "relabel_modules",
    "relabelled_class",
    "rms_norm",
    "rms_norm_quantized",
    "scaled_mm_hip",
    "select_scaled_mm_config",
    "select_scaled_mm_splits",
    "set_weight_streaming",
    "silu_mul",
    "silu_mul_quantized",
    "tile_shape",
    "to_block_scaled_linear",
    "to_int4_linear",
    "to_scaled_mm_linear",
]
