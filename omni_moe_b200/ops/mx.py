"""MX blocks: 32 neighbours of a row share a power-of-two scale (e8m0), each value is held as e4m3 - 1.03 bytes a value.

The scale is the smallest power of two (>= 2^-127) for which 448 scales cover the block's largest finite magnitude; a
value is rounded to 3 mantissa bits (to nearest, ties to even), at most 2^-4 of itself while it is at least 2^-6 scales;
a value that is not finite becomes NaN and does not count for the scale.
"""
from __future__ import annotations

import torch

from .. import _lib

BLOCK = 32
CODE_DTYPE, SCALE_DTYPE = torch.float8_e4m3fn, torch.float8_e8m0fnu


def scale_columns(cols: int) -> int:
    return -(-cols // BLOCK)


def mx_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes [rows, cols], scales [rows, ceil(cols / 32)])`` of a matrix (bf16, fp16 or fp32; rows may have a stride).
    The codes carry no gradient."""
    return _lib.binding().mx_quantize(x)


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that the codes stand for: exact wherever the type's range holds them (a code may stand for up to 2^128:
    infinite in bf16 and fp32; fp16 overflows and underflows earlier).  Scale byte 255 stands for NaN,
    as in ``torch.float8_e8m0fnu``; :func:`mx_quantize` never gives it."""
    return _lib.binding().mx_dequantize(codes, scales, dtype)
