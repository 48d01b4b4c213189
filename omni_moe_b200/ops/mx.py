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


def empty_mx(rows: int, cols: int, dev) -> tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty((rows, cols), device=dev, dtype=CODE_DTYPE),
            torch.empty((rows, scale_columns(cols)), device=dev, dtype=SCALE_DTYPE))


def check_mx(codes: torch.Tensor, scales: torch.Tensor) -> None:
    _lib.require_cuda(codes, scales)
    if codes.dim() != 2 or codes.dtype != CODE_DTYPE or scales.dtype != SCALE_DTYPE:
        raise ValueError("MX blocks are a matrix of float8_e4m3fn codes and one of float8_e8m0fnu scales")
    if scales.shape != (codes.size(0), scale_columns(codes.size(1))):
        raise ValueError(f"codes of shape {tuple(codes.shape)} need scales of shape "
                         f"{(codes.size(0), scale_columns(codes.size(1)))}, got {tuple(scales.shape)}")
    if codes.device != scales.device:
        raise RuntimeError("codes and scales must be on one device")


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x [..., C]`` as a matrix whose rows are contiguous and do not overlap (a view wherever its strides allow)."""
    if x.dim() == 2 and x.is_contiguous():
        return x
    x = x.reshape(-1, x.size(-1))
    contiguous_rows = x.size(1) == 1 or x.stride(1) == 1
    return x if contiguous_rows and (x.size(0) <= 1 or x.stride(0) >= x.size(1)) else x.contiguous()


def mx_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes [rows, cols], scales [rows, ceil(cols / 32)])`` of a matrix (bf16, fp16 or fp32; rows may have a stride)."""
    _lib.require_cuda(x)
    if x.dim() != 2:
        raise ValueError(f"mx_quantize takes a matrix, got a tensor of shape {tuple(x.shape)}")
    code = _lib.dtype_code(x.dtype)
    x = rows_of(x.detach())
    rows, cols = x.shape
    codes, scales = empty_mx(rows, cols, x.device)
    if rows and cols:
        index = x.get_device()
        with _lib.on_device(index):
            _lib.check(_lib.load().omni_mx_quantize(x.data_ptr(), x.stride(0), code, rows, cols, codes.data_ptr(),
                                                    scales.data_ptr(), _lib.stream_ptr(index)))
    return codes, scales


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that the codes stand for: exact wherever the type's range holds them (a code may stand for up to 2^128:
    infinite in bf16 and fp32; fp16 overflows and underflows earlier)."""
    check_mx(codes, scales)
    code = _lib.dtype_code(dtype)
    codes, scales = codes.contiguous(), scales.contiguous()
    rows, cols = codes.shape
    out = torch.empty((rows, cols), device=codes.device, dtype=dtype)
    if rows and cols:
        index = codes.get_device()
        with _lib.on_device(index):
            _lib.check(_lib.load().omni_mx_dequantize(codes.data_ptr(), scales.data_ptr(), rows, cols, code, out.data_ptr(),
                                                      _lib.stream_ptr(index)))
    return out
