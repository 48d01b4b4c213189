"""RMS norm with the residual's addition and an optional 8-bit output, with gradients (the pre-norm of a block whose
second half is the layer; the reference has the layer alone)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib
from .mx import empty_mx, rows_of

MAX_HIDDEN = 16384


class RmsNormOutput(NamedTuple):
    """``y``: the normed rows; ``h``: the sum that was normed (``x`` itself without a residual); ``codes``, ``scales``: the MX
    blocks of ``y`` (None unless asked for)."""
    y: torch.Tensor
    h: torch.Tensor
    codes: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


def _forward(x, residual, weight, eps, quantize, keep):
    """x, residual: matrices with contiguous rows.  Returns y, h (None without a residual), codes, scales, rstd."""
    t, n = x.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = None if residual is None else torch.empty_like(y)
    rstd = torch.empty(t, device=x.device, dtype=torch.float32) if keep else None
    codes, scales = empty_mx(t, n, x.device) if quantize else (None, None)
    if t:
        index = x.get_device()
        with _lib.on_device(index):
            _lib.check(_lib.load().omni_rms_norm(
                x.data_ptr(), x.stride(0), _lib.ptr(residual), residual.stride(0) if residual is not None else 0, weight.data_ptr(),
                _lib.dtype_code(weight.dtype), _lib.dtype_code(x.dtype), t, n, eps, y.data_ptr(), _lib.ptr(h), _lib.ptr(rstd),
                _lib.ptr(codes), _lib.ptr(scales), _lib.stream_ptr(index)))
    return y, h, codes, scales, rstd


def rms_norm_backward(dy: torch.Tensor, dh: Optional[torch.Tensor], h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      need_weight_grad: bool = True):
    """``(dx, dweight)``: ``dx`` is the gradient of ``x`` and of the residual alike."""
    t, n = h.shape
    dx = torch.empty_like(h, memory_format=torch.contiguous_format)
    if t == 0:
        return dx, torch.zeros_like(weight) if need_weight_grad else None
    dw = torch.empty_like(weight) if need_weight_grad else None
    lib, index = _lib.load(), h.get_device()
    with _lib.on_device(index):
        scratch = torch.empty(lib.omni_rms_norm_bwd_scratch_bytes(t, n), device=h.device, dtype=torch.uint8) if need_weight_grad else None
        _lib.check(lib.omni_rms_norm_bwd(
            dy.data_ptr(), dy.stride(0), _lib.ptr(dh), dh.stride(0) if dh is not None else 0, h.data_ptr(), h.stride(0),
            weight.data_ptr(), _lib.dtype_code(weight.dtype), _lib.dtype_code(h.dtype), rstd.data_ptr(), t, n, dx.data_ptr(),
            _lib.ptr(dw), _lib.ptr(scratch), scratch.numel() if scratch is not None else 0, _lib.device_status(h.device).data_ptr(),
            _lib.stream_ptr(index)))
    return dx, dw


class RmsNormFunction(torch.autograd.Function):
    """y, h, codes, scales from matrices x and residual (or None); codes and scales carry no gradient."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, quantize):
        y, h, codes, scales, rstd = _forward(x, residual, weight, eps, quantize, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.has_residual = h is not None
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(v for v in (codes, scales) if v is not None))
        return y, h, codes, scales

    @staticmethod
    def backward(ctx, dy, dh, _dcodes, _dscales):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if dy is None:  # only the sum was used
            dx = dh
            dw = torch.zeros_like(weight) if need_w else None
        else:
            dx, dw = rms_norm_backward(rows_of(dy), None if dh is None else rows_of(dh), h, weight, rstd, need_w)
        return dx if need_x else None, dx if need_r and ctx.has_residual else None, dw, None, None


def omni_rms_norm_func(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       quantize: bool = False) -> RmsNormOutput:
    """``h = x + residual``; ``y = h * (mean(h^2) + eps)^-1/2 * weight`` over the last dimension.

    :param x: (..., hidden_size) bf16, fp16 or fp32, hidden_size <= 16384
    :param weight: (hidden_size,) of the type of ``x`` or float32
    :param residual: of the shape and type of ``x``, or None.  The sum is rounded to the type before it is normed, so what
        is normed is what is handed on (and what the backward reads).
    :param quantize: also return the MX blocks of ``y`` (see :mod:`omni_moe_b200.ops.mx`): matrices (rows, hidden_size) and
        (rows, ceil(hidden_size / 32)), taken from the fp32 values.  They carry no gradient; as an activation checkpoint
        they go to ``omni_mlp_ckpt_func(..., x_mx=(codes, scales))``.
    :return: :class:`RmsNormOutput`

    Sums are fp32.  Differentiable in ``x``, ``residual`` and ``weight``; the weight's gradient is summed in a fixed order.
    """
    index = x.get_device()
    if index < 0 or weight.get_device() != index or (residual is not None and residual.get_device() != index):
        _lib.require_cuda(x, weight, residual)
        raise RuntimeError(f"all tensors must be on {x.device}")
    _lib.dtype_code(x.dtype)
    shape = x.shape
    n = shape[-1] if shape else 0
    if not 1 <= n <= MAX_HIDDEN:
        raise ValueError(f"the last dimension must be in [1, {MAX_HIDDEN}], got shape {tuple(shape)}")
    if weight.shape != (n,):
        raise ValueError(f"weight must be ({n},), got {tuple(weight.shape)}")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise ValueError("the residual must have the shape and type of x")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    xr, rr, w = rows_of(x), None if residual is None else rows_of(residual), weight.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        y, h, codes, scales = RmsNormFunction.apply(xr, rr, w, eps, bool(quantize))
    else:
        y, h, codes, scales, _ = _forward(xr, rr, w, eps, bool(quantize), False)
    if len(shape) != 2:
        y, h = y.view(shape), None if h is None else h.view(shape)
    return RmsNormOutput(y, x if h is None else h, codes, scales)
