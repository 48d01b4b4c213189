"""Shared SwiGLU MLP whose backward reads 8-bit activation checkpoints (reference MLP: omni_moe/ops/triton/interface.py:7-29;
the checkpoints have no counterpart there)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ._common import aligned, as_bf16, pad_both, pad_last, refuse_tangents
from .mx import CODE_DTYPE, SCALE_DTYPE, mx_dequantize, mx_quantize, scale_columns


def _gate_up_blocks(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The gate | up values ``[T, 2I]`` in bf16 (each half has its own blocks)."""
    i, b = codes.size(1) // 2, scales.size(1) // 2
    return torch.cat([mx_dequantize(codes[:, j * i:(j + 1) * i], scales[:, j * b:(j + 1) * b]) for j in range(2)], 1)


def mlp_ckpt_backward(dy: torch.Tensor, x: Optional[torch.Tensor], codes: torch.Tensor, scales: torch.Tensor, gate_weight: torch.Tensor,
                      up_weight: torch.Tensor, down_weight: torch.Tensor, limit: float = 0.0, need_x: bool = True,
                      need_gate_up: bool = True, need_down: bool = True):
    """Gradients ``(dx, d_gate, d_up, d_down)`` (None where not needed) from the MX blocks of the gate | up pre-activations and
    ``x`` as the weight gradients are to see it (needed for ``need_gate_up`` only)."""
    from .autograd import _operands_in_place, mlp_backward
    if _operands_in_place():
        return tuple(_lib.binding().mlp_ckpt_backward(dy, x, codes, scales, gate_weight, up_weight, down_weight, limit, need_x, need_gate_up,
                                                      need_down, _lib.status_ptr(dy)))
    # the GEMMs that read transposed operands in place are switched off: the same values as bf16 copies
    t, h = dy.shape
    x = x if x is not None else torch.zeros((t, h), device=dy.device, dtype=torch.bfloat16)
    dx, d_wg, d_wu, d_wd = mlp_backward(dy, x, gate_weight, up_weight, down_weight, need_weight_grads=need_gate_up or need_down,
                                        gate_up=_gate_up_blocks(codes, scales), limit=limit or None)
    return (dx if need_x else None, d_wg if need_gate_up else None, d_wu if need_gate_up else None, d_wd if need_down else None)


class MlpCkptCopiesFunction(torch.autograd.Function):
    """The same operator with the gradient GEMMs through transposed copies (``OMNI_MOE_B200_MLP_BWD=copies``,
    ``OMNI_MOE_B200_GEMM=1cta``); otherwise the node of the torch binding is used."""

    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, down_weight, limit, x_codes, x_scales, keep_x):
        xb, wg, wu, wd = as_bf16(x), as_bf16(gate_weight), as_bf16(up_weight), as_bf16(down_weight)
        t, h = xb.shape
        i = wg.size(0)
        bf = dict(device=xb.device, dtype=torch.bfloat16)
        act, y = torch.empty((t, i), **bf), torch.empty((t, h), **bf)
        codes = torch.empty((t, 2 * i), device=xb.device, dtype=CODE_DTYPE)
        scales = torch.empty((t, 2 * scale_columns(i)), device=xb.device, dtype=SCALE_DTYPE)
        if t:
            lib, status = _lib.load(), _lib.status_ptr(xb)
            with torch.cuda.device(xb.device):
                st = _lib.stream_ptr()
                _lib.check(lib.omni_mlp_gate_up_save_mx(xb.data_ptr(), wg.data_ptr(), wu.data_ptr(), t, h, i, limit, act.data_ptr(),
                                                        codes.data_ptr(), scales.data_ptr(), status, st))
                _lib.check(lib.omni_mlp_down(act.data_ptr(), wd.data_ptr(), t, h, i, None, y.data_ptr(), status, st))
        kept = (xb, None) if keep_x else (x_codes, x_scales) if x_codes is not None else mx_quantize(xb)
        ctx.save_for_backward(wg, wu, wd, codes, scales, *kept)
        ctx.limit, ctx.keep_x = limit, keep_x
        ctx.dtypes = (x.dtype, gate_weight.dtype, up_weight.dtype, down_weight.dtype)
        return y.to(x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        wg, wu, wd, codes, scales, xk, xs = ctx.saved_tensors
        need = ctx.needs_input_grad
        x = xk if ctx.keep_x else mx_dequantize(xk, xs)
        grads = mlp_ckpt_backward(aligned(as_bf16(dy)), x, codes, scales, wg, wu, wd, ctx.limit, need_x=need[0], need_gate_up=need[1] or need[2],
                                  need_down=need[3])
        return tuple(g.to(dt) if n and g is not None else None for g, dt, n in zip(grads, ctx.dtypes, need)) + (None,) * 4


def omni_mlp_ckpt_func(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, down_weight: torch.Tensor,
                       limit: Optional[float] = None, x_mx: Optional[tuple[torch.Tensor, torch.Tensor]] = None,
                       keep_x: bool = False) -> torch.Tensor:
    """``(silu(x Wg^T) * (x Wu^T)) Wd^T`` as :func:`omni_mlp_func`, keeping for the backward 1.03 bytes a value instead of 2:
    the MX blocks (see :mod:`omni_moe_b200.ops.mx`) of the two pre-activations and of ``x``.

    The output does not depend on the checkpoints.  The gradients are those of the formula at the values that the codes
    stand for: ``dWd = dy^T act^``, ``(dWg ; dWu) = (dg | du)^T x^``, ``dx = dg Wg + du Wu`` with ``dg``, ``du``, ``act^`` from the
    decoded pre-activations.

    :param x: (num_tokens, hidden_size);  gate_weight, up_weight: (intermediate_size, hidden_size);
        down_weight: (hidden_size, intermediate_size)
    :param limit: optional clamp of gate and up before the activation, as in :func:`omni_mlp_func`; the backward applies it
        to the decoded values
    :param x_mx: MX blocks ``(codes, scales)`` of ``x`` that the caller has already, such as
        ``omni_rms_norm_func(..., quantize=True)`` gives; without them ``x`` is encoded here (where the weights need
        gradients)
    :param keep_x: keep ``x`` itself instead of its blocks (another operator keeps the same tensor anyway)
    :return y: (num_tokens, hidden_size), dtype of ``x``

    Operands other than bf16 are rounded to it; sums are fp32.
    """
    tensors = (x, gate_weight, up_weight, down_weight)
    refuse_tangents("omni_mlp_ckpt_func", *tensors)
    _lib.require_cuda(*tensors)
    if x.dim() != 2 or gate_weight.dim() != 2:
        raise ValueError("omni_mlp_ckpt_func takes matrices")
    (t, h), i = x.shape, gate_weight.size(0)
    if gate_weight.shape != (i, h) or up_weight.shape != (i, h) or down_weight.shape != (h, i):
        raise ValueError("gate_weight and up_weight must be (intermediate, hidden), down_weight (hidden, intermediate)")
    index = x.get_device()
    if gate_weight.get_device() != index or up_weight.get_device() != index or down_weight.get_device() != index:
        raise RuntimeError(f"all tensors must be on {x.device}")
    if limit is not None and not limit > 0:
        raise ValueError("limit must be positive")
    codes = scales = None
    if x_mx is not None:
        if keep_x:
            raise ValueError("x_mx and keep_x exclude one another")
        codes, scales = x_mx
        if codes.dtype != CODE_DTYPE or scales.dtype != SCALE_DTYPE:
            raise ValueError("MX blocks are a matrix of float8_e4m3fn codes and one of float8_e8m0fnu scales")
        if codes.shape != (t, h) or scales.shape != (t, scale_columns(h)) or codes.get_device() != index or scales.get_device() != index:
            raise ValueError(f"x_mx must be the blocks of x: codes of shape {(t, h)} and scales of shape {(t, scale_columns(h))} on {x.device}")
    padded = h % 8 or i % 8
    if not (torch.is_grad_enabled() and (x.requires_grad or gate_weight.requires_grad or up_weight.requires_grad or down_weight.requires_grad)):
        from .mlp import mlp_forward
        x, gate_weight, up_weight, down_weight = (as_bf16(v) for v in tensors)
        y = mlp_forward(*(aligned(v) for v in (pad_last(x), pad_both(gate_weight), pad_both(up_weight), pad_both(down_weight))), limit=limit)
        return (y[:, :h].contiguous() if padded else y).to(tensors[0].dtype)
    if padded:
        # zero columns: gate = up = 0 there, nothing is added and their gradients are cut off again; a block of 32 that is
        # filled up with zeros keeps its scale
        if codes is not None:
            codes = pad_last(codes.view(torch.uint8)).view(CODE_DTYPE)
        x, gate_weight, up_weight, down_weight = pad_last(x), pad_both(gate_weight), pad_both(up_weight), pad_both(down_weight)
    x, gate_weight, up_weight, down_weight = (aligned(v) for v in (x, gate_weight, up_weight, down_weight))
    from .autograd import _operands_in_place
    if _operands_in_place():
        y = _lib.binding().mlp_ckpt(x, gate_weight, up_weight, down_weight, float(limit or 0.0), codes, scales, bool(keep_x),
                                    _lib.status_ptr(x))
    else:
        y = MlpCkptCopiesFunction.apply(x, gate_weight, up_weight, down_weight, float(limit or 0.0), codes, scales, bool(keep_x))
    return y[:, :h].contiguous() if padded else y
