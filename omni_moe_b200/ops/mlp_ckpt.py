"""Shared SwiGLU MLP whose backward reads 8-bit activation checkpoints (reference MLP: omni_moe/ops/triton/interface.py:7-29;
the checkpoints have no counterpart there)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ._common import as_bf16, pad_both, pad_last
from .mx import SCALE_DTYPE, CODE_DTYPE, check_mx, mx_dequantize, mx_quantize, scale_columns


def _gate_up_blocks(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The gate | up values ``[T, 2I]`` in bf16 (each half has its own blocks)."""
    i, b = codes.size(1) // 2, scales.size(1) // 2
    return torch.cat([mx_dequantize(codes[:, j * i:(j + 1) * i], scales[:, j * b:(j + 1) * b]) for j in range(2)], 1)


def mlp_ckpt_backward(dy: torch.Tensor, x: Optional[torch.Tensor], codes: torch.Tensor, scales: torch.Tensor, gate_weight: torch.Tensor,
                      up_weight: torch.Tensor, down_weight: torch.Tensor, limit: float = 0.0, need_x: bool = True,
                      need_gate_up: bool = True, need_down: bool = True):
    """Gradients ``(dx, d_gate, d_up, d_down)`` (None where not needed) from the MX blocks of the gate | up pre-activations and
    ``x`` as the weight gradients are to see it (needed for ``need_gate_up`` only)."""
    from .autograd import _operands_in_place, gemm, mlp_backward
    t, i = codes.size(0), gate_weight.size(0)
    h = gate_weight.size(1)
    dev = dy.device
    bf = dict(device=dev, dtype=torch.bfloat16)
    if t == 0:
        z = lambda need, *s: torch.zeros(s, **bf) if need else None
        return z(need_x, 0, h), z(need_gate_up, i, h), z(need_gate_up, i, h), z(need_down, h, i)
    if not _operands_in_place():
        # the GEMMs that read transposed operands in place are switched off: the same values as bf16 copies
        dx, d_wg, d_wu, d_wd = mlp_backward(dy, x if x is not None else torch.zeros((t, h), **bf), gate_weight, up_weight, down_weight,
                                            need_weight_grads=need_gate_up or need_down, gate_up=_gate_up_blocks(codes, scales),
                                            limit=limit or None)
        return (dx if need_x else None, d_wg if need_gate_up else None, d_wu if need_gate_up else None, d_wd if need_down else None)
    lib = _lib.load()
    status = _lib.device_status(dev)
    dx = d_wg = d_wu = d_wd = None
    dgu = torch.empty((t, 2 * i), **bf)
    act = torch.empty((t, i), **bf) if need_down else None
    dact = gemm(dy, down_weight, False, True, status=status)              # dy [T,H] @ Wd [H,I]
    with _lib.on_device(dev.index):
        _lib.check(lib.omni_swiglu_bwd_mx(codes.data_ptr(), scales.data_ptr(), dact.data_ptr(), t, i, limit, dgu.data_ptr(),
                                          _lib.ptr(act), _lib.stream_ptr()))
    if need_down:
        d_wd = gemm(dy, act, True, True, status=status)                   # dy^T [H,T] @ act [T,I]
    if need_x:
        if i % 64 == 0:
            # dx = dgate @ Wg + dup @ Wu: the two weight matrices as one B operand stacked along K
            dx = torch.empty((t, h), **bf)
            with _lib.on_device(dev.index):
                _lib.check(lib.omni_gemm_bf16_stacked_b(dgu.data_ptr(), 0, 2 * i, gate_weight.data_ptr(), up_weight.data_ptr(), i, h,
                                                        t, h, 2 * i, dx.data_ptr(), h, status.data_ptr(), _lib.stream_ptr()))
        else:
            dx = gemm(dgu, torch.cat((gate_weight, up_weight), 0), False, True, status=status)
    if need_gate_up:
        d_wgu = gemm(dgu, x, True, True, status=status)                   # (dgate | dup)^T [2I,T] @ x [T,H]
        d_wg, d_wu = d_wgu[:i], d_wgu[i:]
    return dx, d_wg, d_wu, d_wd


class MlpCkptFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, down_weight, limit, x_codes, x_scales, keep_x):
        xb, wg, wu, wd = as_bf16(x), as_bf16(gate_weight), as_bf16(up_weight), as_bf16(down_weight)
        t, h = xb.shape
        i = wg.size(0)
        dev = xb.device
        act = torch.empty((t, i), device=dev, dtype=torch.bfloat16)
        codes = torch.empty((t, 2 * i), device=dev, dtype=CODE_DTYPE)
        scales = torch.empty((t, 2 * scale_columns(i)), device=dev, dtype=SCALE_DTYPE)
        y = torch.empty((t, h), device=dev, dtype=torch.bfloat16)
        if t:
            lib, status = _lib.load(), _lib.device_status(dev).data_ptr()
            with _lib.on_device(dev.index):
                st = _lib.stream_ptr()
                _lib.check(lib.omni_mlp_gate_up_save_mx(xb.data_ptr(), wg.data_ptr(), wu.data_ptr(), t, h, i, limit, act.data_ptr(),
                                                        codes.data_ptr(), scales.data_ptr(), status, st))
                _lib.check(lib.omni_mlp_down(act.data_ptr(), wd.data_ptr(), t, h, i, None, y.data_ptr(), status, st))
        kept = (None, None)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            kept = (xb, None) if keep_x else (x_codes, x_scales) if x_codes is not None else mx_quantize(xb)
        ctx.save_for_backward(wg, wu, wd, codes, scales, *kept)
        ctx.limit, ctx.keep_x = limit, keep_x
        ctx.dtypes = (x.dtype, gate_weight.dtype, up_weight.dtype, down_weight.dtype)
        return y.to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        wg, wu, wd, codes, scales, xk, xs = ctx.saved_tensors
        need = ctx.needs_input_grad
        x = xk if xk is None or ctx.keep_x else mx_dequantize(xk, xs)
        grads = mlp_ckpt_backward(as_bf16(dy), x, codes, scales, wg, wu, wd, ctx.limit, need_x=need[0], need_gate_up=need[1] or need[2],
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
    _lib.require_cuda(*tensors)
    if any(v.dim() != 2 for v in tensors):
        raise ValueError("omni_mlp_ckpt_func takes matrices")
    (t, h), i = x.shape, gate_weight.size(0)
    if gate_weight.shape != (i, h) or up_weight.shape != (i, h) or down_weight.shape != (h, i):
        raise ValueError("gate_weight and up_weight must be (intermediate, hidden), down_weight (hidden, intermediate)")
    if any(v.device != x.device for v in tensors):
        raise RuntimeError(f"all tensors must be on {x.device}")
    if limit is not None and not limit > 0:
        raise ValueError("limit must be positive")
    if x_mx is not None:
        if keep_x:
            raise ValueError("x_mx and keep_x exclude one another")
        codes, scales = x_mx
        check_mx(codes, scales)
        if codes.shape != x.shape or codes.device != x.device:
            raise ValueError(f"x_mx must be the blocks of x: codes of shape {tuple(x.shape)} on {x.device}")
    if not (torch.is_grad_enabled() and any(v.requires_grad for v in tensors)):
        from .mlp import mlp_forward
        x, gate_weight, up_weight, down_weight = (as_bf16(v) for v in tensors)
        y = mlp_forward(pad_last(x), pad_both(gate_weight), pad_both(up_weight), pad_both(down_weight), limit=limit)
        return y[:, :h].contiguous().to(tensors[0].dtype)
    codes, scales = x_mx if x_mx is not None else (None, None)
    if h % 8 or i % 8:
        # zero columns: gate = up = 0 there, nothing is added and their gradients are cut off again; a block of 32 that is
        # filled up with zeros keeps its scale
        if codes is not None:
            codes = pad_last(codes.view(torch.uint8)).view(CODE_DTYPE)
        y = MlpCkptFunction.apply(pad_last(x), pad_both(gate_weight), pad_both(up_weight), pad_both(down_weight), float(limit or 0.0),
                                  codes, scales, bool(keep_x))
        return y[:, :h].contiguous()
    return MlpCkptFunction.apply(x, gate_weight, up_weight, down_weight, float(limit or 0.0), codes, scales, bool(keep_x))
