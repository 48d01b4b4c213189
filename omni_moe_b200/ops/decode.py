"""The whole layer for a few tokens in one kernel: the serving form of ``OmniMoE.forward``
(reference: omni_moe/modules/omni_moe.py:60-106)."""
from __future__ import annotations

import torch

from .. import _lib
from ._common import aligned, as_bf16, in_dual_level, pad_both, pad_last, refuse_tangents


def omni_decode_func(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, down_weight: torch.Tensor,
                     router_x: torch.Tensor, router_y: torch.Tensor, up_embed: torch.Tensor, down_embed: torch.Tensor,
                     num_experts_per_token: int, bn_scale: torch.Tensor | None = None,
                     bn_shift: torch.Tensor | None = None) -> torch.Tensor:
    """``y = SwiGLU_MLP(x) + sum_j g[t,j] silu(x[t] . Up[e[t,j]]) Down[e[t,j]]`` for at most 64 tokens, in one kernel.

    The router (gates, the folded BatchNorm ``logit * bn_scale + bn_shift``, log-softmax per axis, product-key top-k,
    ``g = exp(score)``) is part of it; ties go to the lower index, as in :func:`router_topk`.

    :param x: (num_tokens, hidden_size), at most 64 tokens
    :param gate_weight, up_weight: (intermediate_size, hidden_size);  down_weight: (hidden_size, intermediate_size)
    :param router_x, router_y: (sqrt_n, hidden_size) sub-keys, sqrt_n <= 1024
    :param up_embed, down_embed: (num_experts, hidden_size), at least sqrt_n ** 2 rows
    :param num_experts_per_token: k <= 128
    :param bn_scale, bn_shift: (2 * sqrt_n,) float32, x axis first; both or neither
    :return y: (num_tokens, hidden_size), dtype of ``x``

    Operands are bf16 (others are rounded to it per call), sums fp32.  Inference only: with gradients enabled, a call with a
    tensor that requires them is refused.  Device-side faults are reported by ``check_device_status``.
    """
    if in_dual_level():
        refuse_tangents("omni_decode_func", x, gate_weight, up_weight, down_weight, router_x, router_y, up_embed, down_embed, bn_scale, bn_shift)
    k = int(num_experts_per_token)
    y = _lib.binding().decode(x, gate_weight, up_weight, down_weight, router_x, router_y, up_embed, down_embed, k, bn_scale, bn_shift,
                              _lib.status_ptr(x))
    if y is None:  # something to convert, copy or pad first
        y = _prepared((x, gate_weight, up_weight, down_weight, router_x, router_y, up_embed, down_embed), k, bn_scale, bn_shift)
    return y


def _prepared(tensors, k, bn_scale, bn_shift):
    """The call on bf16 operands that are contiguous, aligned and a multiple of 8 wide."""
    x = tensors[0]
    x, wg, wu, wd, kx, ky, up, down = (as_bf16(v) for v in tensors)
    h = x.size(1)
    # zero columns add nothing to a dot product and give output columns that are cut off again
    ready = (pad_last(x), pad_both(wg), pad_both(wu), pad_both(wd), pad_last(kx), pad_last(ky), pad_last(up), pad_last(down))
    y = omni_decode_func(*(aligned(v) for v in ready), k, bn_scale, bn_shift)
    return (y if y.size(1) == h else y[:, :h].contiguous()).to(tensors[0].dtype)
