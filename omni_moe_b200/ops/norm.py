"""RMS norm with the residual's addition and an optional 8-bit output, with gradients (the pre-norm of a block whose
second half is the layer; the reference has the layer alone)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib
from ._common import refuse_tangents


class RmsNormOutput(NamedTuple):
    """``y``: the normed rows; ``h``: the sum that was normed (``x`` itself without a residual); ``codes``, ``scales``: the MX
    blocks of ``y`` (None unless asked for)."""
    y: torch.Tensor
    h: torch.Tensor
    codes: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


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

    Sums are fp32; rows may have any mean square that fp32 holds.  (With ``eps`` below 1e-30, rows whose root mean square is below
    1e-17 leave fp32's normal range and lose precision, below 1e-19 all of it.)  Differentiable in ``x``, ``residual`` and
    ``weight``; the weight's gradient is summed in a fixed order.
    """
    refuse_tangents("omni_rms_norm_func", x, weight, residual)
    return RmsNormOutput(*_lib.binding().rms_norm(x, weight, residual, float(eps), bool(quantize), _lib.status_ptr(x)))
