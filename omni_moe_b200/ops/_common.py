"""Helpers shared by the op wrappers."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def in_dual_level() -> bool:
    """Whether tensors can have forward-mode derivatives at all."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def refuse_tangents(name: str, *tensors) -> None:
    """Raises for tensors with a forward-mode derivative (``None`` entries are skipped): the kernels carry none, and an output
    without one would pass for a derivative of zero."""
    if in_dual_level() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative")


def as_bf16(t: torch.Tensor) -> torch.Tensor:
    """Contiguous bf16 view or copy (the kernels compute on bf16 operands with fp32 accumulation)."""
    t = t.detach()
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    return t.contiguous()


def aligned(t: torch.Tensor) -> torch.Tensor:
    """``t``, copied (differentiably) where its first value is not on a 16-byte boundary, which the GEMMs' operands need."""
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def pad_last(t: torch.Tensor, multiple: int = 8) -> torch.Tensor:
    """``t`` with its last dimension zero-padded up to a multiple (differentiable).  The kernels move
    rows in 16-byte pieces, i.e. want row lengths that are multiples of 8 bf16 elements; other lengths
    (the reference masks its tails instead, e.g. omni_moe/ops/triton/omni_expert.py:67,123) take this
    slower way round: pad with zeros, compute, cut the result back."""
    pad = (-t.size(-1)) % multiple
    return torch.nn.functional.pad(t, (0, pad)) if pad else t


def pad_both(t: torch.Tensor, multiple: int = 8) -> torch.Tensor:
    """2-D ``t`` zero-padded in both dimensions up to multiples (differentiable)."""
    pr, pc = (-t.size(0)) % multiple, (-t.size(1)) % multiple
    return torch.nn.functional.pad(t, (0, pc, 0, pr)) if (pr or pc) else t
