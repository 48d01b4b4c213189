"""The whole layer for a few tokens in one kernel: the serving form of ``OmniMoE.forward``
(reference: omni_moe/modules/omni_moe.py:60-106)."""
from __future__ import annotations

import torch

from .. import _lib
from ._common import as_bf16, pad_both, pad_last

MAX_TOKENS = 64
_WORKSPACES: dict = {}


def _workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    """Scratch of a call on the current stream; its head holds counters that every launch finds and leaves at zero.
    One buffer for each (device, stream): launches on one stream follow one another, launches on different streams may
    overlap and must not share.  While a graph is captured the buffer belongs to the graph (zeroed in every replay),
    so graphs that replay beside each other or beside eager calls share nothing."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, device=dev, dtype=torch.uint8)
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(nbytes, device=dev, dtype=torch.uint8)
        _WORKSPACES.pop(key, None)
        while len(_WORKSPACES) >= 16:  # a freed buffer goes back to its own stream's pool: in-flight launches keep it
            _WORKSPACES.pop(next(iter(_WORKSPACES)))
        _WORKSPACES[key] = ws
    return ws


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t if t.data_ptr() % 16 == 0 else t.clone()


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

    Operands are bf16 (others are rounded to it per call), sums fp32.  Inference only: a call whose ``x`` carries a
    graph is refused.  Device-side faults are reported by ``check_device_status``.
    """
    tensors = (x, gate_weight, up_weight, down_weight, router_x, router_y, up_embed, down_embed)
    _lib.require_cuda(*tensors, bn_scale, bn_shift)
    for v in tensors:
        if v.dim() != 2:
            raise ValueError(f"omni_decode_func takes matrices, got a tensor of shape {tuple(v.shape)}")
        if v.device != x.device:
            raise RuntimeError(f"all tensors must be on {x.device}, got one on {v.device}")
    t, h = x.shape
    i, n, k = gate_weight.size(0), router_x.size(0), int(num_experts_per_token)
    if t > MAX_TOKENS:
        raise ValueError(f"omni_decode_func takes at most {MAX_TOKENS} tokens, got {t}: use OmniMoE.forward")
    if gate_weight.shape != (i, h) or up_weight.shape != (i, h) or down_weight.shape != (h, i):
        raise ValueError("gate_weight and up_weight must be (intermediate, hidden), down_weight (hidden, intermediate)")
    if router_x.shape != (n, h) or router_y.shape != (n, h):
        raise ValueError("router_x and router_y must both be (sqrt_n, hidden)")
    if up_embed.shape != down_embed.shape or up_embed.size(1) != h or up_embed.size(0) < n * n:
        raise ValueError("up_embed and down_embed must both be (num_experts, hidden) with at least sqrt_n ** 2 rows")
    if min(h, i, n) < 1 or not 1 <= k <= min(128, n * n):
        raise ValueError(f"num_experts_per_token must be in [1, {min(128, n * n)}], got {k}")
    if (bn_scale is None) != (bn_shift is None):
        raise ValueError("bn_scale and bn_shift must be given together")
    for v in (bn_scale, bn_shift):
        if v is not None and (v.shape != (2 * n,) or v.dtype != torch.float32 or v.device != x.device):
            raise ValueError("bn_scale and bn_shift must be float32 vectors of 2 * sqrt_n values on the device of x")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("omni_decode_func has no backward: call it under torch.no_grad(), or OmniMoE.forward to train")
    if h % 8 or i % 8:
        # zero columns add nothing to a dot product and give output columns that are cut off again
        x, gate_weight, up_weight, down_weight, router_x, router_y, up_embed, down_embed = (v.detach() for v in tensors)
        y = omni_decode_func(pad_last(x), pad_both(gate_weight), pad_both(up_weight), pad_both(down_weight), pad_last(router_x),
                             pad_last(router_y), pad_last(up_embed), pad_last(down_embed), k, bn_scale, bn_shift)
        return y[:, :h].contiguous()
    xb, *w = (_aligned(as_bf16(v)) for v in tensors)
    if bn_scale is not None:
        bn_scale, bn_shift = bn_scale.detach().contiguous(), bn_shift.detach().contiguous()
    y = torch.empty((t, h), device=x.device, dtype=torch.bfloat16)
    if t > 0:
        lib = _lib.load()
        with torch.cuda.device(x.device):
            ws = _workspace(lib.omni_decode_workspace_bytes(t, i, n, k), x.device)
            _lib.check(lib.omni_decode(xb.data_ptr(), *(v.data_ptr() for v in w), _lib.ptr(bn_scale), _lib.ptr(bn_shift), t, h, i, n,
                                       k, up_embed.size(0), y.data_ptr(), ws.data_ptr(), ws.numel(),
                                       _lib.device_status(x.device).data_ptr(), _lib.stream_ptr()))
    return y.to(x.dtype)
