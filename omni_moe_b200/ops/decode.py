"""The whole layer for a few tokens in one kernel: the serving form of ``OmniMoE.forward``
(reference: omni_moe/modules/omni_moe.py:60-106)."""
from __future__ import annotations

import torch

from .. import _lib
from ._common import as_bf16, pad_both, pad_last

MAX_TOKENS = 64
_WORKSPACES: dict = {}


def _workspace(nbytes: int, index: int, stream: int) -> torch.Tensor:
    """Scratch of a call on the current stream; its head holds counters that every launch finds and leaves at zero.
    One buffer for each (device, stream): launches on one stream follow one another, launches on different streams may
    overlap and must not share.  While a graph is captured the buffer belongs to the graph (zeroed in every replay),
    so graphs that replay beside each other or beside eager calls share nothing."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, device=torch.device("cuda", index), dtype=torch.uint8)
    key = (index, stream)
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(nbytes, device=torch.device("cuda", index), dtype=torch.uint8)
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
    index = x.get_device()
    if index < 0:
        _lib.require_cuda(x)
    if x.dim() != 2:
        raise ValueError(f"omni_decode_func takes a matrix of tokens, got a tensor of shape {tuple(x.shape)}")
    t, h = x.shape
    i, n, k = gate_weight.size(0), router_x.size(0), int(num_experts_per_token)
    if t > MAX_TOKENS:
        raise ValueError(f"omni_decode_func takes at most {MAX_TOKENS} tokens, got {t}: use OmniMoE.forward")
    if gate_weight.shape != (i, h) or up_weight.shape != (i, h) or down_weight.shape != (h, i):
        raise ValueError("gate_weight and up_weight must be (intermediate, hidden), down_weight (hidden, intermediate)")
    if router_x.shape != (n, h) or router_y.shape != (n, h):
        raise ValueError("router_x and router_y must both be (sqrt_n, hidden)")
    experts = up_embed.size(0)
    if up_embed.shape != (experts, h) or down_embed.shape != (experts, h) or experts < n * n:
        raise ValueError("up_embed and down_embed must both be (num_experts, hidden) with at least sqrt_n ** 2 rows")
    if min(h, i, n) < 1 or not 1 <= k <= min(128, n * n):
        raise ValueError(f"num_experts_per_token must be in [1, {min(128, n * n)}], got {k}")
    if (bn_scale is None) != (bn_shift is None):
        raise ValueError("bn_scale and bn_shift must be given together")
    if bn_scale is not None:
        for v in (bn_scale, bn_shift):
            if v.shape != (2 * n,) or v.dtype != torch.float32 or v.get_device() != index:
                raise ValueError("bn_scale and bn_shift must be float32 vectors of 2 * sqrt_n values on the device of x")
        bn_scale, bn_shift = bn_scale.contiguous(), bn_shift.contiguous()
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("omni_decode_func has no backward: call it under torch.no_grad(), or OmniMoE.forward to train")
    pointers = []
    for v in tensors:
        if v.get_device() != index:
            _lib.require_cuda(v)
            raise RuntimeError(f"all tensors must be on {x.device}, got one on {v.device}")
        p = v.data_ptr()
        if v.dtype != torch.bfloat16 or p % 16 or h % 8 or i % 8 or not v.is_contiguous():
            # something to convert, copy or pad first
            return _prepared(tensors, k, bn_scale, bn_shift)
        pointers.append(p)
    y = torch.empty_like(x)
    if t:
        lib = _lib.load()
        with _lib.on_device(index):
            stream = _lib.stream_ptr(index)
            ws = _workspace(lib.omni_decode_workspace_bytes(t, h, i, n, k), index, stream)
            _lib.check(lib.omni_decode(*pointers, _lib.ptr(bn_scale), _lib.ptr(bn_shift), t, h, i, n, k, experts, y.data_ptr(),
                                       ws.data_ptr(), ws.numel(), _lib.device_status(x.device).data_ptr(), stream))
    return y


def _prepared(tensors, k, bn_scale, bn_shift):
    """The call on bf16 operands that are contiguous, aligned and a multiple of 8 wide."""
    x = tensors[0]
    x, wg, wu, wd, kx, ky, up, down = (as_bf16(v) for v in tensors)
    h = x.size(1)
    # zero columns add nothing to a dot product and give output columns that are cut off again
    ready = (pad_last(x), pad_both(wg), pad_both(wu), pad_both(wd), pad_last(kx), pad_last(ky), pad_last(up), pad_last(down))
    y = omni_decode_func(*(_aligned(v) for v in ready), k, bn_scale, bn_shift)
    return (y if y.size(1) == h else y[:, :h].contiguous()).to(tensors[0].dtype)
