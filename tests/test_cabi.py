"""The C-ABI library loads and exports everything the header declares; argument checks that need
no device are exercised.  No kernel is launched here."""
import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from omni_moe_b200 import _lib
    from omni_moe_b200.build import build
    build()
    return _lib.load()


def header_symbols():
    text = open(os.path.join(ROOT, "include", "omni_moe_b200.h")).read()
    return sorted(set(re.findall(r"OMNI_API[^;(]*?\b(omni_\w+)\s*\(", text)))


def test_header_symbols_exported(lib):
    names = header_symbols()
    assert len(names) >= 12
    for n in names:
        assert hasattr(lib, n), f"{n} declared in the header but not exported"


def test_bindings_cover_header():
    from omni_moe_b200 import _lib
    assert sorted(_lib.SIGNATURES) == header_symbols()


def test_version_and_rejections(lib):
    assert lib.omni_version() == 100
    # k out of range is refused before anything touches the device
    rc = lib.omni_router_topk(None, None, 0, 4, 8, 0, None, None, 0, None, None)
    assert rc < 0 and b"k must be" in lib.omni_last_error()
    rc = lib.omni_router_topk(None, None, 0, 4, 2000, 4, None, None, 0, None, None)
    assert rc < 0 and b"sqrt_n" in lib.omni_last_error()
    rc = lib.omni_expert_coef(None, None, None, None, None, 4, 2, 12, 16, None, None, None)
    assert rc < 0 and b"multiple of 8" in lib.omni_last_error()
    rc = lib.omni_mlp_fwd(None, None, None, None, 4, 64, 100, None, None, None, None, None)
    assert rc < 0 and b"intermediate" in lib.omni_last_error()
    # entries of the backward and of the clamp: argument errors come back as codes with a message
    rc = lib.omni_mlp_gate_up_limit(None, None, None, 4, 64, 64, -0.5, None, None, None, None)
    assert rc < 0 and b"limit" in lib.omni_last_error()
    rc = lib.omni_swiglu_bwd_limit(None, None, 4, 64, float("nan"), None, None, None, 0, None, None)
    assert rc < 0 and b"limit" in lib.omni_last_error()
    rc = lib.omni_swiglu_bwd(None, None, 4, 12, None, None, None, 0, None)
    assert rc < 0 and b"multiple of 8" in lib.omni_last_error()
    rc = lib.omni_mlp_gate_up_save(None, None, None, 4, 64, 64, None, None, None, None)
    assert rc < 0 and b"NULL" in lib.omni_last_error()
    assert lib.omni_schedule_workspace_bytes(65536, 4096) > 4 * 65536 * 4
    assert lib.omni_schedule_workspace_bytes(-1, 4096) == 0


def test_no_fallback_when_library_missing(monkeypatch):
    from omni_moe_b200 import _lib
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "LIB_PATH", "/nonexistent/libomni_moe_b200.so")
    with pytest.raises(RuntimeError, match="no fallback"):
        _lib.load()


def test_ops_refuse_cpu_tensors():
    import torch
    from omni_moe_b200.ops import omni_router_func
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        omni_router_func(torch.zeros(4, 8), torch.zeros(4, 8), 8, 2)


def test_reference_assert_messages():
    import torch
    from omni_moe_b200.ops import omni_router_func
    with pytest.raises(AssertionError, match="multiple of 2"):
        omni_router_func(torch.zeros(4, 8), torch.zeros(4, 8), 8, 3)
    with pytest.raises(AssertionError, match="less than or equal to 128"):
        omni_router_func(torch.zeros(4, 16), torch.zeros(4, 16), 16, 130)


def test_module_state_dict_matches_reference_names():
    from omni_moe.modules.omni_moe import OmniMoE, OmniMoEConfig
    m = OmniMoE(OmniMoEConfig(64, 128, "silu", 256, 4))
    keys = set(m.state_dict().keys())
    assert keys == {
        "gate_proj.weight", "up_proj.weight", "down_proj.weight", "router_gate_x.weight", "router_gate_y.weight",
        "router_norm_x.running_mean", "router_norm_x.running_var", "router_norm_x.num_batches_tracked",
        "router_norm_y.running_mean", "router_norm_y.running_var", "router_norm_y.num_batches_tracked",
        "up_embed.weight", "down_embed.weight"}
    assert m.up_embed.weight.shape == (256, 64) and m.router_gate_x.weight.shape == (16, 64)
    with pytest.raises(ValueError):
        OmniMoE(OmniMoEConfig(64, 128, "gelu", 256, 4))


def test_decode_rejections(lib):
    # x .. down_table, bn_scale, bn_shift | tokens, hidden, intermediate, sqrt_n, k, experts | y, workspace, bytes, status, stream
    def call(t=4, h=64, i=64, n=8, k=4, experts=64, bn=(None, None)):
        return lib.omni_decode(*([None] * 8), *bn, t, h, i, n, k, experts, None, None, 0, None, None), lib.omni_last_error()

    for kw, what in ((dict(t=65), b"num_tokens"), (dict(t=-1), b"num_tokens"), (dict(h=60), b"multiple of 8"), (dict(h=0), b"multiple of 8"),
                     (dict(h=16392), b"at most 16384"), (dict(i=4), b"intermediate"), (dict(n=1025, experts=1 << 21), b"sqrt_n"),
                     (dict(k=0), b"k must be"), (dict(k=129, n=16, experts=256), b"k must be"), (dict(k=5, n=2, experts=4), b"exceeds"),
                     (dict(experts=63), b"tables"), (dict(bn=(16, None)), b"together"), (dict(), b"NULL")):
        rc, msg = call(**kw)
        assert rc < 0 and what in msg, (kw, msg)
    assert call(t=0)[0] == 0  # nothing to do
    assert lib.omni_decode_max_tokens() == 64
    assert lib.omni_decode_workspace_bytes(65, 64, 64, 8, 4) == 0
    # counters, partial logits, partial routed sums (one block a token here), activation, partial sums of the down projection
    assert lib.omni_decode_workspace_bytes(3, 24, 40, 5, 7) == 8704 + 4 * 3 * 10 * 4 + 3 * 24 * 4 + 240 + 4 * 3 * 24 * 4


def test_norm_and_mx_rejections(lib):
    def norm(dtype=1, w=1, rows=4, n=64, eps=1e-6, res=(None, None), mx=(None, None)):
        return lib.omni_rms_norm(None, n, res[0], n, None, w, dtype, rows, n, eps, None, res[1], None, *mx, None), lib.omni_last_error()

    for kw, what in ((dict(dtype=3), b"dtype"), (dict(dtype=1, w=2), b"weight"), (dict(rows=-1), b"rows"), (dict(n=0), b"hidden"),
                     (dict(n=16385), b"hidden"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(res=(16, None)), b"together"),
                     (dict(mx=(None, 16)), b"together"), (dict(), b"NULL")):
        rc, msg = norm(**kw)
        assert rc < 0 and what in msg, (kw, msg)
    assert norm(rows=0)[0] == 0
    assert lib.omni_rms_norm(16, 63, None, 0, 16, 1, 1, 2, 64, 1e-6, 16, None, None, None, None, None) < 0
    assert b"row strides" in lib.omni_last_error()
    assert lib.omni_rms_norm_bwd(16, 64, None, 0, 16, 64, 16, 1, 1, 16, 2, 64, 16, 16, None, 0, 16, None) < 0
    assert b"scratch" in lib.omni_last_error()
    assert lib.omni_mx_quantize(None, 4, 0, 2, 0, None, None, None) < 0 and b"cols" in lib.omni_last_error()
    assert lib.omni_mx_quantize(16, 3, 0, 2, 4, 16, 16, None) < 0 and b"row stride" in lib.omni_last_error()
    assert lib.omni_mx_dequantize(None, None, 2, 4, 0, None, None) < 0 and b"NULL" in lib.omni_last_error()


def test_mlp_checkpoint_rejections(lib):
    def save(t=4, h=64, i=64, limit=0.0):
        return lib.omni_mlp_gate_up_save_mx(None, None, None, t, h, i, limit, None, None, None, None, None), lib.omni_last_error()

    for kw, what in ((dict(t=-1), b"num_tokens"), (dict(h=4), b"hidden"), (dict(i=12), b"intermediate"), (dict(limit=-1.0), b"limit"),
                     (dict(limit=float("nan")), b"limit"), (dict(), b"NULL")):
        rc, msg = save(**kw)
        assert rc < 0 and what in msg, (kw, msg)
    assert save(t=0)[0] == 0
    def dact(t=4, h=64, i=64, limit=0.0):
        return lib.omni_mlp_dact_swiglu_mx(None, None, t, h, i, None, None, limit, None, None, None, None), lib.omni_last_error()

    for kw, what in ((dict(t=-1), b"num_tokens"), (dict(h=4), b"hidden"), (dict(i=12), b"intermediate"), (dict(limit=-1.0), b"limit"),
                     (dict(limit=float("nan")), b"limit"), (dict(), b"NULL")):
        rc, msg = dact(**kw)
        assert rc < 0 and what in msg, (kw, msg)
    assert dact(t=0)[0] == 0
