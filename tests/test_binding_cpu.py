"""The torch binding of the short operators: it loads, and its errors arrive as Python exceptions.  No GPU."""
import pytest
import torch


@pytest.fixture(scope="module")
def binding():
    from omni_moe_b200 import _lib
    from omni_moe_b200.build import build
    build()
    return _lib.binding()


def test_refuses_cpu_tensors(binding):
    x, w = torch.zeros(4, 64), torch.zeros(64)
    calls = (lambda: binding.rms_norm(x, w, None, 1e-6, False, 0), lambda: binding.mx_quantize(x),
             lambda: binding.mx_dequantize(x, x, torch.float32), lambda: binding.decode(*[x] * 8, 4, None, None, 0))
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_public_functions_refuse_cpu_tensors():
    from omni_moe_b200 import ops
    x, w = torch.zeros(4, 64), torch.zeros(64)
    for call in (lambda: ops.omni_rms_norm_func(x, w), lambda: ops.mx_quantize(x), lambda: ops.omni_mlp_ckpt_func(x, x, x, x),
                 lambda: ops.omni_decode_func(x, x, x, x, x, x, x, x, 4)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_argument_types(binding):
    with pytest.raises(TypeError):
        binding.rms_norm(torch.zeros(4, 64), None, None, 1e-6, False, 0)


def test_linked_against_the_shared_runtime(binding):
    """A static libstdc++ inside the binding would crash on its first formatted error message."""
    import os
    import subprocess
    out = subprocess.run(["readelf", "-d", os.path.abspath(binding.__file__)], capture_output=True, text=True).stdout
    assert "libstdc++.so" in out and "libomni_moe_b200.so" in out


def test_missing_binding_is_reported(monkeypatch):
    import builtins
    from omni_moe_b200 import _lib
    _lib.load()
    monkeypatch.setattr(_lib, "_binding", None)
    real = builtins.__import__

    def without(name, globals=None, locals=None, fromlist=(), level=0):
        if level and fromlist and "_binding" in fromlist:
            raise ImportError("not built")
        return real(name, globals, locals, fromlist, level)

    monkeypatch.setattr(builtins, "__import__", without)
    with pytest.raises(RuntimeError, match="no fallback"):
        _lib.binding()


def test_block_parameters():
    from omni_moe_b200.modules import OmniMoEBlock, OmniMoEConfig
    b = OmniMoEBlock(OmniMoEConfig(64, 128, "silu", 256, 4), eps=1e-5, checkpoint_bits=8)
    names = set(b.state_dict())
    assert "norm.weight" in names and "layer.gate_proj.weight" in names and b.norm.weight.shape == (64,) and b.norm.eps == 1e-5
    with pytest.raises(ValueError, match="8 or 16"):
        OmniMoEBlock(OmniMoEConfig(64, 128, "silu", 256, 4), checkpoint_bits=32)


def test_forward_mode_is_seen_before_anything_runs():
    """Dual tensors and those of torch.func.jvp, which wraps them."""
    import torch.autograd.forward_ad as fw
    from omni_moe_b200 import ops
    x, w = torch.ones(4, 64), torch.ones(64)
    calls = (lambda v: ops.omni_rms_norm_func(v, w).y, lambda v: ops.omni_mlp_ckpt_func(v, v, v, v), lambda v: ops.omni_decode_func(*[v] * 8, 4))
    for call in calls:
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(fw.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
        with fw.dual_level(), pytest.raises(RuntimeError, match="CUDA tensors only"):
            call(x)


def test_names_under_the_reference_paths():
    """What stands beside the layer is found where the layer is, under either package."""
    import omni_moe.modules
    import omni_moe.ops
    import omni_moe_b200.modules
    import omni_moe_b200.ops
    for ours, theirs in ((omni_moe_b200.modules, omni_moe.modules), (omni_moe_b200.ops, omni_moe.ops)):
        for name in ours.__all__:
            assert getattr(theirs, name) is getattr(ours, name)


def test_the_block_asks_for_no_more_tokens_than_the_kernel_takes():
    from omni_moe_b200 import _lib
    from omni_moe_b200.modules import OmniMoEBlock
    assert OmniMoEBlock.DECODE_TOKENS <= _lib.load().omni_decode_max_tokens()
