"""The operators together, as a pre-norm block uses them: norm with the residual's addition, then the layer, for training
(8-bit checkpoints) and for serving (a few tokens)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = dict(hidden_size=256, intermediate_size=512, hidden_act="silu", num_experts=1024, num_experts_per_token=8)


def blocks(n, bits=16, seed=0, **over):
    from omni_moe_b200.modules import OmniMoEBlock, OmniMoEConfig
    torch.manual_seed(seed)
    made = [OmniMoEBlock(OmniMoEConfig(**{**SIZES, **over}), checkpoint_bits=bits).bfloat16().cuda() for _ in range(n)]
    for b in made:
        b.norm.weight.data += 0.1 * torch.randn_like(b.norm.weight)
    return made


def run(stack, x):
    y, h = x, None
    for b in stack:
        y, h = b(y, h)
    return y + h


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_serving_matches_the_long_form():
    stack = [b.eval() for b in blocks(3)]
    x = torch.randn(2, 40, 256, device="cuda").bfloat16()
    with torch.no_grad():
        long = run(stack, x)                                      # 80 tokens: the layer's forward
        short = torch.cat([run(stack, x[i:i + 1]) for i in range(2)])  # 40 each: one kernel a layer
        one = torch.cat([run(stack, x[:1, j:j + 1]) for j in range(5)], 1)
    for b in stack:
        b.layer.check_status()
    # every block rounds its activation and output to bf16 (2^-8 each at most) on both sides, and what it adds to the
    # residual stream is smaller than the stream: three blocks stay below 3 * 2 * 2^-8
    assert rel(short, long) < 6 * 2 ** -8
    assert rel(one, long[:1, :5]) < 6 * 2 ** -8


def test_serving_in_a_graph():
    stack = [b.eval() for b in blocks(2)]
    x = torch.randn(1, 7, 256, device="cuda").bfloat16()
    with torch.no_grad():
        want = run(stack, x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(stack, x)
        x2 = torch.randn_like(x)
        want2 = run(stack, x2)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        x.copy_(x2)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want2)


@pytest.mark.parametrize("tokens", [(2, 70), (1, 9), (1, 1)])
def test_training_with_checkpoints(tokens):
    full, eight = blocks(2), blocks(2, bits=8)
    x = torch.randn(*tokens, 256, device="cuda").bfloat16()
    c = torch.randn(*tokens, 256, device="cuda").bfloat16()
    for stack in (full, eight):   # running statistics: a batch of one row has no variance to train on
        for b in stack:
            b.layer.eval()
    grads = []
    outs = []
    for stack in (full, eight):
        leaf = x.clone().requires_grad_()
        out = run(stack, leaf)
        out.backward(c)
        outs.append(out.detach())
        grads.append([leaf.grad] + [p.grad for b in stack for p in b.parameters()])
        names = ["x"] + [n for b in stack for n, _ in b.named_parameters()]
    assert torch.equal(outs[0], outs[1])            # what is kept does not change what is computed
    for name, a, b in zip(names, grads[1], grads[0]):
        assert torch.isfinite(a).all()
        # the codes are off by 2^-4 of a value at most, independently: of a gradient's norm less than that
        assert rel(a, b) < 2 ** -4 or float(b.double().norm()) == 0.0, name
    last = dict(eight[1].named_parameters())
    assert any(not torch.equal(a, b) for a, b in zip(grads[1], grads[0]))  # the checkpoints are in use
    assert last["layer.gate_proj.weight"].grad.dtype == torch.bfloat16


def test_training_mode_and_norm_gradient():
    stack = blocks(2, bits=8)
    x = torch.randn(2, 64, 256, device="cuda").bfloat16()
    before = stack[0].layer.router_norm_x.running_mean.clone()
    run(stack, x).float().square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for b in stack for p in b.parameters())
    assert not torch.equal(before, stack[0].layer.router_norm_x.running_mean)


def test_norm_codes_feed_the_mlp():
    """The norm's 8-bit output as the MLP's checkpoint of its input: the chain's gradients are those with the codes that the
    MLP would make itself of the norm's 16-bit output, up to the rounding between the two."""
    from omni_moe_b200.ops import omni_mlp_ckpt_func, omni_rms_norm_func
    torch.manual_seed(1)
    x, r = (torch.randn(96, 256, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w = torch.ones(256, device="cuda").bfloat16().requires_grad_()
    mats = [(torch.randn(*s, device="cuda") / s[1] ** 0.5).bfloat16().requires_grad_() for s in ((512, 256), (512, 256), (256, 512))]
    c = torch.randn(96, 256, device="cuda").bfloat16()
    leaves = [x, r, w, *mats]
    n = omni_rms_norm_func(x, w, r, quantize=True)
    given = torch.autograd.grad(omni_mlp_ckpt_func(n.y, *mats, x_mx=(n.codes, n.scales)) + n.h, leaves, c)
    n = omni_rms_norm_func(x, w, r)
    made = torch.autograd.grad(omni_mlp_ckpt_func(n.y, *mats) + n.h, leaves, c)
    for a, b in zip(given, made):
        # a code of the fp32 value and one of its bf16 rounding differ where the rounding crosses a border of the 3-bit
        # grid: by one step (2^-3) in at most one value of 2^-8 / 2^-4 = 1/16: 2^-3 / 4 of the norm at most
        assert rel(a, b) < 2 ** -5
    assert torch.equal(given[0], given[1])


def test_checkpoint_bits_are_checked():
    from omni_moe_b200.modules import OmniMoE, OmniMoEConfig
    m = OmniMoE(OmniMoEConfig(**SIZES))
    assert m.checkpoint_activations(8) is m
    with pytest.raises(ValueError, match="8 or 16"):
        m.checkpoint_activations(4)


def test_forward_mode_derivatives_are_refused():
    """The kernels carry no tangents: an output without one would be a derivative of zero."""
    from omni_moe_b200.modules import OmniMoE, OmniMoEBlock, OmniMoEConfig
    from omni_moe_b200.ops import omni_decode_func, omni_mlp_ckpt_func, omni_rms_norm_func
    import torch.autograd.forward_ad as fw
    torch.manual_seed(0)
    h, i, n = 64, 128, 8
    r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    x, w = r(4, h), r(h)
    mlp = [r(i, h), r(i, h), r(h, i)]
    rest = [r(n, h), r(n, h), r(n * n, h), r(n * n, h)]
    fold = [torch.ones(2 * n, device="cuda"), torch.zeros(2 * n, device="cuda")]
    calls = [(lambda a: omni_rms_norm_func(a[0], a[1], a[2]), [x, w, x.clone()]),
             (lambda a: omni_mlp_ckpt_func(*a), [x, *mlp]),
             (lambda a: omni_decode_func(*a[:8], 4, *a[8:]), [x, *mlp, *rest, *fold])]
    for call, args in calls:
        call(args)
        with fw.dual_level():
            call(args)             # nothing carries a tangent
            for j in range(len(args)):
                dual = [fw.make_dual(a, torch.ones_like(a)) if q == j else a for q, a in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual)
                leaf = [a.clone().requires_grad_() if q != j and call is not calls[2][0] else a for q, a in enumerate(dual)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(leaf)
        call(args)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: omni_rms_norm_func(v, w).y, (x,), (torch.ones_like(x),))
    config = OmniMoEConfig(h, i, "silu", n * n, 4)
    layer, block = OmniMoE(config).bfloat16().cuda().eval(), OmniMoEBlock(config).bfloat16().cuda().eval()
    x = x[None]
    for call in (layer.decode, block):
        with fw.dual_level(), torch.no_grad():
            call(x)
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(fw.make_dual(x, torch.ones_like(x)))
    weight = layer.gate_proj.weight
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.functional_call(Decoding(layer), {"layer.gate_proj.weight": fw.make_dual(weight.detach(), torch.ones_like(weight))}, (x,))


class Decoding(torch.nn.Module):
    def __init__(self, layer):
        super().__init__()
        self.layer = layer

    def forward(self, x):
        return self.layer.decode(x)


def test_hooks_of_the_layer_run_whatever_the_number_of_tokens():
    b, = [b.eval() for b in blocks(1)]
    few, many = (torch.randn(1, t, 256, device="cuda").bfloat16() for t in (64, 65))
    seen = []
    with torch.no_grad():
        for register in (lambda: b.layer.register_forward_hook(lambda m, a, y: seen.append(y.shape[1]) or 0 * y),
                         lambda: b.layer.register_forward_pre_hook(lambda m, a: seen.append(a[0].shape[1]) or (0 * a[0],)),
                         lambda: torch.nn.modules.module.register_module_forward_hook(
                             lambda m, a, y: (seen.append(y.shape[1]) or 0 * y) if m is b.layer else None)):
            handle = register()
            seen.clear()
            try:
                outs = [b(x)[0] for x in (few, many)]
            finally:
                handle.remove()
            assert seen == [64, 65] and not any(y.any() for y in outs)
        seen.clear()
        assert b(few)[0].any() and not seen


def test_another_layer_in_the_block():
    """A layer that is wrapped or replaced is called as it is."""
    class Twice(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x):
            return 2 * self.inner(x)

    b, = [b.eval() for b in blocks(1)]
    x = torch.randn(1, 5, 256, device="cuda").bfloat16()
    with torch.no_grad():
        n = b.norm(x).y
        want = 2 * b.layer(n)
        b.layer = Twice(b.layer)
        assert torch.equal(b(x)[0], want)
        b.layer = b.layer.inner
        forward = b.layer.forward
        b.layer.forward = lambda v: 2 * forward(v)   # as wrappers of a module's forward do
        assert torch.equal(b(x)[0], want)


def test_no_routing_of_an_earlier_call_is_left():
    b, = [b.eval() for b in blocks(1)]
    with torch.no_grad():
        b(torch.randn(1, 80, 256, device="cuda").bfloat16())
        assert b.layer.last_routing[1].shape == (80, 8)
        b(torch.randn(1, 5, 256, device="cuda").bfloat16())
        assert b.layer.last_routing is None    # the one kernel keeps its selection to itself
