"""The shared MLP with 8-bit activation checkpoints, against its formula in 64 bits.

Tolerances.  A value rounded to bf16 is off by at most 2^-8 of itself.  The gradients go through dact and dgate | dup in
bf16 and come out in bf16: 2^-8 of the result plus 2 * 2^-8 of the sum of magnitudes (worst case, all roundings the same
way), plus 1e-5 of it for fp32 sums and the fast exponential.  A code is off by 2^-4 of the value, or 2^-10 scales.
"""
import pytest
import torch

from _util import gen

pytestmark = pytest.mark.gpu

R = 2 ** -8
SHAPES = [(1, 8, 8), (3, 64, 24), (77, 256, 1024), (130, 264, 200), (256, 512, 64), (300, 72, 136), (515, 1000, 2760), (1024, 1024, 4096),
          (33, 40, 1032)]


def make(t, h, i, seed, dtype=torch.bfloat16):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return [v.to(dtype).cuda() for v in (r(t, h), r(i, h) / h ** 0.5, r(i, h) / h ** 0.5, r(h, i) / i ** 0.5)], (r(t, h) * 0.3).to(dtype).cuda()


def forward(x, wg, wu, limit=0.0):
    from omni_moe_b200 import _lib
    from omni_moe_b200.ops.mx import CODE_DTYPE, SCALE_DTYPE, scale_columns
    t, h = x.shape
    i = wg.size(0)
    act = torch.full((t, i), float("nan"), device="cuda").bfloat16()
    codes = torch.full((t, 2 * i), 0x7f, device="cuda", dtype=torch.uint8).view(CODE_DTYPE)
    scales = torch.full((t, 2 * scale_columns(i)), 255, device="cuda", dtype=torch.uint8).view(SCALE_DTYPE)
    _lib.check(_lib.load().omni_mlp_gate_up_save_mx(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), t, h, i, limit, act.data_ptr(), codes.data_ptr(),
                                                    scales.data_ptr(), _lib.device_status("cuda").data_ptr(), _lib.stream_ptr()))
    _lib.check_device_status()
    return act, codes, scales


def decoded(codes, scales):
    from omni_moe_b200.ops import mx_dequantize
    i, b = codes.size(1) // 2, scales.size(1) // 2
    return [mx_dequantize(codes[:, j * i:(j + 1) * i], scales[:, j * b:(j + 1) * b], torch.float32).double() for j in range(2)]


def derivative(g, u, limit):
    """(act, its slope in g, its slope in u) in 64 bits."""
    gi = g.abs() <= limit if limit else torch.ones_like(g, dtype=torch.bool)
    ui = u.abs() <= limit if limit else torch.ones_like(g, dtype=torch.bool)
    if limit:
        g, u = g.clamp(-limit, limit), u.clamp(-limit, limit)
    s = 1 / (1 + torch.exp(-g))
    return g * s * u, torch.where(gi, u * (s + g * s * (1 - s)), 0.0), torch.where(ui, g * s, 0.0)


@pytest.mark.parametrize("limit", [0.0, 0.8])
@pytest.mark.parametrize("t,h,i", SHAPES)
def test_checkpoint(t, h, i, limit):
    from omni_moe_b200 import _lib
    (x, wg, wu, wd), _ = make(t, h, i, t + h)
    act, codes, scales = forward(x, wg, wu, limit)
    plain = torch.empty_like(act)
    _lib.check(_lib.load().omni_mlp_gate_up_limit(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), t, h, i, limit, plain.data_ptr(), None,
                                                  _lib.device_status("cuda").data_ptr(), _lib.stream_ptr()))
    assert torch.equal(act, plain)       # the output does not depend on what is kept
    b = -(-i // 32)
    for j, (v, w) in enumerate(zip(decoded(codes, scales), (wg, wu))):
        ref, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
        e = scales[:, j * b:(j + 1) * b].contiguous().view(torch.uint8).double() - 127
        scale = torch.exp2(e).repeat_interleave(32, 1)[:, :i]
        assert ((v - ref).abs() <= torch.maximum(2 ** -4 * ref.abs(), 2 ** -10 * scale) + 1e-5 * mag).all()
        top = torch.nn.functional.pad(ref, (0, -i % 32)).view(t, b, 32).abs().amax(2)
        slack = 1e-5 * torch.nn.functional.pad(mag, (0, -i % 32)).view(t, b, 32).amax(2)
        assert (top <= 448 * torch.exp2(e) * (1 + 1e-9) + slack).all()       # covers the block
        assert (top >= 224 * torch.exp2(e) * (1 - 1e-9) - slack).all()       # with the smallest scale


@pytest.mark.parametrize("limit", [0.0, 0.8])
@pytest.mark.parametrize("t,h,i", SHAPES)
def test_gradients_of_given_checkpoints(t, h, i, limit):
    from omni_moe_b200 import _lib
    from omni_moe_b200.ops import mx_dequantize, mx_quantize
    from omni_moe_b200.ops.mlp_ckpt import mlp_ckpt_backward
    (x, wg, wu, wd), dy = make(t, h, i, t + h)
    _, codes, scales = forward(x, wg, wu, limit)
    xq = mx_dequantize(*mx_quantize(x))
    got = mlp_ckpt_backward(dy, xq, codes, scales, wg, wu, wd, limit)
    _lib.check_device_status()
    g, u = decoded(codes, scales)
    act, sg, su = derivative(g, u, limit)
    d = [v.double() for v in (dy, xq, wg, wu, wd)]
    dact, amag = d[0] @ d[4], d[0].abs() @ d[4].abs()
    dg, du, mg, mu = dact * sg, dact * su, amag * sg.abs(), amag * su.abs()
    # what the sums of magnitudes of |dact| (not of its terms) weigh in: a rounding is relative to the value
    rg, ru = dg.abs(), du.abs()
    for a, ref, rounded, terms in (
            (got[0], dg @ d[2] + du @ d[3], rg @ d[2].abs() + ru @ d[3].abs(), mg @ d[2].abs() + mu @ d[3].abs()),
            (got[1], dg.t() @ d[1], rg.t() @ d[1].abs(), mg.t() @ d[1].abs()),
            (got[2], du.t() @ d[1], ru.t() @ d[1].abs(), mu.t() @ d[1].abs()),
            (got[3], d[0].t() @ act, d[0].abs().t() @ act.abs() * 0.5, d[0].abs().t() @ act.abs())):
        assert a.dtype == torch.bfloat16
        off = (a.double() - ref).abs()
        assert (off <= R * ref.abs() + 2.02 * R * rounded + 1e-5 * terms + 1e-9).all(), float((off / (R * ref.abs() + 2 * R * rounded + 1e-9)).max())
        # three roundings in turn (dact, dgate | dup, the result), each of at most R / sqrt(3) in the mean square:
        # R together, where there are many independent ones to average over (t * i values of dact are rounded; with 72
        # of them, a few large ones among them, the sum's worst case of 3 R is in reach and the bound above is what holds)
        if t * i > 10000:
            assert float((a.double() - ref).norm() / ref.norm()) < R


@pytest.mark.parametrize("t,h,i", [(77, 256, 1024), (130, 264, 200), (1, 8, 8)])
@pytest.mark.parametrize("limit", [None, 0.8])
def test_function(t, h, i, limit):
    from omni_moe_b200.ops import mx_dequantize, mx_quantize, omni_mlp_ckpt_func, omni_mlp_func
    from omni_moe_b200.ops.mlp_ckpt import mlp_ckpt_backward
    tensors, dy = make(t, h, i, 5)
    leaves = [v.requires_grad_() for v in tensors]
    x, wg, wu, wd = (v.detach() for v in leaves)
    _, codes, scales = forward(x, wg, wu, limit or 0.0)
    xq = mx_dequantize(*mx_quantize(x))
    want = mlp_ckpt_backward(dy, xq, codes, scales, wg, wu, wd, limit or 0.0)
    exact_x = mlp_ckpt_backward(dy, x, codes, scales, wg, wu, wd, limit or 0.0)
    with torch.no_grad():
        y_plain = omni_mlp_func(x, wg, wu, wd, limit)
        assert torch.equal(omni_mlp_ckpt_func(*leaves, limit=limit), y_plain)
    for kw, ref in ((dict(), want), (dict(x_mx=mx_quantize(x)), want), (dict(keep_x=True), exact_x)):
        y = omni_mlp_ckpt_func(*leaves, limit=limit, **kw)
        assert torch.equal(y, y_plain)
        grads = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(grads, ref))
    for needed in ([0], [1], [2], [3], [0, 3]):   # frozen weights: the gradients asked for are the same
        part = [v.detach().requires_grad_(j in needed) for j, v in enumerate(leaves)]
        grads = torch.autograd.grad(omni_mlp_ckpt_func(*part, limit=limit), [part[j] for j in needed], dy)
        assert all(torch.equal(a, want[j]) for a, j in zip(grads, needed))


def test_gradient_against_differences():
    """The slope of the 64-bit loss along a direction.  The codes move every factor of a gradient term by at most 2^-4
    (x^, g^ and u^, the latter two also through silu', whose relative change is below 2 of theirs here): at most
    (1 + 2^-4)^4 - 1 < 0.28 of the terms' magnitudes, and their signs are independent: 2^-4 of the norm is asked for."""
    from omni_moe_b200.ops import omni_mlp_ckpt_func
    tensors, c = make(64, 128, 256, 3)
    leaves = [v.requires_grad_() for v in tensors]

    def loss(x, wg, wu, wd):
        g = x @ wg.t()
        return ((g / (1 + torch.exp(-g)) * (x @ wu.t()) @ wd.t()) * c.double()).sum()

    grads = torch.autograd.grad(omni_mlp_ckpt_func(*leaves), leaves, c)
    base = [v.detach().double() for v in leaves]
    for j, g in enumerate(grads):
        d = g.double() / g.double().norm()         # along the gradient itself: the slope is its norm
        up, down = ([b + s * 1e-4 * d if i == j else b for i, b in enumerate(base)] for s in (1, -1))
        slope = float(loss(*up) - loss(*down)) / 2e-4
        assert abs(slope - float(g.double().norm())) <= 2 ** -4 * slope


@pytest.mark.parametrize("h,i", [(100, 203), (33, 17), (64, 60)])
def test_sizes_that_are_padded(h, i):
    from omni_moe_b200.ops import mx_quantize, omni_mlp_ckpt_func, omni_mlp_func
    tensors, dy = make(37, h, i, 1)
    leaves = [v.requires_grad_() for v in tensors]
    with torch.no_grad():
        want = omni_mlp_func(*leaves)
        assert torch.equal(omni_mlp_ckpt_func(*leaves), want)
    y = omni_mlp_ckpt_func(*leaves)
    assert torch.equal(y, want)
    a = torch.autograd.grad(y, leaves, dy)
    b = torch.autograd.grad(omni_mlp_ckpt_func(*leaves, x_mx=mx_quantize(leaves[0])), leaves, dy)
    full = torch.autograd.grad(omni_mlp_func(*leaves), leaves, dy)
    for p, q, r, v in zip(a, b, full, leaves):
        assert p.shape == v.shape and torch.equal(p, q)
        assert float((p.double() - r.double()).norm() / r.double().norm()) < 2 ** -4


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_other_types(dtype):
    from omni_moe_b200.ops import omni_mlp_ckpt_func
    tensors, dy = make(20, 64, 96, 2)
    leaves = [v.requires_grad_() for v in tensors]
    other = [v.detach().to(dtype).requires_grad_() for v in leaves]
    want, got = omni_mlp_ckpt_func(*leaves), omni_mlp_ckpt_func(*other)
    assert got.dtype == dtype and torch.equal(got, want.to(dtype))
    for a, b in zip(torch.autograd.grad(got, other, dy.to(dtype)), torch.autograd.grad(want, leaves, dy)):
        assert a.dtype == dtype and torch.equal(a, b.to(dtype))


def test_without_operands_in_place(monkeypatch):
    from omni_moe_b200.ops import omni_mlp_ckpt_func
    tensors, dy = make(72, 128, 96, 2)
    leaves = [v.requires_grad_() for v in tensors]
    want = torch.autograd.grad(omni_mlp_ckpt_func(*leaves), leaves, dy)
    monkeypatch.setenv("OMNI_MOE_B200_MLP_BWD", "copies")
    got = torch.autograd.grad(omni_mlp_ckpt_func(*leaves), leaves, dy)
    for a, b in zip(got, want):  # other kernels, the same roundings: both within the bound of the formula
        assert float((a.double() - b.double()).norm() / b.double().norm()) < R


def test_memory_kept_for_the_backward():
    from omni_moe_b200.ops import omni_mlp_ckpt_func, omni_mlp_func
    tensors, dy = make(512, 256, 1024, 2)
    leaves = [v.requires_grad_() for v in tensors]

    def kept(f):
        torch.cuda.synchronize()
        x = leaves[0].detach().clone().requires_grad_()
        before = torch.cuda.memory_allocated()
        y = f(x, *leaves[1:])
        del x
        after = torch.cuda.memory_allocated()
        del y
        return after - before - 512 * 256 * 2   # the output

    eight, full = kept(omni_mlp_ckpt_func), kept(omni_mlp_func)
    values = 512 * (2 * 1024 + 256)
    assert full >= 2 * 512 * 2 * 1024 and eight + 512 * 256 * 2 <= 1.04 * values + 512 * 256 * 2 + 4096


def test_empty_streams_and_graphs():
    from omni_moe_b200.ops import omni_mlp_ckpt_func
    tensors, dy = make(200, 256, 512, 2)
    leaves = [v.requires_grad_() for v in tensors]
    y = omni_mlp_ckpt_func(leaves[0][:0], *leaves[1:])
    assert y.shape == (0, 256)
    assert not any(g.any() for g in torch.autograd.grad(y.sum(), leaves[1:]))
    del y  # torch refuses to capture a backward while an eager graph of the same leaves lives

    def step():
        y = omni_mlp_ckpt_func(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cap = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(cap, want))


def test_refusals():
    from omni_moe_b200.ops import mx_quantize, omni_mlp_ckpt_func
    (x, wg, wu, wd), _ = make(8, 64, 96, 2)
    for args, kw, what in (((x[0], wg, wu, wd), {}, "matrices"), ((x, wg, wu[:95], wd), {}, "intermediate"), ((x, wg, wu, wd.t()), {}, "intermediate"),
                           ((x, wg, wu, wd), dict(limit=0.0), "limit"), ((x, wg, wu, wd), dict(limit=float("nan")), "limit"),
                           ((x, wg, wu, wd), dict(x_mx=mx_quantize(x[:7])), "blocks of x"),
                           ((x, wg, wu, wd), dict(x_mx=mx_quantize(x), keep_x=True), "exclude"),
                           ((x, wg, wu, wd), dict(x_mx=(x, x)), "float8")):
        with pytest.raises(ValueError, match=what):
            omni_mlp_ckpt_func(*args, **kw)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        omni_mlp_ckpt_func(x.cpu(), wg, wu, wd)


@pytest.mark.parametrize("way", ["", "copies"])
def test_operands_off_alignment(way, monkeypatch):
    """Contiguous tensors that start between 16-byte boundaries, such as views into one flat buffer of parameters."""
    from omni_moe_b200.ops import omni_mlp_ckpt_func
    tensors, dy = make(40, 64, 96, 2)
    leaves = [v.requires_grad_() for v in tensors]
    if way:
        monkeypatch.setenv("OMNI_MOE_B200_MLP_BWD", way)

    def off(v):
        return torch.cat((v.new_zeros(3), v.detach().flatten()))[3:].view(v.shape)

    want = omni_mlp_ckpt_func(*leaves)
    want_grads = torch.autograd.grad(want, leaves, dy)
    moved = [off(v).requires_grad_() for v in leaves]
    assert all(v.data_ptr() % 16 for v in moved)
    got = omni_mlp_ckpt_func(*moved)
    assert torch.equal(got, want)
    with torch.no_grad():
        assert torch.equal(omni_mlp_ckpt_func(*moved), want)
    for a, b in zip(torch.autograd.grad(got, moved, off(dy)), want_grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("way", ["", "copies"])
def test_no_second_derivative(way, monkeypatch):
    from omni_moe_b200.ops import omni_mlp_ckpt_func
    tensors, _ = make(8, 64, 96, 2)
    leaves = [v.requires_grad_() for v in tensors]
    if way:
        monkeypatch.setenv("OMNI_MOE_B200_MLP_BWD", way)
    y = omni_mlp_ckpt_func(*leaves)
    with pytest.raises(RuntimeError, match="no second derivative|once_differentiable"):
        (dx,) = torch.autograd.grad(y.square().sum(), leaves[0], create_graph=True)
        dx.sum().backward()


def test_more_values_than_32_bits_count():
    """The last rows of 2^32 codes and more: the same bits as on their own (no sum runs over rows in what is compared)."""
    from omni_moe_b200.ops import omni_mlp_ckpt_func
    t, h, i, tail = 2 ** 17 + 5, 64, 2 ** 14 + 8, 5
    tensors, _ = make(tail, h, i, 4)
    last = tensors[0].clone().requires_grad_()
    x = torch.zeros(t, h, device="cuda", dtype=torch.bfloat16)
    x[-tail:] = tensors[0]
    x.requires_grad_()
    dy = torch.zeros_like(x)
    dy[-tail:] = 1
    big, small = omni_mlp_ckpt_func(x, *tensors[1:]), omni_mlp_ckpt_func(last, *tensors[1:])
    assert torch.equal(big[-tail:], small) and not big[:-tail].any()
    (dx,), (want,) = torch.autograd.grad(big, x, dy), torch.autograd.grad(small, last, dy[-tail:])
    assert torch.equal(dx[-tail:], want) and not dx[:-tail].any()


@pytest.mark.parametrize("limit", [0.0, 0.8])
@pytest.mark.parametrize("i", [128, 96, 40])   # scales read as one word, byte by byte, and with a block that ends early
def test_scale_that_is_no_number(i, limit):
    """Scale byte 255 stands for NaN: the block's gradients and activation are NaN, all others stay."""
    from omni_moe_b200 import _lib
    (x, wg, wu, wd), dy = make(5, 64, i, 4)
    _, codes, scales = forward(x, wg, wu, limit)
    b = -(-i // 32)

    def start(scales):
        dgu, act = (torch.empty(5, c, device="cuda", dtype=torch.bfloat16) for c in (2 * i, i))
        _lib.check(_lib.load().omni_mlp_dact_swiglu_mx(dy.data_ptr(), wd.data_ptr(), 5, 64, i, codes.data_ptr(), scales.data_ptr(), limit,
                                                       dgu.data_ptr(), act.data_ptr(), _lib.device_status("cuda").data_ptr(), _lib.stream_ptr()))
        _lib.check_device_status()
        return dgu[:, :i], dgu[:, i:], act

    clean = start(scales)
    bad = scales.view(torch.uint8).clone()
    bad[1, b - 1] = 255       # the last block of the gate's row 1
    bad[3, b] = 255           # the first block of the up's row 3
    gate, up = (torch.zeros(5, i, device="cuda", dtype=torch.bool) for _ in range(2))
    gate[1, 32 * (b - 1):] = True
    up[3, :32] = True
    # a gate beyond the clamp passes no gradient, whatever up is, and the other way round; dup does not depend on up's value,
    # but whether it is cut off does (for NaN it is not)
    within = [v.abs() <= limit if limit else torch.ones_like(up) for v in decoded(codes, scales)]
    cut = up & ~within[1]
    for got, was, nan, same in zip(start(bad), clean, (gate | (up & within[0]), gate & within[1], gate | up), (torch.ones_like(cut), ~cut, torch.ones_like(cut))):
        assert torch.isfinite(was).all()
        assert got[nan].isnan().all() and torch.isfinite(got[~nan]).all() and torch.equal(got[~nan & same], was[~nan & same])


@pytest.mark.parametrize("t,h,i", [(77, 256, 1024), (256, 512, 64), (515, 1000, 2760), (1024, 1024, 4096)])
def test_gradients_round_twice(t, h, i):
    """The activation's gradient stays in fp32 on its way to dgate | dup: a gradient has two roundings to bf16 in it, that of
    dgate | dup (or of the activation) and its own.  Each is at most R of the value, so R of the result and 1.01 R (R, and R of
    R again) of the sum of magnitudes.  In the mean square a rounding is R / sqrt(3) of the value at the start of an octave and
    half of that at its end: 0.425 R over values that spread like sums and products of normal ones, 0.60 R for two and 0.74 R
    for three; between them, 0.66 R is asked for."""
    from omni_moe_b200.ops import mx_dequantize, mx_quantize
    from omni_moe_b200.ops.mlp_ckpt import mlp_ckpt_backward
    (x, wg, wu, wd), dy = make(t, h, i, t + h)
    _, codes, scales = forward(x, wg, wu)
    xq = mx_dequantize(*mx_quantize(x))
    got = mlp_ckpt_backward(dy, xq, codes, scales, wg, wu, wd)
    g, u = decoded(codes, scales)
    act, sg, su = derivative(g, u, 0.0)
    d = [v.double() for v in (dy, xq, wg, wu, wd)]
    dact, amag = d[0] @ d[4], d[0].abs() @ d[4].abs()
    dg, du, mg, mu = dact * sg, dact * su, amag * sg.abs(), amag * su.abs()
    for a, ref, rounded, terms in (
            (got[0], dg @ d[2] + du @ d[3], dg.abs() @ d[2].abs() + du.abs() @ d[3].abs(), mg @ d[2].abs() + mu @ d[3].abs()),
            (got[1], dg.t() @ d[1], dg.abs().t() @ d[1].abs(), mg.t() @ d[1].abs()),
            (got[2], du.t() @ d[1], du.abs().t() @ d[1].abs(), mu.t() @ d[1].abs()),
            (got[3], d[0].t() @ act, d[0].abs().t() @ act.abs(), d[0].abs().t() @ act.abs())):
        off = (a.double() - ref).abs()
        assert (off <= R * ref.abs() + 1.01 * R * rounded + 1e-5 * terms + 1e-9).all()
        assert float(off.norm() / ref.norm()) < 0.66 * R
