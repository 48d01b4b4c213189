"""RMS norm with the residual's addition, its 8-bit output and its gradient, and the MX blocks, against 64 bits.

Tolerances.  fp32 sums: a thread adds at most 32 terms in turn, then 5 + 4 levels of a tree: 41 roundings of 2^-24 =
2.4e-6 of the sum of squares, half of it in the root, and two units of the reciprocal root: F = 4e-6 of a value covers
that and the two products after it.  Each rounding to the type costs eps / 2 of the value (and at most half the
smallest subnormal, 2^-25, in fp16).  e4m3 costs 2^-4 of the value, or half a step of 2^-9 scales below 2^-6 scales.
"""
import pytest
import torch

from _util import gen

pytestmark = pytest.mark.gpu

F = 4e-6
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(1, 1), (1, 8), (3, 7), (2, 31), (5, 32), (4, 33), (1, 1024), (7, 1000), (129, 256), (1030, 136), (1025, 4096), (33, 2164),
          (1100, 70), (3, 8192), (2, 16384), (1024, 10000), (2, 16383)]


def half_step(t):
    return torch.finfo(t).eps / 2


def rand(shape, dtype, seed, std=1.0):
    return (torch.randn(*shape, generator=gen(seed)) * std).to(dtype).cuda()


def pow2(e):
    """2^e in 64 bits from the format itself: a library's power may be off in the last place, which moves ties."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def mx_reference(v):
    """Values of the codes and scales (as exponents), from the definition, in 64 bits; finite inputs."""
    v = v.double()
    rows, cols = v.shape
    n = -(-cols // 32)
    b = torch.nn.functional.pad(v, (0, n * 32 - cols)).view(rows, n, 32)
    top = b.abs().amax(2)
    e = torch.ceil(torch.log2(top / 448).clamp(min=-127))
    e = torch.where(top > 448 * pow2(e), e + 1, e)
    e = torch.where((top <= 448 * pow2(e - 1)) & (e > -127), e - 1, e)
    r = b / pow2(e)[..., None]
    step = pow2((torch.frexp(r.abs().clamp(min=2.0 ** -6))[1] - 1) - 3)
    return (torch.round(r / step) * step * pow2(e)[..., None]).view(rows, -1)[:, :cols], e


def exponents(scales):
    return scales.view(torch.uint8).double() - 127


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", SHAPES)
def test_forward(t, n, dtype):
    from omni_moe_b200.ops import mx_dequantize, omni_rms_norm_func
    x, r, w = rand((t, n), dtype, 1), rand((t, n), dtype, 2, 3.0), rand((n,), dtype, 3)
    for residual in (None, r):
        out = omni_rms_norm_func(x, w, residual, eps=1e-5, quantize=True)
        h = x if residual is None else x + r
        assert torch.equal(out.h, h)
        ref = h.double() / torch.sqrt(h.double().square().mean(1, True) + 1e-5) * w.double()
        off = (out.y.double() - ref).abs()
        assert (off <= (half_step(dtype) + F) * ref.abs() + 2 ** -25).all()
        # the scale is the smallest that covers the block, up to the fp32 error of the value at its border
        e = exponents(out.scales)
        pad = torch.nn.functional.pad(ref, (0, -n % 32)).view(t, -1, 32).abs().amax(2)
        assert (pad <= 448 * 2.0 ** e * (1 + F)).all()
        assert ((pad > 224 * 2.0 ** e * (1 - F)) | (e == -127)).all()
        scale = (2.0 ** e).repeat_interleave(32, 1)[:, :n]
        values = mx_dequantize(out.codes, out.scales, torch.float32).double()
        assert ((values - ref).abs() <= torch.maximum(2 ** -4 * ref.abs(), 2 ** -10 * scale) + F * ref.abs()).all()
        plain = omni_rms_norm_func(x, w, residual, eps=1e-5)
        assert plain.codes is None and plain.scales is None and torch.equal(plain.y, out.y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", SHAPES)
def test_gradient(t, n, dtype):
    from omni_moe_b200.ops import omni_rms_norm_func
    x, r, w = rand((t, n), dtype, 1), rand((t, n), dtype, 2, 3.0), rand((n,), dtype, 3)
    dy, dh = rand((t, n), dtype, 4), rand((t, n), dtype, 5)
    for residual in (False, True):
        leaves = [v.requires_grad_() for v in ((x, r, w) if residual else (x, w))]
        out = omni_rms_norm_func(x, w, r if residual else None, eps=1e-5, quantize=residual)
        grads = torch.autograd.grad((out.y, out.h) if residual else out.y, leaves, (dy, dh) if residual else dy)
        h = out.h.detach().double()
        rho = 1 / torch.sqrt(h.square().mean(1, True) + 1e-5)
        nrm, dz = h * rho, dy.double() * w.detach().double()
        m = (dz * nrm).mean(1, True)
        dx = rho * (dz - nrm * m)
        mag = rho * (dz.abs() + nrm.abs() * (dz * nrm).abs().mean(1, True))
        if residual:
            dx = dx + dh.double()
            mag = mag + dh.double().abs()
            assert torch.equal(grads[0], grads[1])
        assert ((grads[0].double() - dx).abs() <= half_step(dtype) * dx.abs() + 2 * F * mag + 2 ** -25).all()
        dw = (dy.double() * nrm).sum(0)
        # at most T / 296 rows in turn, then 296 / 8 + 8 partial rows: fewer than 60 more roundings
        tol = half_step(dtype) * dw.abs() + (F + 60 * 2 ** -24) * (dy.double() * nrm).abs().sum(0) + 2 ** -25
        assert ((grads[-1].double() - dw).abs() <= tol).all()


def test_gradient_against_differences():
    from omni_moe_b200.ops import omni_rms_norm_func
    x, r, w = (rand(s, torch.float32, k) for k, s in enumerate([(5, 72), (5, 72), (72,)]))
    cy, ch = rand((5, 72), torch.float32, 7), rand((5, 72), torch.float32, 8)

    def loss(x, r, w):  # the definition, in 64 bits
        h = x + r
        return (cy.double() * h / torch.sqrt(h.square().mean(1, True) + 1e-6) * w).sum() + (ch.double() * h).sum()

    leaves = [v.requires_grad_() for v in (x, r, w)]
    out = omni_rms_norm_func(x, w, r)
    grads = torch.autograd.grad((out.y * cy).sum() + (out.h * ch).sum(), leaves)
    base = [v.detach().double() for v in leaves]
    for j, g in enumerate(grads):
        d = rand(tuple(g.shape), torch.float64, 20 + j)
        up, down = ([b + s * 1e-4 * d if i == j else b for i, b in enumerate(base)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / 2e-4
        # central differences are off by 1e-8 of the third derivative; h itself was rounded to fp32 (2^-24 a value)
        assert abs(float(slope - (g.double() * d).sum())) <= 1e-5 * float((g.double() * d).abs().sum()) + 1e-5


@pytest.mark.parametrize("w_dtype", [torch.float32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weight_in_float32(dtype, w_dtype):
    from omni_moe_b200.ops import omni_rms_norm_func
    for t, n in ((5, 96), (3, 33)):
        x, w = rand((t, n), dtype, 1).requires_grad_(), rand((n,), w_dtype, 2).requires_grad_()
        y = omni_rms_norm_func(x, w).y
        h = x.detach().double()
        nrm = h / torch.sqrt(h.square().mean(1, True) + 1e-6)
        assert y.dtype == dtype
        assert ((y.double() - nrm * w.double()).abs() <= (half_step(dtype) + F) * (nrm * w.double()).abs() + 2 ** -25).all()
        dx, dw = torch.autograd.grad(y.float().sum(), (x, w))  # an expanded gradient of ones
        assert dx.dtype == dtype and dw.dtype == w_dtype
        assert ((dw.double() - nrm.sum(0)).abs() <= 1e-5 * nrm.abs().sum(0)).all()


def test_only_one_output_used_and_partial_needs():
    from omni_moe_b200.ops import omni_rms_norm_func
    x, r, w = rand((4, 64), torch.float32, 1), rand((4, 64), torch.float32, 2), rand((64,), torch.float32, 3)
    c = rand((4, 64), torch.float32, 4)
    x.requires_grad_()
    out = omni_rms_norm_func(x, w, r)
    assert torch.equal(torch.autograd.grad(out.h, x, c)[0], c)     # the sum alone hands its gradient through
    w.requires_grad_()
    out = omni_rms_norm_func(x, w, r)
    dx, dw = torch.autograd.grad(out.h, (x, w), c, allow_unused=True)
    assert torch.equal(dx, c) and (dw is None or not dw.any())
    full = torch.autograd.grad(omni_rms_norm_func(x, w, r).y, (x, w), c)
    only_w = torch.autograd.grad(omni_rms_norm_func(x.detach(), w, r).y, w, c)[0]
    assert torch.equal(only_w, full[1])
    shared = torch.autograd.grad(omni_rms_norm_func(x, w, x).y, x, c)[0]   # the same tensor twice: both shares
    h = 2 * x.detach()
    single = torch.autograd.grad(omni_rms_norm_func(h.requires_grad_(), w).y, h, c)[0]
    assert torch.equal(shared, 2 * single)


def test_strides_alignment_and_dimensions():
    from omni_moe_b200.ops import omni_rms_norm_func
    x, r, w = rand((6, 128), torch.bfloat16, 1), rand((6, 128), torch.bfloat16, 2), rand((128,), torch.bfloat16, 3)
    want = omni_rms_norm_func(x, w, r, quantize=True)
    wide = torch.zeros(6, 300).bfloat16().cuda()

    def same(a, b):  # the row's values move one by one there: another order of the same sum
        assert torch.equal(a.h, b.h)
        assert ((a.y.double() - b.y.double()).abs() <= (2 * half_step(torch.bfloat16) + 2 * F) * b.y.double().abs()).all()

    wide[:, 5:133] = x
    same(omni_rms_norm_func(wide[:, 5:133], w, r, quantize=True), want)        # odd offset, row stride
    wide[:, 8:136] = x
    got = omni_rms_norm_func(wide[:, 8:136], w, r, quantize=True)              # row stride that is no multiple of 16 bytes
    same(got, want)
    same(omni_rms_norm_func(x, torch.cat((w[:1], w))[1:], r), want)             # weight off its alignment
    t = omni_rms_norm_func(x.t().contiguous().t(), w, r.t().contiguous().t())   # columns first
    assert torch.equal(t.y, want.y)
    b = omni_rms_norm_func(x.view(2, 3, 128), w, r.view(2, 3, 128), quantize=True)
    assert b.y.shape == (2, 3, 128) and b.h.shape == (2, 3, 128) and b.codes.shape == (6, 128) and b.scales.shape == (6, 4)
    assert torch.equal(b.y.view(6, 128), want.y) and torch.equal(b.codes.view(torch.uint8), want.codes.view(torch.uint8))
    v = omni_rms_norm_func(x[0], w)
    assert v.y.shape == (128,)
    one = omni_rms_norm_func(x[:1].expand(6, 128), w)                           # one row seen six times
    assert torch.equal(one.y, v.y.expand(6, 128))
    for shape in ((0, 128), (2, 0, 128)):
        e = omni_rms_norm_func(torch.empty(shape, device="cuda").bfloat16().requires_grad_(), w.clone().requires_grad_(), quantize=True)
        assert e.y.shape == shape and e.scales.shape == (0, 4)
        e.y.sum().backward()


@pytest.mark.parametrize("n,pad", [(256, 8), (512, 4), (96, 32)])
def test_many_rows_with_a_stride(n, pad):
    """The gradient of many rows whose x, dy and dh lie in wider matrices (copied row by row), as of contiguous ones."""
    from omni_moe_b200.ops import omni_rms_norm_func
    t = 2500
    wide = [rand((t, n + pad), torch.bfloat16, k) for k in range(3)]
    w = rand((n,), torch.bfloat16, 5).requires_grad_()

    def grads(x, dy, dh):
        x = x.detach().requires_grad_()
        r = torch.zeros_like(x)
        out = omni_rms_norm_func(x, w, r)
        alone = omni_rms_norm_func(x, w)
        return torch.autograd.grad((out.y, out.h), (x, w), (dy, dh)) + torch.autograd.grad(alone.y, (x, w), dy)

    for a, b in zip(grads(*(v[:, :n] for v in wide)), grads(*(v[:, :n].contiguous() for v in wide))):
        same = (a.double() - b.double()).abs() <= (2 * half_step(torch.bfloat16) + 1e-4) * b.double().abs() + 1e-5 * float(b.double().abs().max())
        assert same.all()   # a stride that is no multiple of 16 bytes takes the other kernel: another order of the sums


def test_rows_of_zeros_and_not_finite_values():
    from omni_moe_b200.ops import mx_dequantize, omni_rms_norm_func
    x = rand((5, 96), torch.float32, 1)
    w = rand((96,), torch.float32, 2)
    clean = omni_rms_norm_func(x, w, quantize=True)
    x[1] = 0
    x[2, 40] = float("nan")
    x[3, 7] = float("inf")
    out = omni_rms_norm_func(x, w, eps=1e-6, quantize=True)
    assert torch.equal(out.y[1], torch.zeros(96, device="cuda")) and torch.isnan(out.y[2]).all()
    assert torch.isnan(out.y[3, 7])                       # inf * 0
    v = mx_dequantize(out.codes, out.scales, torch.float32)
    assert torch.equal(v[1], torch.zeros(96, device="cuda")) and torch.isnan(v[2]).all()
    for row in (0, 4):
        assert torch.equal(out.y[row], clean.y[row]) and torch.equal(out.codes.view(torch.uint8)[row], clean.codes.view(torch.uint8)[row])
    huge = omni_rms_norm_func(torch.full((2, 64), 3e18, device="cuda"), torch.ones(64, device="cuda"))
    assert ((huge.y - 1).abs() < 1e-6).all()              # the sum of squares still fits


def test_streams_and_graphs():
    from omni_moe_b200.ops import omni_rms_norm_func
    x, r, w = rand((300, 512), torch.bfloat16, 1), rand((300, 512), torch.bfloat16, 2), rand((512,), torch.bfloat16, 3)
    dy = rand((300, 512), torch.bfloat16, 4)
    leaves = [v.requires_grad_() for v in (x, r, w)]

    def step():
        out = omni_rms_norm_func(x, w, r, quantize=True)
        grads = torch.autograd.grad(out.y, leaves, dy)
        # detached: torch refuses to capture a backward while an eager graph of the same leaves lives
        return (out.y.detach(), out.h.detach(), out.codes.view(torch.uint8), out.scales.view(torch.uint8)) + grads

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
    for v in cap:
        v.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(cap, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 1000), (64, 4096), (3, 70), (1, 100001), (513, 24)])
def test_mx_blocks_bit_for_bit(t, n, dtype):
    from omni_moe_b200.ops import mx_dequantize, mx_quantize
    x = torch.randn(t, n, generator=gen(n)) * torch.exp(torch.randn(t, 1, generator=gen(t)) * 3)
    x = x.to(dtype).cuda()
    codes, scales = mx_quantize(x)
    assert codes.shape == (t, n) and scales.shape == (t, -(-n // 32))
    ref, e = mx_reference(x)
    assert torch.equal(exponents(scales), e)
    assert torch.equal(mx_dequantize(codes, scales, torch.float32).double(), ref)
    assert torch.equal(mx_dequantize(codes, scales), ref.bfloat16()) and torch.equal(ref.bfloat16().double(), ref)
    assert torch.equal(mx_dequantize(codes, scales, torch.float16), ref.half())
    # torch reads the two formats the same way
    assert torch.equal(codes.float() * scales.float().repeat_interleave(32, 1)[:, :n], ref.float())


def test_mx_borders():
    from omni_moe_b200.ops import mx_dequantize, mx_quantize
    tops = [0.0, 448.0, 448.0 * (1 + 2 ** -23), 447.9999, 896.0, 3.4e38, 2.0 ** -126, 2.0 ** -127, 2.0 ** -149, 1.75, 1.75 * (1 + 2 ** -23), 2.0 ** -118, 448 * 2.0 ** -127]
    x = torch.zeros(len(tops), 32)
    x[:, 0] = torch.tensor(tops)
    x[:, 1] = -x[:, 0]
    x[:, 2:] = x[:, :1] * torch.linspace(-1, 1, 30)
    x = x.cuda()
    codes, scales = mx_quantize(x)
    ref, e = mx_reference(x)
    assert torch.equal(exponents(scales), e)
    # 3.4e38 is 255.8 * 2^120, whose code stands for 256 * 2^120 = 2^128: beyond fp32, so infinite there
    assert torch.equal(mx_dequantize(codes, scales, torch.float32), ref.float())
    assert torch.isinf(ref.float()).any() and float(ref.max()) == 2.0 ** 128
    # every tie between two neighbouring codes goes to the even one: the midpoints of all 126 steps of the format
    grid = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (grid[1:] + grid[:-1]) / 2
    row = torch.cat((mid, torch.tensor([448.0, 0.0]))).view(4, 32)
    row[:, 31] = 448.0
    row = row.cuda()
    assert torch.equal(mx_dequantize(*mx_quantize(row), torch.float32).double(), mx_reference(row)[0])


def test_mx_not_finite_and_empty():
    from omni_moe_b200.ops import mx_dequantize, mx_quantize
    x = rand((3, 64), torch.float32, 1)
    want = mx_dequantize(*mx_quantize(x), torch.float32)
    x[1, 3], x[1, 40], x[2, 63] = float("nan"), float("inf"), float("-inf")
    clean = x.clone()
    clean[~torch.isfinite(x)] = 0
    got, ref = mx_dequantize(*mx_quantize(x), torch.float32), mx_reference(clean)[0].float()
    bad = ~torch.isfinite(x)
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], ref[~bad]) and torch.equal(got[0], want[0])
    c, s = mx_quantize(x[:0])
    assert c.shape == (0, 64) and s.shape == (0, 2) and mx_dequantize(c, s).shape == (0, 64)
    c, s = mx_quantize(x[:, 1:40])                                          # a view with a row stride, off alignment
    assert torch.equal(mx_dequantize(c, s, torch.float32)[0].double(), mx_reference(x[:1, 1:40])[0][0])
    c, s = mx_quantize(x[:1].t())                                            # a column
    assert c.shape == (64, 1)


def test_refusals():
    from omni_moe_b200.ops import mx_dequantize, mx_quantize, omni_rms_norm_func
    x, w = rand((4, 64), torch.bfloat16, 1), rand((64,), torch.bfloat16, 2)
    with pytest.raises(ValueError, match="last dimension"):
        omni_rms_norm_func(torch.zeros(1, 16385, device="cuda"), torch.zeros(16385, device="cuda"))
    with pytest.raises(ValueError, match="weight must be"):
        omni_rms_norm_func(x, w[:63])
    with pytest.raises(TypeError, match="weight"):
        omni_rms_norm_func(x, w.half())
    with pytest.raises(TypeError, match="dtype"):
        omni_rms_norm_func(x.double(), w.double())
    with pytest.raises(ValueError, match="residual"):
        omni_rms_norm_func(x, w, x[:3])
    with pytest.raises(ValueError, match="residual"):
        omni_rms_norm_func(x, w, x.float())
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            omni_rms_norm_func(x, w, eps=eps)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        omni_rms_norm_func(x.cpu(), w.cpu())
    with pytest.raises(ValueError, match="matrix"):
        mx_quantize(x[0])
    with pytest.raises(TypeError, match="dtype"):
        mx_quantize(x.double())
    c, s = mx_quantize(x)
    with pytest.raises(ValueError, match="scales of shape"):
        mx_dequantize(c, s[:, :1])
    with pytest.raises(ValueError, match="float8"):
        mx_dequantize(c.view(torch.uint8), s)


@pytest.mark.parametrize("n", [2 ** 31 - 80, 2 ** 31 - 65])
def test_mx_of_the_longest_rows(n):
    """The last block of threads reaches past column 2^31."""
    from omni_moe_b200.ops import mx_dequantize, mx_quantize
    x = torch.zeros(1, n, device="cuda", dtype=torch.bfloat16)
    x[0, -5000:] = rand((5000,), torch.bfloat16, 1)
    codes, scales = mx_quantize(x)
    out = mx_dequantize(codes, scales)
    from_block = (n - 6000) // 32 * 32
    ref, _ = mx_reference(x[:, from_block:])
    assert torch.equal(out[:, from_block:].double(), ref)
    assert not out[:, :from_block].view(torch.uint8)[:, ::1021].any()
    assert out[0, :8].tolist() == [0.0] * 8


def test_no_second_derivative():
    from omni_moe_b200.ops import omni_rms_norm_func
    x, w = rand((4, 64), torch.float32, 1).requires_grad_(), rand((64,), torch.float32, 2)
    y = omni_rms_norm_func(x, w).y
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(y.square().sum(), x, create_graph=True)


def test_more_values_than_32_bits_count():
    """The last rows of 2^31 values and more: the same bits as on their own."""
    from omni_moe_b200.ops import mx_dequantize, omni_rms_norm_func
    t, n, tail = 2 ** 17 + 9, 16384, 9
    x = torch.zeros(t, n, device="cuda", dtype=torch.bfloat16)
    x[-tail:] = rand((tail, n), torch.bfloat16, 1)
    w = rand((n,), torch.bfloat16, 2).requires_grad_()
    last = x[-tail:].clone().requires_grad_()
    x.requires_grad_()
    dy = torch.zeros_like(x)
    dy[-tail:] = rand((tail, n), torch.bfloat16, 3)
    big, small = omni_rms_norm_func(x, w, quantize=True), omni_rms_norm_func(last, w, quantize=True)
    assert torch.equal(big.y[-tail:], small.y) and not big.y[-tail - 1].any()
    assert torch.equal(mx_dequantize(big.codes, big.scales)[-tail:], mx_dequantize(small.codes, small.scales))
    dx, dw = torch.autograd.grad(big.y, (x, w), dy)
    want, dw_want = torch.autograd.grad(small.y, (last, w), dy[-tail:])
    # (rows of another number go to other threads: the sums of a row are ordered differently)
    assert ((dx[-tail:].double() - want.double()).abs() <= 2 * half_step(torch.bfloat16) * want.double().abs() + 1e-5 * want.double().abs().max()).all()
    assert ((dw.double() - dw_want.double()).abs() <= 2 * half_step(torch.bfloat16) * dw_want.double().abs() + 1e-5 * dw_want.double().abs().max()).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 48, 33])
def test_every_scale_byte(cols, dtype):
    """A scale byte b stands for 2^(b - 127), 255 for NaN: blocks may come from elsewhere than mx_quantize."""
    from omni_moe_b200.ops import mx_dequantize
    b = -(-cols // 32)
    byte = torch.arange(256 * b, device="cuda").view(256, b) % 256
    codes = (torch.arange(256 * cols, device="cuda").view(256, cols) * 37 % 127).to(torch.uint8)  # finite, both kinds of exponent
    got = mx_dequantize(codes.view(torch.float8_e4m3fn), byte.to(torch.uint8).view(torch.float8_e8m0fnu), dtype)
    c = codes.long()
    value = torch.where(c < 8, c.double() / 8, (1 + (c % 8).double() / 8) * pow2((c // 8) - 1)) * 2.0 ** -6  # e4m3, from its definition
    scale = pow2(byte - 127).masked_fill(byte == 255, float("nan")).repeat_interleave(32, 1)[:, :cols]
    want = (value * scale).to(dtype)
    assert torch.equal(got.isnan(), (byte == 255).repeat_interleave(32, 1)[:, :cols])
    assert torch.equal(got.nan_to_num(nan=0.0, posinf=float("inf")), want.nan_to_num(nan=0.0, posinf=float("inf")))


def weight_sum_depth(t, n, dtype):
    """Roundings that a term of the weight's gradient goes through, from the launch's shape: rows of a block in turn, the block's
    row groups, every 32nd block's partial row in turn, and a tree over 32 of those sums."""
    ve = 128 // torch.finfo(dtype).bits
    per = 16 if n % ve == 0 and t >= 1024 else 8
    while 512 * per < n:
        per *= 2
    warps = -(-n // (32 * per))
    rpc = min(t, 8 // warps or 1)
    threads, turns, sms = 32 * warps * rpc, -(-t // rpc), torch.cuda.get_device_properties(0).multi_processor_count
    most = (3 if threads < 256 else max(1, 768 // threads)) * sms
    blocks = min(most, min(turns, sms) if turns // 4 < sms else turns // 4)
    return -(-turns // blocks) + rpc + -(-blocks // 32) + 5, blocks


@pytest.mark.parametrize("t,n,dtype", [(16384, 4096, torch.bfloat16), (16384, 1024, torch.float32), (30001, 136, torch.float16),
                                       (5000, 8192, torch.bfloat16), (20000, 70, torch.bfloat16), (100000, 256, torch.bfloat16), (1, 40, torch.float32)])
def test_weight_gradient_of_many_rows(t, n, dtype):
    from omni_moe_b200.ops import omni_rms_norm_func
    g = torch.Generator("cuda").manual_seed(t + n)
    x, dy, w = (torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((t, n), (t, n), (n,)))
    w.requires_grad_()
    dw, = torch.autograd.grad(omni_rms_norm_func(x, w, eps=1e-5).y, w, dy)
    depth, blocks = weight_sum_depth(t, n, dtype)
    if (t, n) == (16384, 4096):
        assert blocks == 3 * torch.cuda.get_device_properties(0).multi_processor_count  # every block there is, 37 rows in turn
    h = x.double()
    terms = dy.double() * (h / torch.sqrt(h.square().mean(1, True) + 1e-5))
    ref = terms.sum(0)
    tol = half_step(dtype) * ref.abs() + (F + depth * 2 ** -24) * terms.abs().sum(0) * (1 + half_step(dtype)) + 2 ** -25
    assert ((dw.double() - ref).abs() <= tol).all()
