"""The few-token layer kernel (omni_decode) against the layer's definition in 64 bits.

Tolerance.  The kernel's roundings: the activation to bf16 (at most 2^-8 of each value, which the down projection sums
up: 2^-8 * sum |act| |Wd|), the output to bf16 (2^-8 of the value), and fp32 sums and special functions (1e-5 of the sum
of magnitudes covers 16384 terms and the fast exponential).  The bound is evaluated per element in 64 bits.
Rows whose k-th and (k+1)-th scores are nearer than 1e-5 are left out: fp32 may rank them the other way.
"""
import pytest
import torch

from _util import gen

pytestmark = pytest.mark.gpu


def make(t, h, i, n, k, seed, table_std=1.0, extra_rows=0):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    p = dict(x=r(t, h), wg=r(i, h) / h ** 0.5, wu=r(i, h) / h ** 0.5, wd=r(h, i) / i ** 0.5, kx=r(n, h) / h ** 0.5,
             ky=r(n, h) / h ** 0.5, up=r(n * n + extra_rows, h) * table_std, down=r(n * n + extra_rows, h) * table_std)
    p = {a: v.bfloat16().cuda() for a, v in p.items()}
    p["scale"] = (torch.rand(2 * n, generator=g) + 0.5).cuda()
    p["shift"] = (r(2 * n) * 0.3).cuda()
    p["k"] = k
    return p


def call(p, **kw):
    from omni_moe_b200.ops import omni_decode_func
    a = {**p, **kw}
    return omni_decode_func(a["x"], a["wg"], a["wu"], a["wd"], a["kx"], a["ky"], a["up"], a["down"], a["k"], a["scale"], a["shift"])


def reference(p):
    """(y, bound, rows whose selection is clear) in 64 bits."""
    d = {a: v.double() for a, v in p.items() if torch.is_tensor(v) and a not in ("up", "down")}
    x, k, n = d["x"], p["k"], p["kx"].size(0)
    g, u = x @ d["wg"].t(), x @ d["wu"].t()
    act = g / (1 + torch.exp(-g)) * u
    y = act @ d["wd"].t()
    mag = act.abs() @ d["wd"].abs().t()
    z = torch.cat((x @ d["kx"].t(), x @ d["ky"].t()), 1)
    if p["scale"] is not None:
        z = z * d["scale"] + d["shift"]
    lx, ly = torch.log_softmax(z[:, :n], 1), torch.log_softmax(z[:, n:], 1)
    grid = (lx[:, :, None] + ly[:, None, :]).flatten(1)
    best, at = torch.topk(grid, min(k + 1, n * n), dim=1)
    clear = (best[:, k - 1] - best[:, k] > 1e-5) if n * n > k else torch.ones(len(x), dtype=torch.bool, device="cuda")
    at, w = at[:, :k], best[:, :k].exp()
    rows = p["up"][at].double()
    dot = (rows * x[:, None]).sum(2)
    # a dot product's error, through silu (whose slope is at most 1.1)
    dot_err = 1e-5 * (rows * x[:, None]).abs().sum(2)
    coef = w * dot / (1 + torch.exp(-dot))
    down = p["down"][at].double()
    y = y + (coef[:, :, None] * down).sum(1)
    slack = ((1e-4 * coef.abs() + 1.1 * w * dot_err)[:, :, None] * down.abs()).sum(1)
    return y, 2 ** -8 * y.abs() + (2 ** -8 + 1e-5) * mag + slack + 1e-6, clear


def check(p, y):
    from omni_moe_b200 import _lib
    _lib.check_device_status()
    ref, bound, clear = reference(p)
    assert clear.sum() >= 0.9 * len(clear)
    off = (y.double() - ref).abs()[clear]
    assert torch.isfinite(y.float()).all()
    assert (off <= bound[clear]).all(), f"worst {float((off / bound[clear]).max()):.3g} of the bound"
    # the roundings are independent: together far less than the sum of their magnitudes
    rel = float(off.norm() / ref[clear].norm())
    assert rel < 2 ** -8, rel


@pytest.mark.parametrize("t", [1, 2, 7, 8, 9, 16, 17, 32, 33, 64])
def test_tokens(t):
    p = make(t, 256, 1024, 32, 8, 10 + t)
    check(p, call(p))


@pytest.mark.parametrize("t,h,i,n,k", [
    (1, 8, 8, 1, 1),          # the smallest layer there is
    (3, 8, 16, 2, 4),         # every expert selected
    (5, 24, 40, 5, 25),       # every expert of a larger grid, fewer output groups than blocks
    (1, 1024, 4096, 64, 16),
    (13, 1000, 2760, 100, 10),
    (2, 2048, 5632, 256, 16),
    (4, 520, 136, 300, 50),   # router rows cross from one axis to the other inside a block's range
    (6, 64, 64, 1024, 64),
    (64, 136, 264, 17, 128),
    (31, 4096, 1408, 128, 33),
    (40, 600, 3000, 65, 31),
    (1, 16384, 64, 8, 8),
    (33, 16384, 72, 9, 7),
])
def test_shapes(t, h, i, n, k):
    p = make(t, h, i, n, k, t + h + i, table_std=0.3)
    check(p, call(p))


def test_without_batchnorm_and_more_rows_than_the_grid():
    p = make(5, 128, 256, 16, 8, 3, extra_rows=11)
    p["scale"] = p["shift"] = None
    check(p, call(p))


@pytest.mark.parametrize("h,i", [(100, 200), (104, 203), (33, 17)])
def test_sizes_that_are_padded(h, i):
    p = make(4, h, i, 12, 6, h)
    check(p, call(p))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_other_types_are_rounded_to_bf16(dtype):
    p = make(3, 64, 128, 8, 4, 5)
    q = {a: (v.to(dtype) if torch.is_tensor(v) and v.dtype == torch.bfloat16 else v) for a, v in p.items()}
    y = call(q)
    assert y.dtype == dtype
    assert torch.equal(y, call(p).to(dtype))


def test_views_and_strides():
    p = make(6, 128, 256, 16, 8, 9)
    want = call(p)
    wide = torch.randn(6, 300, device="cuda").bfloat16()
    wide[:, 3:131] = p["x"]
    assert torch.equal(call(p, x=wide[:, 3:131]), want)                       # rows with a stride, from an odd offset
    flat = torch.cat((torch.zeros(1, device="cuda").bfloat16(), p["x"].flatten()))[1:].view(6, 128)
    assert flat.data_ptr() % 16 and torch.equal(call(p, x=flat), want)        # contiguous, not 16-byte aligned
    assert torch.equal(call(p, wd=p["wd"].t().contiguous().t()), want)        # a transposed weight
    y = call(p, x=p["x"].expand(6, 128))
    assert torch.equal(y, want) and y.is_contiguous()


def test_no_tokens():
    p = make(1, 64, 64, 4, 2, 1)
    assert call(p, x=p["x"][:0]).shape == (0, 64)


def test_repeats_bit_for_bit_and_leaves_inputs_alone():
    p = make(24, 512, 2048, 64, 16, 4)
    before = {a: v.clone() for a, v in p.items() if torch.is_tensor(v)}
    first = call(p)
    other = make(64, 1024, 512, 200, 40, 5)  # a call of another size uses the same workspace in between
    for _ in range(3):
        call(other)
        assert torch.equal(call(p), first)
    assert all(torch.equal(p[a], v) for a, v in before.items())


def test_streams_and_graphs_do_not_share_scratch():
    p, q = make(8, 512, 2048, 64, 16, 6), make(8, 512, 2048, 64, 16, 7)
    want_p, want_q = call(p), call(q)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):
        for j, v in enumerate((p, q)):
            with torch.cuda.stream(streams[j]):
                got[j] = call(v)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want_p) and torch.equal(got[1], want_q)
    graphs, outs = [], []
    for v in (p, q):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(v))
        graphs.append(g)
    for _ in range(20):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                graphs[j].replay()
        eager = call(p)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want_p) and torch.equal(outs[1], want_q) and torch.equal(eager, want_p)
    p["x"].copy_(q["x"])   # a replay reads the inputs as they are then
    want = call(p)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)


def test_not_finite_tokens_stay_in_their_rows():
    p = make(9, 128, 256, 16, 8, 8)
    want = call(p)
    x = p["x"].clone()
    x[4] = float("nan")
    x[7, 5] = float("inf")
    y = call(p, x=x)
    keep = [0, 1, 2, 3, 5, 6, 8]
    assert torch.equal(y[keep], want[keep])
    assert torch.isnan(y[4].float()).all()
    from omni_moe_b200 import _lib
    try:
        _lib.check_device_status()   # a row of NaN scores may select nothing valid: that is reported, not followed
    except RuntimeError as e:
        assert "expert index" in str(e)


def test_equal_scores_go_to_the_lower_index():
    p = make(3, 64, 64, 8, 5, 2)
    p["kx"].zero_(), p["ky"].zero_()
    p["scale"] = p["shift"] = None
    best = torch.arange(5, device="cuda")                # all scores equal: experts 0..4
    x = p["x"].double()
    dot = x @ p["up"][best].double().t()
    coef = dot / (1 + torch.exp(-dot)) / 64
    act = x @ p["wg"].double().t()
    act = act / (1 + torch.exp(-act)) * (x @ p["wu"].double().t())
    want = act @ p["wd"].double().t() + coef @ p["down"][best].double()
    bound = 2 ** -8 * want.abs() + (2 ** -8 + 1e-4) * (act.abs() @ p["wd"].double().abs().t() + coef.abs() @ p["down"][best].double().abs())
    assert ((call(p).double() - want).abs() <= bound).all()


def test_module_decode_matches_its_forward():
    from omni_moe_b200.modules.omni_moe import OmniMoE, OmniMoEConfig
    torch.manual_seed(0)
    m = OmniMoE(OmniMoEConfig(256, 512, "silu", 1024, 8)).bfloat16().cuda()
    x = torch.randn(2, 11, 256, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="eval"):
        m.decode(x)
    m.eval()
    y, z = m.decode(x), m(x)
    m.check_status()
    assert y.shape == x.shape and y.dtype == x.dtype
    # both paths round the activation and the output to bf16: they differ by less than both errors together
    assert float((y.double() - z.double()).norm() / z.double().norm()) < 2 ** -7
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out = m.decode(x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, y)


def test_refusals():
    p = make(4, 64, 64, 8, 4, 1)
    long = make(65, 64, 64, 8, 4, 1)
    with pytest.raises(ValueError, match="at most 64"):
        call(long)
    for kw, what in ((dict(k=0), "num_experts_per_token"), (dict(k=65), "num_experts_per_token"), (dict(ky=p["ky"][:7]), "router"),
                     (dict(up=p["up"][:60], down=p["down"][:60]), "rows"), (dict(down=p["down"][:63]), "rows"),
                     (dict(wd=p["wd"][:, :56]), "down_weight"), (dict(scale=None), "together"),
                     (dict(scale=p["scale"][:15]), "float32 vectors"), (dict(shift=p["shift"].half()), "float32 vectors"),
                     (dict(x=p["x"][0]), "matrix of tokens")):
        with pytest.raises(ValueError, match=what):
            call(p, **kw)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call(p, x=p["x"].cpu())
    with pytest.raises(RuntimeError, match="no backward"):
        call(p, x=p["x"].clone().requires_grad_())
    check(p, call(p))


@pytest.mark.parametrize("t,h,i,n,k", [
    (9, 4096, 8192, 64, 16),   # the ring form: 16, 32 and 64 token columns
    (16, 4096, 8192, 30, 16),
    (17, 1024, 4096, 64, 16),
    (48, 2048, 8192, 256, 16),
    (20, 64, 20000, 8, 4),     # more than 128 gate / up columns a block
    (64, 128, 40000, 4, 4),
    (18, 8, 8, 3, 2),          # fewer columns than blocks everywhere
    (30, 264, 1000, 1000, 64),  # router rows of both axes in one tile
    (25, 16, 264, 1024, 128),
    (33, 8192, 520, 40, 20),
])
def test_ring_form(t, h, i, n, k):
    p = make(t, h, i, n, k, t + h + i, table_std=0.1)
    check(p, call(p))


@pytest.mark.parametrize("t", [3, 20])
@pytest.mark.parametrize("n,k", [(40, 12), (200, 16), (300, 64), (1024, 64)])
def test_ties_go_to_the_lower_index(t, n, k):
    """Sub-keys that come in equal pairs and fours: whole groups of scores are equal, inside and across the border of
    the k best.  The selection is compared through the output of a layer whose MLP is zero."""
    g = gen(n + t)
    h = 64
    p = make(t, h, 64, n, k, 11, table_std=0.5)
    p["wd"].zero_()
    p["kx"], p["ky"] = p["kx"][torch.arange(n) // 2 * 2], p["ky"][torch.arange(n) // 4 * 4]
    p["scale"] = p["shift"] = None
    x = p["x"].double()
    z = [torch.log_softmax(x @ p[w].double().t(), 1) for w in ("kx", "ky")]
    grid = (z[0][:, :, None] + z[1][:, None, :]).flatten(1)
    # equal rows of a matrix product are equal whatever the summation, so the 64-bit scores tie exactly where fp32's do;
    # a stable descending sort ranks them by index
    # (in 64 bits equal sums of different parts would also be kept apart: nearer than 1e-5 is left to fp32)
    order = torch.sort(grid, dim=1, descending=True, stable=True)
    best, at = order.values[:, :k], order.indices[:, :k]
    gaps = order.values[:, :k] - order.values[:, 1:k + 1]
    clear = ~((gaps > 1e-12) & (gaps < 1e-5)).any(1)
    dot = (p["up"][at].double() * x[:, None]).sum(2)
    coef = best.exp() * dot / (1 + torch.exp(-dot))
    terms = coef[:, :, None] * p["down"][at].double()
    bound = 2 ** -8 * terms.sum(1).abs() + 1e-3 * terms.abs().sum(1) + 1e-7
    assert clear.sum() >= t // 2
    off = (call(p).double() - terms.sum(1)).abs()
    assert (off <= bound)[clear].all()


def layer():
    from omni_moe_b200.modules.omni_moe import OmniMoE, OmniMoEConfig
    torch.manual_seed(0)
    m = OmniMoE(OmniMoEConfig(256, 512, "silu", 1024, 8)).bfloat16().cuda().eval()
    return m, torch.randn(1, 5, 256, device="cuda").bfloat16()


def move_statistics(m, to):
    with torch.no_grad():
        for bn in (m.router_norm_x, m.router_norm_y):
            bn.running_mean.fill_(to)
            bn.running_var.copy_(torch.linspace(0.5, 2.0, bn.running_var.numel()))


def test_capture_before_the_first_call():
    """The BatchNorm fold that a capture computes lives in the graph: calls outside must not read it."""
    m, x = layer()
    other, _ = layer()
    want = other.decode(x)
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out = m.decode(x)
    assert torch.equal(m.decode(x), want)   # before any replay
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_statistics_that_change_between_replays():
    m, x = layer()
    m.decode(x)
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out = m.decode(x)
    for to in (0.25, -0.5):
        move_statistics(m, to)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = m.decode(x)
        again = m.decode(x)      # on another stream than the fold was computed on
        junk = [torch.full((64,), float("nan"), device="cuda") for _ in range(64)]  # would land in memory given back
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, want) and torch.equal(out, want)
        del junk


def test_fold_made_in_inference_mode():
    m, x = layer()
    with torch.inference_mode():
        m.decode(x)
    move_statistics(m, 0.5)
    fresh, _ = layer()
    move_statistics(fresh, 0.5)
    assert torch.equal(m.decode(x), fresh.decode(x))


def test_statistics_that_change_before_a_backward():
    """What an eval-mode graph has kept of the statistics stays as it was when decode() follows new ones."""
    m, x = layer()
    grads = []
    for decode in (False, True):
        move_statistics(m, 0.25)
        leaf = x.clone().requires_grad_()
        y = m(leaf)
        if decode:
            m.decode(x)
            move_statistics(m, -0.5)
            m.decode(x), m(x)
        grads.append(torch.autograd.grad(y.float().square().sum(), leaf)[0])
    assert torch.equal(*grads)


def test_capture_after_the_forward_alone():
    m, x = layer()
    with torch.no_grad():
        m(x)
        want = layer()[0].decode(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m.decode(x)
    move_statistics(m, 0.25)   # the fold that the forward made goes
    m(x)
    changed = m.decode(x)
    junk = [torch.full((64,), float("nan"), device="cuda") for _ in range(64)]
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, changed) and not torch.equal(want, changed)
    del junk


def test_weights_that_require_gradients_are_refused():
    """With gradients enabled a result without a graph would train nothing, in silence."""
    p = make(3, 64, 64, 8, 4, 1)
    want = call(p)
    for name in ("wg", "wu", "wd", "kx", "ky", "up", "down", "scale", "shift"):
        leaf = p[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            call(p, **{name: leaf})
        with torch.no_grad():
            assert torch.equal(call(p, **{name: leaf}), want)
    odd = make(3, 60, 64, 8, 4, 1)   # sizes that are padded first
    with pytest.raises(RuntimeError, match="no backward"):
        call(odd, wg=odd["wg"].clone().requires_grad_())


@pytest.mark.parametrize("t,h,i,n,k", [(3, 256, 1024, 32, 8), (14, 512, 1024, 64, 16), (24, 512, 2048, 64, 16), (64, 1024, 512, 200, 40),
                                       (18, 8, 8, 3, 2), (16, 4096, 8192, 30, 16)])
def test_workspace_of_the_c_entry(t, h, i, n, k):
    """Only the counters at its head need to be zero: whatever else is there is written before it is read."""
    from omni_moe_b200 import _lib
    lib = _lib.load()
    p = make(t, h, i, n, k, 3, table_std=0.1)
    head, size = lib.omni_decode_counter_bytes(), lib.omni_decode_workspace_bytes(t, h, i, n, k)
    assert 0 < head < size and head % 16 == 0
    ws = torch.full((size + 64,), 0xff, device="cuda", dtype=torch.uint8)   # NaN in fp32 and bf16
    ws[:head] = 0
    for _ in range(2):
        y = torch.empty_like(p["x"])
        _lib.check(lib.omni_decode(*(p[a].data_ptr() for a in ("x", "wg", "wu", "wd", "kx", "ky", "up", "down", "scale", "shift")), t, h, i, n, k,
                                   n * n, y.data_ptr(), ws.data_ptr(), size, _lib.device_status("cuda").data_ptr(), _lib.stream_ptr()))
        _lib.check_device_status()
        assert torch.equal(y, call(p))
        assert not ws[:head].any() and (ws[size:] == 0xff).all()
        ws[head:size] = 0xff
