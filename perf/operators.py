"""Cases of the layer's operators for serving and training: the whole layer for a few tokens, the RMS norm with the residual's
addition and an 8-bit output, and the shared MLP whose backward reads 8-bit activation checkpoints.

``run`` computes them in plain torch operations in 32 bits, or, with ``own`` set, through the framework's entry points.
"""
import math
import types

import torch

own = False

BLOCK = 32      # values that share one scale
EPS = 1e-6


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _decode(name, t, h, i, n, k, table_std):
    return {"name": name, "op": "decode", "t": t, "h": h, "i": i, "n": n, "k": k, "table_std": table_std}


def _norm(name, t, h, dtype, residual, quantize, backward):
    return {"name": name, "op": "norm", "t": t, "h": h, "dtype": dtype, "residual": residual, "quantize": quantize,
            "backward": backward}


def _mlp(name, t, h, i, given):
    return {"name": name, "op": "mlp", "t": t, "h": h, "i": i, "given": given}


def listed():
    return [
        # serving: one token through the smallest configuration of the layer
        _decode("decode 1x256", 1, 256, 1024, 32, 8, 1.0),
        # serving: one token through the quick-start configuration
        _decode("decode 1x1024", 1, 1024, 4096, 64, 16, 1.0),
        # serving: an odd batch of requests, sizes that are no multiple of a tile
        _decode("decode 13x1000", 13, 1000, 2760, 100, 10, 0.02),
        # serving: the router and table of the router benchmark, a batch of short drafts
        _decode("decode 64x2048", 64, 2048, 8192, 256, 16, 0.02),
        # serving: the largest configuration (2^20 experts, 64 a token)
        _decode("decode 24x4096", 24, 4096, 11008, 1024, 64, 0.02),
        # serving: the norm in front of the layer for one token
        _norm("norm 1x1024", 1, 1024, "bfloat16", True, False, False),
        # training, forward: the block's input with the 8-bit checkpoint for the MLP
        _norm("norm8 4096x1024", 4096, 1024, "bfloat16", True, True, False),
        # training, forward and backward of odd rows in half precision
        _norm("norm bwd 1023x1000", 1023, 1000, "float16", True, False, True),
        # training, forward and backward at the largest configuration's width
        _norm("norm8 bwd 16384x4096", 16384, 4096, "bfloat16", True, True, True),
        # training step of the shared MLP: a small ragged batch
        _mlp("mlp8 77x256", 77, 256, 1024, False),
        # training step of the shared MLP: the quick-start configuration, the norm's codes at hand
        _mlp("mlp8 4096x1024", 4096, 1024, 4096, True),
        # training step of the shared MLP: the largest configuration's width
        _mlp("mlp8 8192x4096", 8192, 4096, 11008, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "norm", "norm", "mlp"])
    if op == "decode":
        # few tokens; sizes from the smallest configuration to the largest
        t, h, i, n = _log(rng, 1, 64), 8 * _log(rng, 32, 512), 8 * _log(rng, 96, 1376), _log(rng, 24, 1024)
        k = rng.randint(2, min(64, n))
        t = max(1, min(t, int(3.4e9 / (h * (3 * i + 2 * n + 2 * k)))))
        return {"op": op, "t": t, "h": h, "i": i, "n": n, "k": k, "table_std": rng.choice([0.02, 1.0])}
    if op == "norm":
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        return {"op": op, "t": _log(rng, 1, 8192 if dtype == "float32" else 16384), "h": _log(rng, 200, 4096),
                "dtype": dtype, "residual": rng.random() < 0.75,
                "quantize": rng.random() < 0.5, "backward": rng.random() < 0.5}
    return {"op": op, "t": _log(rng, 16, 8192), "h": 8 * _log(rng, 24, 512), "i": 8 * _log(rng, 64, 1376),
            "given": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _linear(gen, rows, cols, dev):
    """A weight as torch.nn.Linear initialises it."""
    return torch.empty((rows, cols), device=dev, dtype=torch.bfloat16).uniform_(-cols ** -0.5, cols ** -0.5, generator=gen)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = types.SimpleNamespace(**case)

    def normal(shape, dtype=torch.bfloat16, std=1.0):
        return torch.empty(shape, device=dev, dtype=dtype).normal_(0.0, std, generator=gen)

    t, h = s.t, s.h
    if s.op == "decode":
        s.x = normal((t, h))
        s.gate, s.up, s.down = _linear(gen, s.i, h, dev), _linear(gen, s.i, h, dev), _linear(gen, h, s.i, dev)
        s.router_x, s.router_y = _linear(gen, s.n, h, dev), _linear(gen, s.n, h, dev)
        s.up_embed, s.down_embed = normal((s.n * s.n, h), std=s.table_std), normal((s.n * s.n, h), std=s.table_std)
        # the router's running statistics, folded into one scale and shift for each logit as a serving program keeps them
        mean = normal((2 * s.n,), torch.float32, 0.1)
        var = torch.empty(2 * s.n, device=dev).uniform_(0.2, 0.5, generator=gen)
        s.bn_scale = torch.rsqrt(var + 1e-5)
        s.bn_shift = -mean * s.bn_scale
    elif s.op == "norm":
        dt = getattr(torch, s.dtype)
        s.x = normal((t, h), dt, 0.5)
        s.res = normal((t, h), dt, 2.0) if s.residual else None
        s.w = (normal((h,), torch.float32, 0.1) + 1).to(dt)
        if s.backward:
            s.dy = normal((t, h), dt, 0.01)
            s.dh = normal((t, h), dt, 0.01) if s.residual else None
            for v in (s.x, s.res, s.w):
                if v is not None:
                    v.requires_grad_(True)
    else:
        s.x = normal((t, h))
        s.gate, s.up, s.down = _linear(gen, s.i, h, dev), _linear(gen, s.i, h, dev), _linear(gen, h, s.i, dev)
        s.dy = normal((t, h), std=0.01)
        s.leaves = (s.x, s.gate, s.up, s.down)
        for v in s.leaves:
            v.requires_grad_(True)
        if s.given:
            # the norm in front of the layer has made these already
            s.codes, s.exponents = _encode(s.x.detach().float())
            s.codes = s.codes.to(torch.float8_e4m3fn)
            s.scales = (s.exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _encode(v):
    """Codes (e4m3 values as floats) and the exponents of the scales: the smallest for which 448 * scale covers the block."""
    rows, cols = v.shape
    blocks = torch.nn.functional.pad(v, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    top = blocks.abs().amax(-1)
    m, e = torch.frexp(top)                      # top = m * 2^e with m in [0.5, 1): 448 = 0.875 * 2^9
    exponent = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-127)
    exponent = torch.where(top == 0, torch.full_like(exponent, -127), exponent)
    codes = torch.ldexp(blocks, -exponent.unsqueeze(-1)).to(torch.float8_e4m3fn).float()
    return codes.reshape(rows, -1)[:, :cols], exponent


def _decoded(v):
    codes, exponent = _encode(v)
    scale = exponent.repeat_interleave(BLOCK, dim=1)[:, :v.shape[1]]
    return torch.ldexp(codes, scale)


def _plain_decode(s):
    x = s.x.float()
    act = x @ s.gate.float().t()
    act = act * torch.sigmoid(act) * (x @ s.up.float().t())
    y = act @ s.down.float().t()
    # values next to the border of the k best: 64 bits
    z = torch.cat((s.x.double() @ s.router_x.double().t(), s.x.double() @ s.router_y.double().t()), 1)
    z = z * s.bn_scale.double() + s.bn_shift.double()
    zx, zy = z[:, :s.n], z[:, s.n:]
    lx = zx - zx.amax(1, True)
    ly = zy - zy.amax(1, True)
    lx = lx - lx.exp().sum(1, True).log()
    ly = ly - ly.exp().sum(1, True).log()
    kk = min(s.n, s.k)
    lx, ix = (v[:, :kk] for v in torch.sort(lx, dim=1, descending=True, stable=True))
    ly, iy = (v[:, :kk] for v in torch.sort(ly, dim=1, descending=True, stable=True))
    score = (lx.unsqueeze(2) + ly.unsqueeze(1)).view(s.t, -1)
    expert = (ix.unsqueeze(2) * s.n + iy.unsqueeze(1)).view(s.t, -1)
    score, at = (v[:, :s.k] for v in torch.sort(score, dim=1, descending=True, stable=True))
    expert = torch.gather(expert, 1, at)
    d = (s.up_embed[expert].float() * x.unsqueeze(1)).sum(2)
    coef = score.exp().float() * d * torch.sigmoid(d)
    y = y + (s.down_embed[expert].float() * coef.unsqueeze(2)).sum(1)
    return y.to(s.x.dtype)


def _plain_norm(s):
    with torch.no_grad():
        h = s.x + s.res if s.residual else s.x
        hf, w = h.float(), s.w.float()
        rho = torch.rsqrt(hf.square().mean(1, True) + EPS)
        y = hf * rho * w
        out = {"y": y.to(s.x.dtype)}
        if s.residual:
            out["h"] = h
        if s.quantize:
            out["values"] = _decoded(y).to(torch.bfloat16)
        if s.backward:
            dy = s.dy.float()
            dz = dy * w
            dx = rho * (dz - hf * rho.square() * (dz * hf).mean(1, True))
            if s.residual:
                dx = dx + s.dh.float()
                out["dres"] = dx.to(s.x.dtype)
            out["dx"] = dx.to(s.x.dtype)
            out["dw"] = (dy * hf * rho).sum(0).to(s.x.dtype)
        return out


def _plain_mlp(s):
    with torch.no_grad():
        x, wg, wu, wd, dy = (v.float() for v in (s.x, s.gate, s.up, s.down, s.dy))
        g, u = x @ wg.t(), x @ wu.t()
        y = (g * torch.sigmoid(g) * u) @ wd.t()
        xq = _decoded(x)
        g, u = _decoded(g), _decoded(u)
        sig = torch.sigmoid(g)
        act = g * sig
        da = dy @ wd
        dg, du = da * u * sig * (1 + g * (1 - sig)), da * act
        dt = s.x.dtype
        return {"y": y.to(dt), "dx": (dg @ wg + du @ wu).to(dt), "dgate": (dg.t() @ xq).to(dt), "dup": (du.t() @ xq).to(dt),
                "ddown": (dy.t() @ (act * u)).to(dt)}


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(s):
    if not own:
        return {"decode": _plain_decode, "norm": _plain_norm, "mlp": _plain_mlp}[s.op](s)
    from omni_moe_b200 import ops
    if s.op == "decode":
        return ops.omni_decode_func(s.x, s.gate, s.up, s.down, s.router_x, s.router_y, s.up_embed, s.down_embed, s.k,
                                    s.bn_scale, s.bn_shift)
    if s.op == "norm":
        got = ops.omni_rms_norm_func(s.x, s.w, residual=s.res, eps=EPS, quantize=s.quantize)
        out = {"y": got.y}
        if s.residual:
            out["h"] = got.h
        if s.quantize:
            out["values"] = ops.mx_dequantize(got.codes, got.scales)
        if s.backward:
            if s.residual:
                out["dx"], out["dres"], out["dw"] = torch.autograd.grad((got.y, got.h), (s.x, s.res, s.w), (s.dy, s.dh))
            else:
                out["dx"], out["dw"] = torch.autograd.grad(got.y, (s.x, s.w), s.dy)
        return out
    y = ops.omni_mlp_ckpt_func(s.x, s.gate, s.up, s.down, x_mx=(s.codes, s.scales) if s.given else None)
    dx, dgate, dup, ddown = torch.autograd.grad(y, s.leaves, s.dy)
    return {"y": y, "dx": dx, "dgate": dgate, "dup": dup, "ddown": ddown}


def work(case):
    t, h = case["t"], case["h"]
    if case["op"] == "decode":
        i, n, k = case["i"], case["n"], case["k"]
        return {"bytes": 2 * (3 * i * h + 2 * n * h + 2 * t * k * h + 2 * t * h), "flops": 2 * t * (3 * i * h + 2 * n * h + 2 * k * h)}
    if case["op"] == "norm":
        e = 4 if case["dtype"] == "float32" else 2
        res, mx, bwd = case["residual"], case["quantize"], case["backward"]
        rows = e * ((4 if res else 2) + (bwd and (5 if res else 3)))      # x, res, y, h; dy, h, dh, dx, dres
        if mx:
            rows += 2 * (1 + 1 / BLOCK) + 2                               # codes written and read, values written
        return {"bytes": t * h * rows + e * h, "flops": t * h * (6 + 10 * bwd)}
    i = case["i"]
    ckpt = (1 + 1 / BLOCK) * t * (2 * i + h)
    return {"bytes": 2 * (4 * t * h + 6 * i * h) + 2 * ckpt, "flops": 18 * t * h * i}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_mx(v):
    """The values that the codes stand for, from the definition: a grid of 3 mantissa bits down to 2^-9, up to 448."""
    rows, cols = v.shape
    out = torch.empty_like(v)
    for b in range(0, cols, BLOCK):
        c = v[:, b:b + BLOCK]
        top = c.abs().max(1, keepdim=True).values
        e = torch.ceil(torch.log2(top / 448).clamp(min=-127))
        e = torch.where(top > 448 * 2.0 ** e, e + 1, e)
        e = torch.where((top <= 448 * 2.0 ** (e - 1)) & (e > -127), e - 1, e)
        r = c / 2.0 ** e
        step = 2.0 ** (torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, b:b + BLOCK] = torch.round(r / step) * step * 2.0 ** e
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    d = lambda v: v.detach().double()  # noqa: E731
    x = d(s.x)
    if s.op == "decode":
        gate, up = torch.einsum("th,ih->ti", x, d(s.gate)), torch.einsum("th,ih->ti", x, d(s.up))
        y = torch.einsum("ti,hi->th", gate / (1 + torch.exp(-gate)) * up, d(s.down))
        rows = []
        for t in range(s.t):
            axis = []
            for a, w in enumerate((s.router_x, s.router_y)):
                z = d(w) @ x[t] * d(s.bn_scale[a * s.n:(a + 1) * s.n]) + d(s.bn_shift[a * s.n:(a + 1) * s.n])
                axis.append(z - torch.logsumexp(z, 0))
            grid = (axis[0][:, None] + axis[1][None, :]).reshape(-1)
            best, at = torch.topk(grid, s.k)
            dot = d(s.up_embed[at]) @ x[t]
            rows.append((best.exp() * dot / (1 + torch.exp(-dot))) @ d(s.down_embed[at]))
        return y + torch.stack(rows)
    if s.op == "norm":
        # the sum is rounded to the type before it is normed, as it is handed on
        h = (x + d(s.res)).to(s.x.dtype).double() if s.residual else x
        w = d(s.w)
        r = 1 / torch.sqrt((h * h).sum(1, keepdim=True) / s.h + EPS)
        out = {"y": h * r * w}
        if s.residual:
            out["h"] = h
        if s.quantize:
            out["values"] = _exact_mx(out["y"])
        if s.backward:
            n, gz = h * r, d(s.dy) * w
            dx = r * (gz - n * (gz * n).sum(1, keepdim=True) / s.h)
            if s.residual:
                dx = dx + d(s.dh)
                out["dres"] = dx
            out["dx"] = dx
            out["dw"] = (d(s.dy) * n).sum(0)
        return out
    wg, wu, wd, dy = d(s.gate), d(s.up), d(s.down), d(s.dy)
    g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    y = torch.matmul(g / (1 + torch.exp(-g)) * u, wd.t())
    g, u, xq = _exact_mx(g), _exact_mx(u), _exact_mx(x)
    p = 1 / (1 + torch.exp(-g))
    a = torch.matmul(dy, wd)
    dg, du = a * u * (p + g * p * (1 - p)), a * g * p
    return {"y": y, "dx": torch.matmul(dg, wg) + torch.matmul(du, wu), "dgate": torch.matmul(dg.t(), xq),
            "dup": torch.matmul(du.t(), xq), "ddown": torch.matmul(dy.t(), g * p * u)}
