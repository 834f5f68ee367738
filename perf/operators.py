"""LayerNorm and Dense, forward and backward, as measurable cases.

Every case is one call of `maxim_amd.ops` on device tensors. `listed()` names
fixed cases, `draw()` more of the same ranges; `prepare` / `run` make and run
one, in plain torch operations or, with `own` set, through the framework's
kernels; `exact` evaluates the definition in 64 bits.

Operators (rows r are tokens or pixels, columns features):
  ln         y = (x - mean) rstd scale + bias; mean and rstd are outputs too
  ln_bwd     dx (+ the residual branch's gradient `add`), dscale, dbias
  dense      y = act(x w^T + b) (+ residual), z = x w^T + b kept when save is set
  dense_bwd  dx, dw, db from dy through act'(z)

Keys of a case: type (of activations and weights), rows, c (LayerNorm's
features) or k and n (Dense's inputs and outputs), planar (features outermost,
the executor's [c][h w] order; otherwise one row per token), pad (extra
elements between rows, as in a slice of a wider buffer), wt (the weight stored
[k][n]), f32_params (scale and bias held in fp32), act, residual, save, add.
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6
_SLOPE = 0.2

# What one drawn case may cost at most: the largest listed cases
_MOST_ELEMENTS = 1 << 25
_MOST_FLOPS = 2.7e11
_MOST_FLOPS_F32 = 3.5e10


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "maxim-rs_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from maxim_amd import ops
    return ops


def _ln(name, type, rows, c, planar=False, pad=0, f32_params=False):
    return {"name": name, "op": "ln", "type": type, "rows": rows, "c": c, "planar": planar, "pad": pad,
            "f32_params": f32_params}


def _ln_bwd(name, type, rows, c, planar=False, pad=0, f32_params=False, add=False):
    return {"name": name, "op": "ln_bwd", "type": type, "rows": rows, "c": c, "planar": planar, "pad": pad,
            "f32_params": f32_params, "add": add}


def _dense(name, type, rows, k, n, planar=False, pad=0, wt=False, act="none", residual=False, save=False):
    return {"name": name, "op": "dense", "type": type, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad,
            "wt": wt, "act": act, "residual": residual, "save": save}


def _dense_bwd(name, type, rows, k, n, planar=False, pad=0, wt=False, act="none"):
    return {"name": name, "op": "dense_bwd", "type": type, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad,
            "wt": wt, "act": act}


def listed():
    return [
        # serving, one token: latency
        _ln("ln_token_bf16_1024", "bf16", 1, 1024, f32_params=True),
        # the executor's own layout: 64 channels of a 640x448 image in training
        _ln("ln_planar_f32_c64_448x640", "f32", 448 * 640, 64, planar=True),
        # a training batch of tokens
        _ln("ln_rows_bf16_8192x4096", "bf16", 8192, 4096),
        # its backward pass, joined with the residual branch's gradient
        _ln_bwd("ln_bwd_rows_bf16_8192x4096", "bf16", 8192, 4096, f32_params=True, add=True),
        # an odd width in the middle of a wider buffer
        _ln_bwd("ln_bwd_rows_f16_1237x777", "f16", 1237, 777, pad=3),
        # the widest image of the executor's 32-channel level
        _ln_bwd("ln_bwd_planar_f32_c32_448x640", "f32", 448 * 640, 32, planar=True),
        # serving, one token through a square projection with the residual
        _dense("dense_token_bf16_4096x4096", "bf16", 1, 4096, 4096, residual=True),
        # the expanding product of a training batch, pre-activation kept
        _dense("dense_rows_bf16_8192_2048x8192_gelu", "bf16", 8192, 2048, 8192, act="gelu", save=True),
        # odd sizes throughout, with the contracting product's residual
        _dense("dense_rows_f16_1237_1001x777", "f16", 1237, 1001, 777, residual=True),
        # the executor's own Dense and GELU: 64 channels to 128 over 256x256
        _dense("dense_planar_f32_64x128_256", "f32", 256 * 256, 64, 128, planar=True, act="gelu", save=True),
        # the expanding product's backward pass
        _dense_bwd("dense_bwd_rows_bf16_4096_1024x4096_gelu", "bf16", 4096, 1024, 4096, act="gelu"),
        # the backward pass of a planar Dense: few channels, many pixels
        _dense_bwd("dense_bwd_planar_f32_128x128_224x320", "f32", 224 * 320, 128, 128, planar=True, act="lrelu"),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(["ln", "ln_bwd", "dense", "dense_bwd"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    planar = rng.random() < 0.35
    step = rng.choice([1, 1, 8, 64])
    # slices of wider buffers: aligned to 16 bytes or not
    pad = rng.choice([0, 0, 0, 8, 64, 3])
    if op in ("ln", "ln_bwd"):
        c = _log_int(rng, 8 if step < 64 else 64, 512 if planar else 16384, step)
        rows = _log_int(rng, 1, max(2, min(1 << 19, _MOST_ELEMENTS // c)), rng.choice([1, 1, 64]) if planar else 1)
        rows = max(1, min(rows, _MOST_ELEMENTS // c))
        if op == "ln":
            return {"op": op, "type": t, "rows": rows, "c": c, "planar": planar, "pad": pad,
                    "f32_params": rng.random() < 0.5}
        return {"op": op, "type": t, "rows": rows, "c": c, "planar": planar, "pad": pad,
                "f32_params": rng.random() < 0.5, "add": rng.random() < 0.5}
    hi = 512 if planar else 8192
    k = _log_int(rng, 16 if step < 64 else 64, hi, step)
    n = _log_int(rng, 16 if step < 64 else 64, hi, step)
    flops = _MOST_FLOPS_F32 if t == "f32" else _MOST_FLOPS
    most = min(1 << 18, int(flops / (4.0 * k * n)), _MOST_ELEMENTS // max(k, n))
    rows = max(1, min(_log_int(rng, 1, max(2, most), rng.choice([1, 1, 64])), most))
    act = rng.choice(["none", "gelu", "gelu_tanh", "silu", "lrelu", "sigmoid"])
    wt = rng.random() < 0.25
    if op == "dense":
        return {"op": op, "type": t, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad, "wt": wt, "act": act,
                "residual": rng.random() < 0.5, "save": rng.random() < 0.5}
    return {"op": op, "type": t, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad, "wt": wt, "act": act}


# ---------------------------------------------------------------- inputs


def _matrix(gen, case, cols, std=1.0, mean=0.0):
    """[rows][cols] activations, or [cols][rows] in the planar order, in the
    middle of a buffer `pad` elements wider."""
    r, c = (cols, case["rows"]) if case["planar"] else (case["rows"], cols)
    t = torch.randn(r, c + case["pad"], generator=gen, device="cuda") * std + mean
    return t.to(_TYPES[case["type"]])[:, :c]


def _vector(gen, n, dtype, std, mean=0.0):
    return (torch.randn(n, generator=gen, device="cuda") * std + mean).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _TYPES[case["type"]]
    s = {"case": case}
    if case["op"] in ("ln", "ln_bwd"):
        c = case["c"]
        pt = torch.float32 if case["f32_params"] else dt
        # a residual stream: of order one, off zero by a few tenths
        s["x"] = _matrix(gen, case, c, 1.5, 0.3)
        s["scale"] = _vector(gen, c, pt, 0.1, 1.0)
        if case["op"] == "ln":
            s["bias"] = _vector(gen, c, pt, 0.1)
        else:
            s["dy"] = _matrix(gen, case, c)
            s["add"] = _matrix(gen, case, c) if case["add"] else None
            # what the forward pass kept
            dim = 0 if case["planar"] else 1
            xf = s["x"].float()
            s["mean"] = xf.mean(dim)
            s["rstd"] = torch.rsqrt((xf - s["mean"].unsqueeze(dim)).square().mean(dim) + _EPS)
        return s
    k, n = case["k"], case["n"]
    s["x"] = _matrix(gen, case, k)
    # weights of variance 1 / k, as trained and initialised ones are
    w = torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)
    s["w"] = (w.t().contiguous().to(dt).t()) if case["wt"] else w.to(dt)
    if case["op"] == "dense":
        s["bias"] = _vector(gen, n, dt, 0.2)
        s["residual"] = _matrix(gen, case, n) if case["residual"] else None
    else:
        s["dy"] = _matrix(gen, case, n)
        s["z"] = _matrix(gen, case, n) if case["act"] != "none" else None
    return s


# ------------------------------------------------------------ plain forms


def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "lrelu":
        return torch.where(z >= 0, z, _SLOPE * z)
    return z


def _act_grad(z, act):
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 - s)
    return torch.where(z >= 0, 1.0, _SLOPE)


def _run_own(s):
    case, ops = s["case"], _ops()
    planar = case["planar"]
    if case["op"] == "ln":
        return ops.layernorm(s["x"], s["scale"], s["bias"], eps=_EPS, planar=planar, stats=True)
    if case["op"] == "ln_bwd":
        return ops.layernorm_backward(s["dy"], s["x"], s["scale"], s["mean"], s["rstd"], add=s["add"], planar=planar)
    act = None if case["act"] == "none" else case["act"]
    if case["op"] == "dense":
        return ops.dense(s["x"], s["w"], s["bias"], act=act, slope=_SLOPE, residual=s["residual"], planar=planar,
                         save=case["save"])
    return ops.dense_backward(s["dy"], s["x"], s["w"], z=s["z"], act=act, slope=_SLOPE, planar=planar)


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    planar = case["planar"]
    dim = 0 if planar else 1  # the features'
    dt = _TYPES[case["type"]]
    along = (lambda v: v.unsqueeze(1)) if planar else (lambda v: v.unsqueeze(0))
    x = state["x"].float()
    if case["op"] == "ln":
        mean = x.mean(dim)
        d = x - mean.unsqueeze(dim)
        rstd = torch.rsqrt((d * d).mean(dim) + _EPS)
        y = d * rstd.unsqueeze(dim) * along(state["scale"].float()) + along(state["bias"].float())
        return y.to(dt), mean, rstd
    if case["op"] == "ln_bwd":
        dy, rstd = state["dy"].float(), state["rstd"].unsqueeze(dim)
        xh = (x - state["mean"].unsqueeze(dim)) * rstd
        g = dy * along(state["scale"].float())
        dx = rstd * (g - g.mean(dim, keepdim=True) - xh * (g * xh).mean(dim, keepdim=True))
        if state["add"] is not None:
            dx = dx + state["add"].float()
        pt = state["scale"].dtype
        return dx.to(dt), (dy * xh).sum(1 - dim).to(pt), dy.sum(1 - dim).to(pt)
    w = state["w"].float()
    if case["op"] == "dense":
        z = (w @ x if planar else x @ w.t()) + along(state["bias"].float())
        y = _act(z, case["act"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return (y.to(dt), z.to(dt)) if case["save"] else y.to(dt)
    dz = state["dy"].float()
    if state["z"] is not None:
        dz = dz * _act_grad(state["z"].float(), case["act"])
    dx = w.t() @ dz if planar else dz @ w
    dw = dz @ x.t() if planar else dz.t() @ x
    return dx.to(dt), dw.to(dt), dz.sum(1 - dim).to(dt)


# ----------------------------------------------------------------- 64 bits


def _phi(z):
    """The normal distribution function, and its density."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _act64(z, act):
    """The activation's value and derivative."""
    if act == "gelu":
        p, d = _phi(z)
        return z * p, p + z * d
    if act == "gelu_tanh":
        # tanh(u) = 2 sigmoid(2 u) - 1
        u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        s = torch.special.expit(u)
        return z * s, s + z * s * torch.special.expit(-u) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    if act == "silu":
        s = torch.special.expit(z)
        return z * s, s + z * s * torch.special.expit(-z)
    if act == "sigmoid":
        s = torch.special.expit(z)
        return s, s * torch.special.expit(-z)
    if act == "lrelu":
        step = (z >= 0).double() * (1 - _SLOPE) + _SLOPE
        return z * step, step
    return z, torch.ones_like(z)


def exact(case, seed):
    s = prepare(case, seed)
    # token-major, whatever the case's order
    rows = (lambda t: t.double().t().contiguous()) if case["planar"] else (lambda t: t.double().contiguous())
    back = (lambda t: t.t().contiguous()) if case["planar"] else (lambda t: t)
    x = rows(s["x"])
    if case["op"] == "ln":
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + _EPS) ** -0.5
        y = torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], s["scale"].double())
        return back(y), mean, rstd
    if case["op"] == "ln_bwd":
        dy, scale, c = rows(s["dy"]), s["scale"].double(), case["c"]
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
        xh = (x - mean) * rstd
        p = (dy @ scale)[:, None] / c
        q = ((dy * xh) @ scale)[:, None] / c
        dx = (dy * scale - p - xh * q) * rstd
        if s["add"] is not None:
            dx += rows(s["add"])
        ones = torch.ones(case["rows"], dtype=torch.float64, device="cuda")
        return back(dx), ones @ (dy * xh), ones @ dy
    w = s["w"].double().contiguous()
    if case["op"] == "dense":
        z = torch.addmm(s["bias"].double(), x, w.t())
        y = _act64(z, case["act"])[0]
        if s["residual"] is not None:
            y = y + rows(s["residual"])
        return (back(y), back(z)) if case["save"] else back(y)
    dz = rows(s["dy"])
    if s["z"] is not None:
        dz = dz * _act64(rows(s["z"]), case["act"])[1]
    return back(dz @ w), dz.t() @ x, dz.sum(0)


def work(case):
    e, r = _SIZE[case["type"]], case["rows"]
    if case["op"] in ("ln", "ln_bwd"):
        c, p = case["c"], 4 if case["f32_params"] else _SIZE[case["type"]]
        if case["op"] == "ln":
            return {"bytes": 2 * r * c * e + 2 * c * p + 8 * r, "flops": 8 * r * c}
        return {"bytes": (3 + case["add"]) * r * c * e + 3 * c * p + 8 * r, "flops": 14 * r * c}
    k, n = case["k"], case["n"]
    if case["op"] == "dense":
        moved = r * k + n * k + n + r * n * (1 + case["residual"] + case["save"])
        return {"bytes": moved * e, "flops": 2 * r * n * k}
    moved = 2 * r * k + 2 * n * k + n + r * n * (2 if case["act"] != "none" else 1)
    return {"bytes": moved * e, "flops": 4 * r * n * k}
