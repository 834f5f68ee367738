"""The gated Dense (forward and backward), gradient clipping and 4-bit Dense, as
measurable cases.

Every case is one use of `maxim_amd.ops` on device tensors. `listed()` names
fixed cases, `draw()` more of the same ranges; `prepare` / `run` make and run
one, in plain torch operations or, with `own` set, through the framework's
kernels; `exact` evaluates the definition in 64 bits.

Operators (rows r are tokens or pixels, columns features):
  gated      z = x w^T + b with w [2n][k], its halves (a | c): y = act(a) c; z kept when save is set
  gated_bwd  dx, dw, db from dy and z: dz = (dy c act'(a) | dy act(a)), dx = dz w, dw = dz^T x, db = sum_r dz
  clip       N = sqrt(sum of g^2 over all tensors), and g max_norm / N where N > max_norm, else g, into tensors
             of their own (a training program's other copy of its gradients)
  mx4_round  x as blocks of 32 features with a power of two for a scale and 4-bit elements (1 sign, 2 exponent, 1
             mantissa bit), and back: the values that the codes stand for
  mx4_dense  y = act(X W^T + b) (+ residual), X the 4-bit form of x taken in the call, W a weight held in that form

Keys of a case: type (of activations and weights), rows, k and n (inputs and
outputs of a product; c for mx4_round), planar (features outermost, the
executor's [c][h w] order; otherwise one row per token), pad (extra elements
between rows, as in a slice of a wider buffer), wt (the weight stored [k][2n]),
act, residual, save. For clip: layers of LayerNorm, gated and contracting
Dense with c features and `hidden` between, vec_f32 (the vectors' gradients in
fp32), max_norm.
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_SLOPE = 0.2

# What one drawn case may cost at most: the largest listed cases
_MOST_ELEMENTS = 1 << 25
_MOST_FLOPS = 2.7e11
_MOST_FLOPS_F32 = 1.7e10
_MOST_GRADIENTS = 1 << 27


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "maxim-rs_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from maxim_amd import ops
    return ops


def _gated(name, type, rows, k, n, planar=False, pad=0, wt=False, act="silu", save=False):
    return {"name": name, "op": "gated", "type": type, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad,
            "wt": wt, "act": act, "save": save}


def _gated_bwd(name, type, rows, k, n, planar=False, pad=0, wt=False, act="silu"):
    return {"name": name, "op": "gated_bwd", "type": type, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad,
            "wt": wt, "act": act}


def _clip(name, type, layers, c, hidden, vec_f32=False, max_norm=1.0):
    return {"name": name, "op": "clip", "type": type, "layers": layers, "c": c, "hidden": hidden, "vec_f32": vec_f32,
            "max_norm": max_norm}


def _mx4_round(name, type, rows, c, planar=False, pad=0):
    return {"name": name, "op": "mx4_round", "type": type, "rows": rows, "c": c, "planar": planar, "pad": pad}


def _mx4_dense(name, type, rows, k, n, planar=False, pad=0, act="none", residual=False):
    return {"name": name, "op": "mx4_dense", "type": type, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad,
            "act": act, "residual": residual}


def listed():
    return [
        # serving, one token through the gated product
        _gated("gated_token_bf16_2048x8192_silu", "bf16", 1, 2048, 8192),
        # a training batch, both halves kept for the backward pass
        _gated("gated_rows_bf16_8192_2048x4096_silu", "bf16", 8192, 2048, 4096, save=True),
        # odd sizes throughout, serving
        _gated("gated_rows_f16_1237_1001x777_gelu", "f16", 1237, 1001, 777, act="gelu"),
        # the executor's own order and type in training: 64 channels of 256x256
        _gated("gated_planar_f32_64x64_256_gelu", "f32", 256 * 256, 64, 64, planar=True, act="gelu", save=True),
        # a training batch's backward pass
        _gated_bwd("gated_bwd_rows_bf16_4096_1024x2048_silu", "bf16", 4096, 1024, 2048),
        # few channels and many pixels
        _gated_bwd("gated_bwd_planar_f32_64x64_224x320_sigmoid", "f32", 224 * 320, 64, 64, planar=True, act="sigmoid"),
        # the LayerNorm and Dense layers of one 64-channel block: latency
        _clip("clip_f32_block_64", "f32", 1, 64, 64),
        # a token model's gradients, 403 MB, with the vectors' in fp32
        _clip("clip_bf16_8_layers_2048x4096", "bf16", 8, 2048, 4096, vec_f32=True),
        # a batch of activations
        _mx4_round("mx4_round_bf16_8192x4096", "bf16", 8192, 4096),
        # planes of channels whose last block is a part of one
        _mx4_round("mx4_round_planar_f32_c100_256", "f32", 256 * 256, 100, planar=True),
        # serving, one token with the residual
        _mx4_dense("mx4_dense_token_bf16_4096x4096", "bf16", 1, 4096, 4096, residual=True),
        # serving, a prompt's tokens
        _mx4_dense("mx4_dense_rows_bf16_8192_4096x4096_gelu", "bf16", 8192, 4096, 4096, act="gelu"),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_bwd", "clip", "mx4_round", "mx4_dense", "mx4_dense"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    planar = rng.random() < 0.35
    step = rng.choice([1, 1, 8, 64])
    # slices of wider buffers: aligned to 16 bytes or not
    pad = rng.choice([0, 0, 0, 8, 64, 3])
    if op == "clip":
        layers = rng.randint(1, 8)
        c, hidden = (_log_int(rng, 16, 4096, step) for _ in range(2))
        while layers * (3 * c * hidden + 2 * hidden + 3 * c) > _MOST_GRADIENTS:
            c, hidden = (c + 1) // 2, (hidden + 1) // 2
        return {"op": op, "type": t, "layers": layers, "c": c, "hidden": hidden, "vec_f32": rng.random() < 0.5,
                "max_norm": rng.choice([1.0, 0.1, 1e6])}
    if op == "mx4_round":
        c = _log_int(rng, 8 if step < 64 else 64, 512 if planar else 16384, step)
        most = max(2, min(1 << 19, _MOST_ELEMENTS // c))
        rows = max(1, min(_log_int(rng, 1, most, rng.choice([1, 1, 64]) if planar else 1), _MOST_ELEMENTS // c))
        return {"op": op, "type": t, "rows": rows, "c": c, "planar": planar, "pad": pad}
    hi = 512 if planar else 8192
    k = _log_int(rng, 16 if step < 64 else 64, hi, step)
    n = _log_int(rng, 16 if step < 64 else 64, hi if op == "mx4_dense" else hi // 2, step)
    # twice as many weights, and in the backward pass two products
    times = {"gated": 4.0, "gated_bwd": 8.0, "mx4_dense": 2.0}[op]
    flops = _MOST_FLOPS_F32 if t == "f32" and op != "mx4_dense" else _MOST_FLOPS
    most = min(1 << 18, int(flops / (times * k * n)), _MOST_ELEMENTS // max(k, 2 * n))
    rows = max(1, min(_log_int(rng, 1, max(2, most), rng.choice([1, 1, 64])), most))
    act = rng.choice(["none", "gelu", "gelu_tanh", "silu", "silu", "lrelu", "sigmoid"])
    case = {"op": op, "type": t, "rows": rows, "k": k, "n": n, "planar": planar, "pad": pad, "act": act}
    if op == "mx4_dense":
        return dict(case, residual=rng.random() < 0.5)
    case["wt"] = rng.random() < 0.25
    return dict(case, save=rng.random() < 0.5) if op == "gated" else case


# ---------------------------------------------------------------- inputs


def _matrix(gen, case, cols, std=1.0):
    """[rows][cols] activations, or [cols][rows] in the planar order, in the
    middle of a buffer `pad` elements wider."""
    r, c = (cols, case["rows"]) if case["planar"] else (case["rows"], cols)
    t = torch.randn(r, c + case["pad"], generator=gen, device="cuda") * std
    return t.to(_TYPES[case["type"]])[:, :c]


def _shapes(case):
    """A layer's parameters: LayerNorm's, the gated Dense's, the contracting Dense's."""
    c, h = case["c"], case["hidden"]
    return [(c,), (c,), (2 * h, c), (2 * h,), (c, h), (c,)] * case["layers"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "clip":
        s["grads"] = []
        for i, shape in enumerate(_shapes(case)):
            # gradients' sizes differ from layer to layer
            g = torch.randn(shape, generator=gen, device="cuda") * (0.01 * (1 + i % 5))
            s["grads"].append(g.to(torch.float32 if case["vec_f32"] and len(shape) == 1 else dt))
        s["out"] = [torch.empty_like(g) for g in s["grads"]]
        return s
    if case["op"] == "mx4_round":
        # a residual stream: features of different sizes
        s["x"] = _matrix(gen, case, case["c"])
        size = torch.exp(torch.randn(case["c"], generator=gen, device="cuda"))
        s["x"] *= (size[:, None] if case["planar"] else size[None, :]).to(dt)
        return s
    k, n = case["k"], case["n"]
    s["x"] = _matrix(gen, case, k)
    # weights of variance 1 / k, as trained and initialised ones are
    outs = n if case["op"] == "mx4_dense" else 2 * n
    w = torch.randn(outs, k, generator=gen, device="cuda") / math.sqrt(k)
    w = w.t().contiguous().to(dt).t() if case.get("wt") else w.to(dt)
    if case["op"] == "gated_bwd":
        s["w"] = w
        s["dy"] = _matrix(gen, case, n)
        s["z"] = _matrix(gen, case, 2 * n)
        return s
    s["bias"] = (torch.randn(outs, generator=gen, device="cuda") * 0.2).to(dt)
    if case["op"] == "gated":
        s["w"] = w
        return s
    s["residual"] = _matrix(gen, case, n) if case["residual"] else None
    # the weight as a serving program holds it
    if own:
        s["wq"] = _ops().mx4_quantize(w)
    else:
        s["codes"], s["scales"] = _mx4(w.float())
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
    if act == "lrelu":
        return torch.where(z >= 0, 1.0, _SLOPE)
    return torch.ones_like(z)


def _mx4(x):
    """Rows of fp32 values as 4-bit codes, one a byte ([rows][blocks][32], the
    sign in bit 3), and scales (2^e each, [rows][blocks])."""
    r, k = x.shape
    blocks = (k + 31) // 32
    v = torch.zeros(r, blocks * 32, device=x.device)
    v[:, :k] = x
    v = v.view(r, blocks, 32)
    # the largest magnitude's exponent, 2 less: frexp's mantissa is below 1
    e = torch.frexp(v.abs().amax(2)).exponent - 3
    e = torch.where(v.abs().amax(2) == 0, -127, e).clamp(min=-127)
    scale = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    m = torch.ldexp(v, -e.unsqueeze(2)).abs()
    # halfway values go to the even code
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    return code + 8 * torch.signbit(v), scale


def _mx4_values(codes, scales, k):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = table[codes.long()] * scales.unsqueeze(2)
    return v.view(codes.shape[0], -1)[:, :k]


def _run_own(s):
    case, ops = s["case"], _ops()
    if case["op"] == "clip":
        return ops.clip_grads(s["grads"], case["max_norm"], out=s["out"]), s["out"]
    planar = case["planar"]
    if case["op"] == "mx4_round":
        return ops.mx4_dequantize(ops.mx4_quantize(s["x"], planar=planar), planar=planar)
    act = None if case["act"] == "none" else case["act"]
    if case["op"] == "gated":
        return ops.gated(s["x"], s["w"], s["bias"], act=act, slope=_SLOPE, planar=planar, save=case["save"])
    if case["op"] == "gated_bwd":
        return ops.gated_backward(s["dy"], s["x"], s["w"], s["z"], act=act, slope=_SLOPE, planar=planar)
    return ops.mx4_dense(s["x"], s["wq"], s["bias"], act=act, slope=_SLOPE, residual=s["residual"], planar=planar)


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    dt = _TYPES[case["type"]]
    if case["op"] == "clip":
        # 64 bits for the norm: a sum of up to 2^28 squares
        norm = torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt().float()
        factor = torch.where(norm > case["max_norm"], case["max_norm"] / norm, 1.0)
        return norm, [o.copy_((g.float() * factor).to(g.dtype)) for g, o in zip(state["grads"], state["out"])]
    planar = case["planar"]
    dim = 0 if planar else 1  # the features'
    along = (lambda v: v.unsqueeze(1)) if planar else (lambda v: v.unsqueeze(0))
    x = state["x"].float()
    if case["op"] == "mx4_round":
        y = _mx4_values(*_mx4(x.t() if planar else x), case["c"])
        return (y.t() if planar else y).to(dt).contiguous()
    if case["op"] == "mx4_dense":
        w = _mx4_values(state["codes"], state["scales"], case["k"])
        x = _mx4_values(*_mx4(x.t() if planar else x), case["k"])
        y = _act((w @ x.t() if planar else x @ w.t()) + along(state["bias"].float()), case["act"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return y.to(dt)
    w, n = state["w"].float(), case["n"]
    if case["op"] == "gated":
        z = (w @ x if planar else x @ w.t()) + along(state["bias"].float())
        y = _act(z.narrow(dim, 0, n), case["act"]) * z.narrow(dim, n, n)
        return (y.to(dt), z.to(dt)) if case["save"] else y.to(dt)
    dy, z = state["dy"].float(), state["z"].float()
    a, c = z.narrow(dim, 0, n), z.narrow(dim, n, n)
    dz = torch.cat([dy * c * _act_grad(a, case["act"]), dy * _act(a, case["act"])], dim)
    dx = w.t() @ dz if planar else dz @ w
    dw = dz @ x.t() if planar else dz.t() @ x
    return dx.to(dt), dw.to(dt), dz.sum(1 - dim).to(dt)


# ----------------------------------------------------------------- 64 bits


def _act64(z, act):
    """The activation's value and derivative."""
    if act == "gelu":
        p, d = 0.5 * torch.special.erfc(-z / math.sqrt(2.0)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * p, p + z * d
    if act == "gelu_tanh":
        # tanh(u) = 2 sigmoid(2 u) - 1
        s = torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
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


def _mx4_64(x):
    """Rows of values to the nearest that 4-bit blocks hold, in 64 bits."""
    r, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(r, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    # a float's exponent, from its own bits; zero and the smallest go to -127
    e = ((top.view(torch.int64) >> 52) - 1025).clamp(min=-127)
    scale = ((e + 1023) << 52).view(torch.float64)
    m = (v / scale).abs().clamp(max=6.0)
    # steps of a half below 2, of 1 below 4, of 2 up to 6; round() takes halves to even
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).double()
    return (torch.copysign((m / step).round() * step, v) * scale).view(r, -1)[:, :k].contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        flat = [g.double().flatten() for g in s["grads"]]
        norm = sum(g @ g for g in flat) ** 0.5
        scale = min(1.0, case["max_norm"] / float(norm))
        return norm, [(g * scale).view(o.shape) for g, o in zip(flat, s["out"])]
    # token-major, whatever the case's order
    rows = (lambda t: t.double().t().contiguous()) if case["planar"] else (lambda t: t.double().contiguous())
    back = (lambda t: t.t().contiguous()) if case["planar"] else (lambda t: t)
    x = rows(s["x"])
    if case["op"] == "mx4_round":
        return back(_mx4_64(x))
    if case["op"] == "mx4_dense":
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        _matrix(gen, case, case["k"])
        w = (torch.randn(case["n"], case["k"], generator=gen, device="cuda") / math.sqrt(case["k"])).to(_TYPES[case["type"]])
        y = _act64(torch.addmm(s["bias"].double(), _mx4_64(x), _mx4_64(w).t()), case["act"])[0]
        return back(y if s["residual"] is None else y + rows(s["residual"]))
    w, n = s["w"].double().contiguous(), case["n"]
    if case["op"] == "gated":
        z = torch.addmm(s["bias"].double(), x, w.t())
        y = _act64(z[:, :n], case["act"])[0] * z[:, n:]
        return (back(y), back(z)) if case["save"] else back(y)
    z, dy = rows(s["z"]), rows(s["dy"])
    value, slope = _act64(z[:, :n], case["act"])
    dz = torch.empty_like(z)
    torch.mul(dy * slope, z[:, n:], out=dz[:, :n])
    torch.mul(dy, value, out=dz[:, n:])
    return back(dz @ w), dz.t() @ x, dz.sum(0)


def work(case):
    e = _SIZE[case["type"]]
    if case["op"] == "clip":
        n = sum(math.prod(t) * (4 if case["vec_f32"] and len(t) == 1 else e) for t in _shapes(case))
        return {"bytes": 2 * n + 4, "flops": 3 * sum(math.prod(t) for t in _shapes(case))}
    r = case["rows"]
    if case["op"] == "mx4_round":
        return {"bytes": 2 * r * case["c"] * e, "flops": 4 * r * case["c"]}
    k, n = case["k"], case["n"]
    if case["op"] == "mx4_dense":
        held = n * ((k + 31) // 32) * 17
        return {"bytes": (r * k + n + r * n * (1 + case["residual"])) * e + held, "flops": 2 * r * n * k}
    if case["op"] == "gated":
        return {"bytes": (r * k + 2 * n * k + 2 * n + r * n * (3 if case["save"] else 1)) * e, "flops": 4 * r * n * k}
    return {"bytes": (2 * r * k + 4 * n * k + 2 * n + 3 * r * n) * e, "flops": 8 * r * n * k}
