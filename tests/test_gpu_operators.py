"""LayerNorm and Dense on device tensors, forward and backward, against their
formulas in 64 bits on the CPU.

Tolerances, element by element, with u = 2^-24 (fp32's half step), h half a
step of the result's type and S the sum of a result's terms' absolute values:
  a sum of k terms in fp32, in any order: k u S at most (each of k - 1 adds
  rounds once, and fp32 products once more); a result's own rounding: h |y|;
  GELU, SiLU and the logistic function are fits and hardware exponentials
  within 3e-7 (1 + |z|), their derivatives, all below 1.2, within 6e-7 (1 + |z|);
  an error e of z moves act(z) by 1.2 e at most;
  dz is rounded to the products' type where there is an activation: h |dz|
  more, summed against the other operand's absolute values.
A row sum of C terms inside LayerNorm runs over lanes and waves, in chains of
C / 64 terms and a tree at most; (C / 64 + 32) u bounds each, relative to the
mean of the absolute values."""

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = [None, "gelu", "gelu_tanh", "silu", "lrelu", "sigmoid"]
SLOPE = 0.2


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half a step at the bottom of the type's range (fp16 results can be subnormal)."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2 if dt == torch.float16 else 1e-37


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()


def make(seed, rows, cols, dt, planar=False, pad=0, std=1.0, mean=0.0):
    """A device tensor in either order, in the middle of a wider buffer, and
    its values [rows][cols] in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    a, b = (cols, rows) if planar else (rows, cols)
    buf = (torch.randn(a, b + pad, generator=g) * std + mean).to(dt)
    t = buf.cuda()[:, :b]
    v = buf[:, :b].double()
    return t, v.t() if planar else v


def vec(seed, n, dt, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    v = (torch.randn(n, generator=g) * std + mean).to(dt)
    return v.cuda(), v.double()


def values(t, planar=False):
    v = t.double().cpu()
    return v.t() if planar else v


def near(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got - want).abs() - tol
    worst = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or (bool((off <= 0).all())), "%s: off by %.3g where %.3g is allowed (%.6g, expected %.6g)" % (
        what, float((got - want).abs().flatten()[worst]), float(tol.flatten()[worst]), float(got.flatten()[worst]),
        float(want.flatten()[worst]))


# ------------------------------------------------------------- LayerNorm

LN_SHAPES = [(1, 1), (1, 7), (3, 64), (5, 100), (65, 8), (2, 777), (7, 1024), (130, 96), (33, 2048), (3, 5000),
             (2, 8192), (2, 20000), (1, 70001), (257, 33), (1000, 16), (300, 512)]


def ln_reference(x, scale, bias, eps):
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = ((d * d).mean(1) + eps) ** -0.5
    xh = d * rstd[:, None]
    return xh * scale + bias, mean, rstd, xh


def check_layernorm(rows, cols, dt, planar, pad, param_dt, mean=0.3, eps=1e-6, seed=0):
    x, xv = make(seed, rows, cols, dt, planar, pad, 1.5, mean)
    s, sv = vec(seed + 1, cols, param_dt, 0.1, 1.0)
    b, bv = vec(seed + 2, cols, param_dt, 0.1)
    y, m, r = O.layernorm(x, s, b, eps=eps, planar=planar, stats=True)
    want, mw, rw, xh = ln_reference(xv, sv, bv, eps)
    n = cols / 64 + 32
    me = n * U * xv.abs().mean(1)  # the mean's error
    near(m.double().cpu(), mw, me + U * mw.abs(), "mean")
    # the variance is taken about a mean off by me, whose square alone enters;
    # each term d^2 is off by 2 u |d| (|x| + |d|), the sum by n u of itself
    d = (xv - mw[:, None]).abs()
    ve = me ** 2 + ((n + 4) * U * d * d + 2 * U * d * xv.abs()).mean(1)
    var = (d * d).mean(1)
    rel = 0.5 * ve / (var + eps) * 1.01 + 6 * U
    near(r.double().cpu(), rw, rw * rel, "rstd")
    err = (rw[:, None] * (me[:, None] + U * xv.abs()) + xh.abs() * (rel[:, None] + 4 * U)) * sv.abs()
    tol = err + 2 * U * (want.abs() + bv.abs()) + half(dt) * (want.abs() + err) + tiny(dt)
    near(values(y, planar), want, tol, "y")


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,cols", LN_SHAPES)
def test_layernorm(rows, cols, dt, planar):
    if planar:
        rows, cols = cols, rows
    for pad in (0, 8, 3):
        check_layernorm(rows, cols, dt, planar, pad, dt if pad else torch.float32, seed=pad)


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
def test_layernorm_far_from_zero_and_of_one_value(dt):
    check_layernorm(9, 640, dt, False, 0, torch.float32, mean=300.0)
    check_layernorm(640, 64, dt, True, 0, torch.float32, mean=300.0)
    x = torch.full((3, 100), 5.0, dtype=dt, device="cuda")  # no variance: eps alone
    s = torch.full((100,), 2.0, device="cuda")
    b = torch.arange(100.0, device="cuda")
    y, m, r = O.layernorm(x, s, b, eps=1e-6, stats=True)
    assert torch.equal(y, b.to(dt).expand(3, 100)) and torch.all(m == 5.0)
    near(r.double().cpu(), torch.full((3,), 1e3, dtype=torch.float64), torch.full((3,), 1e3 * 6 * U, dtype=torch.float64), "rstd")


def test_layernorm_keeps_to_its_rows():
    """NaN and infinity stay in their rows; what lies beside a slice is not
    written; in place; no bias; more than two dimensions."""
    buf, _ = make(3, 40, 72, torch.float32)
    buf[7, 3] = float("nan")
    buf[9, 60] = float("inf")
    before = buf.clone()
    x = buf[5:25, 2:66]
    s, _ = vec(1, 64, torch.float32)
    want = torch.nn.functional.layer_norm(x.double().cpu(), (64,), s.double().cpu(), None, 1e-6)
    got = O.layernorm(x, s)
    bad = torch.zeros(20, dtype=torch.bool)
    bad[2] = bad[4] = True
    assert torch.isnan(got[2]).all() and torch.isnan(got[4]).all()
    assert torch.isfinite(got[~bad.cuda()]).all()
    near(got.double().cpu()[~bad], want[~bad], torch.full((18, 64), 1e-5, dtype=torch.float64), "y")
    assert torch.equal(got.isnan(), O.layernorm(x, s, out=x).isnan())
    assert torch.equal(x[~bad.cuda()], got[~bad.cuda()])
    after = buf.clone()
    after[5:25, 2:66] = before[5:25, 2:66]
    assert torch.equal(after.nan_to_num(), before.nan_to_num())
    x4, _ = make(4, 6 * 5, 32, torch.float32, planar=True)
    y4, m4, _ = O.layernorm(x4.view(32, 6, 5), s[:32].contiguous(), planar=True, stats=True)
    assert y4.shape == (32, 6, 5) and m4.shape == (6, 5)
    assert torch.equal(y4.view(32, 30), O.layernorm(x4, s[:32].contiguous(), planar=True))
    assert O.layernorm(x4.t().reshape(2, 3, 5, 32), s[:32].contiguous()).shape == (2, 3, 5, 32)


def ln_backward_reference(dy, x, scale, mean, rstd, add):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * scale
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return (dx if add is None else dx + add), (dy * xh).sum(0), dy.sum(0), xh, g


def check_ln_backward(rows, cols, dt, planar, pad, param_dt, add, seed=0):
    x, xv = make(seed, rows, cols, dt, planar, pad, 1.5, 0.3)
    dy, dyv = make(seed + 1, rows, cols, dt, planar, pad)
    a, av = make(seed + 2, rows, cols, dt, planar, pad) if add else (None, None)
    s, sv = vec(seed + 3, cols, param_dt, 0.1, 1.0)
    mean = xv.mean(1).float()
    rstd = (((xv - mean.double()[:, None]) ** 2).mean(1) + 1e-6).rsqrt().float()
    dx, ds, db = O.layernorm_backward(dy, x, s, mean.cuda(), rstd.cuda(), add=a, planar=planar)
    mv, rv = mean.double(), rstd.double()
    wx, ws, wb, xh, g = ln_backward_reference(dyv, xv, sv, mv, rv, av)
    n = cols / 64 + 40
    xe = 2 * U * (xh.abs() + rv[:, None] * xv.abs())  # xh's own error
    p, q = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    qe = n * U * q + (g.abs() * xe).mean(1, keepdim=True)
    err = rv[:, None] * (4 * U * g.abs() + n * U * p + xh.abs() * qe + xe * q + 4 * U * (xh.abs() * q + p))
    tol = err + 4 * U * (wx.abs() + (av.abs() if add else 0)) + half(dt) * (wx.abs() + err) + tiny(dt)
    near(values(dx, planar), wx, tol, "dx")
    ht = half(param_dt)
    es = (dyv.abs() * (xe + (rows + 4) * U * xh.abs())).sum(0)
    near(ds.double().cpu(), ws, es + ht * (ws.abs() + es) + tiny(param_dt), "dscale")
    eb = rows * U * dyv.abs().sum(0)
    near(db.double().cpu(), wb, eb + ht * (wb.abs() + eb) + tiny(param_dt), "dbias")


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,cols", LN_SHAPES)
def test_layernorm_backward(rows, cols, dt, planar):
    if planar:
        rows, cols = cols, rows
    for pad in (0, 8, 3):
        check_ln_backward(rows, cols, dt, planar, pad, dt if pad else torch.float32, pad == 8, seed=pad)


def test_layernorm_backward_of_nothing_and_of_parts():
    dt = torch.bfloat16
    x, _ = make(0, 50, 96, dt)
    dy, _ = make(1, 50, 96, dt)
    add, _ = make(2, 50, 96, dt)
    s, _ = vec(3, 96, dt)
    _, m, r = O.layernorm(x, s, stats=True)
    dx, ds, db = O.layernorm_backward(dy, x, s, m, r, add=add)
    assert torch.equal(O.layernorm_backward(dy, x, s, m, r, add=add, params=False)[0], dx)
    only = O.layernorm_backward(dy, x, s, m, r, dx=False)
    assert only[0] is None and torch.equal(only[1], ds) and torch.equal(only[2], db)
    # over dy, over add
    for over in (0, 1):
        d2, a2 = dy.clone(), add.clone()
        got = O.layernorm_backward(d2, x, s, m, r, add=a2, out=(d2, a2)[over])
        assert torch.equal(got[0], dx) and torch.equal(got[1], ds) and torch.equal(got[2], db)
    # no rows: no gradient
    e = x[:0]
    dx, ds, db = O.layernorm_backward(e, e, s, m[:0], r[:0])
    assert dx.shape == (0, 96) and not ds.any() and not db.any()
    assert O.layernorm(e, s).shape == (0, 96)


def at_ends(rows):
    """Positions from both ends and from between, across several tiles' borders."""
    g = torch.Generator().manual_seed(rows)
    return torch.cat([torch.arange(1100), torch.randint(0, rows, (500,), generator=g), torch.arange(rows - 1100, rows)])


# channels: one up to each of the widths that the kernels of many positions
# hold, odd ones and those of an image's stages
MANY = [(262144 + 520, 3), (262144 + 1, 16), (262144 + 24, 27), (262144 + 5, 32), (262144 + 8, 40), (300003, 64),
        (140000, 72), (131072 + 9, 100), (131072 + 8, 128), (131072 + 3, 200), (66000, 256)]


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,cols", MANY)
def test_layernorm_of_many_positions(rows, cols, dt):
    """Planar order with positions enough for the kernels of many lanes. Each
    position's bounds are those of check_layernorm and check_ln_backward. The
    parameters' sums: a lane adds at most 64 terms (eight of a vector, eight
    tiles at most here), lanes and waves 16 more, the joining of the blocks' 64
    more: 144 roundings."""
    x, xv = make(cols, rows, cols, dt, True, 0, 1.5, 0.3)
    s, sv = vec(cols + 1, cols, dt, 0.1, 1.0)
    b, bv = vec(cols + 2, cols, dt, 0.1)
    y, m, r = O.layernorm(x, s, b, planar=True, stats=True)
    at = at_ends(rows)
    xs = xv[at]
    want, mw, rw, xh = ln_reference(xs, sv, bv, 1e-6)
    n = cols / 64 + 32
    me = n * U * xs.abs().mean(1)
    near(m.double().cpu()[at], mw, me + U * mw.abs(), "mean")
    d = (xs - mw[:, None]).abs()
    ve = me ** 2 + ((n + 4) * U * d * d + 2 * U * d * xs.abs()).mean(1)
    rel = 0.5 * ve / ((d * d).mean(1) + 1e-6) * 1.01 + 6 * U
    near(r.double().cpu()[at], rw, rw * rel, "rstd")
    err = (rw[:, None] * (me[:, None] + U * xs.abs()) + xh.abs() * (rel[:, None] + 4 * U)) * sv.abs()
    near(y.cpu()[:, at].t().double(), want, err + 2 * U * (want.abs() + bv.abs()) + half(dt) * (want.abs() + err) + tiny(dt), "y")

    dy, dyv = make(cols + 3, rows, cols, dt, True)
    dx, ds, db = O.layernorm_backward(dy, x, s, m, r, add=y, planar=True)
    mv, rv, av = m.double().cpu()[at], r.double().cpu()[at], y.cpu()[:, at].t().double()
    wx, _, _, xh, g = ln_backward_reference(dyv[at], xs, sv, mv, rv, av)
    n = cols / 64 + 40
    xe = 2 * U * (xh.abs() + rv[:, None] * xs.abs())
    p, q = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    qe = n * U * q + (g.abs() * xe).mean(1, keepdim=True)
    err = rv[:, None] * (4 * U * g.abs() + n * U * p + xh.abs() * qe + xe * q + 4 * U * (xh.abs() * q + p))
    near(dx.cpu()[:, at].t().double(), wx, err + 4 * U * (wx.abs() + av.abs()) + half(dt) * (wx.abs() + err) + tiny(dt), "dx")
    x64, dy64 = x.double(), dy.double()
    xh = (x64 - m.double()) * r.double()
    es = (dy64.abs() * (144 * U * xh.abs() + 2 * U * (xh.abs() + r.double() * x64.abs()))).sum(1).cpu()
    ws, wb = (dy64 * xh).sum(1).cpu(), dy64.sum(1).cpu()
    near(ds.double().cpu(), ws, es + half(dt) * (ws.abs() + es) + tiny(dt), "dscale")
    eb = 144 * U * dy64.abs().sum(1).cpu()
    near(db.double().cpu(), wb, eb + half(dt) * (wb.abs() + eb) + tiny(dt), "dbias")


# rows enough that each kernel's blocks take several in turn
MANY_ROWS = [(65536 + 77, 20), (33000, 100), (17000, 256), (8200, 500), (4200, 777), (2100, 2048), (1100, 4096), (530, 8192),
             (530, 16384)]


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,cols", MANY_ROWS)
def test_layernorm_of_many_rows(rows, cols, dt):
    check_layernorm(rows, cols, dt, False, 0, dt)
    check_ln_backward(rows, cols, dt, False, 0, dt, True)


def test_layernorm_gradient_against_differences():
    """<dx, v> is the derivative of <dy, y> along v, and so for the parameters:
    central differences of the formula in 64 bits, off by step^2 / 6 of the
    third derivative (measured below 1e-8 here), and fp32 sums of 24 * 48
    terms, each within the bounds above: 1e-5 of the sum of their magnitudes."""
    for planar in (False, True):
        x, xv = make(0, 24, 48, torch.float32, planar)
        dy, dyv = make(1, 24, 48, torch.float32, planar)
        s, sv = vec(2, 48, torch.float32, 0.2, 1.0)
        b, bv = vec(3, 48, torch.float32)
        _, m, r = O.layernorm(x, s, b, planar=planar, stats=True)
        dx, ds, db = O.layernorm_backward(dy, x, s, m, r, planar=planar)
        g = torch.Generator().manual_seed(9)
        vx, vs, vb = (torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (xv, sv, bv))
        t = 1e-5
        f = lambda k: (dyv * ln_reference(xv + k * vx, sv + k * vs, bv + k * vb, 1e-6)[0]).sum()  # noqa: E731
        want = (f(t) - f(-t)) / (2 * t)
        parts = [(values(dx, planar) * vx), ds.double().cpu() * vs, db.double().cpu() * vb]
        got, size = sum(p.sum() for p in parts), sum(p.abs().sum() for p in parts)
        assert abs(got - want) <= 1e-5 * size + 1e-6, (float(got), float(want))


# ----------------------------------------------------------------- Dense


def act64(z, act):
    """The activation and its derivative."""
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    if act == "silu":
        return z * s, s + z * s * (1 - s)
    if act == "sigmoid":
        return s, s * (1 - s)
    if act == "lrelu":
        return torch.where(z >= 0, z, SLOPE * z), torch.where(z >= 0, 1.0, SLOPE).double()
    return z, torch.ones_like(z)


def act_error(z, ze, act):
    """How far act(z) may be off for z off by ze; the derivative likewise."""
    e = 1.2 * ze
    return e if act in (None, "lrelu") else e + 3e-7 * (1 + z.abs())


DENSE_SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 257), (2, 33, 5), (3, 128, 48), (7, 777, 130), (16, 512, 640),
                (17, 96, 100), (64, 64, 64), (65, 72, 129), (100, 1, 100), (128, 128, 128), (129, 65, 257),
                (200, 40, 300), (256, 192, 512), (300, 256, 32), (33, 2500, 40), (520, 64, 264), (1030, 32, 96)]


def weight(seed, n, k, dt, wt):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(n, k, generator=g) / math.sqrt(k)).to(dt)
    d = w.cuda()
    return (d.t().contiguous().t() if wt else d), w.double()


def check_dense(rows, k, n, dt, planar, pad, wt, act, residual, save, bias, seed=0):
    x, xv = make(seed, rows, k, dt, planar, pad)
    w, wv = weight(seed + 1, n, k, dt, wt)
    b, bv = vec(seed + 2, n, bias) if bias else (None, torch.zeros(n, dtype=torch.float64))
    r, rv = make(seed + 3, rows, n, dt, planar, pad) if residual else (None, 0)
    got = O.dense(x, w, b, act=act, slope=SLOPE, residual=r, planar=planar, save=save)
    y, z = got if save else (got, None)
    zw = xv @ wv.t() + bv
    ze = (k + 1) * U * (xv.abs() @ wv.abs().t()) + U * (zw.abs() + bv.abs())
    if save:
        near(values(z, planar), zw, ze + half(dt) * (zw.abs() + ze) + tiny(dt), "z")
    want = act64(zw, act)[0] + rv
    err = act_error(zw, ze, act) + 2 * U * want.abs() + (U * rv.abs() if residual else 0)
    near(values(y, planar), want, err + half(dt) * (want.abs() + err) + tiny(dt), "y")


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", DENSE_SHAPES)
def test_dense(rows, k, n, dt, planar):
    i = (rows * 7 + k * 3 + n) % 6
    for j, (pad, wt) in enumerate([(0, False), (8, True), (3, False), (0, True)]):
        act = ACTS[(i + j) % 6]
        check_dense(rows, k, n, dt, planar, pad, wt, act, j % 2 == 0, j in (0, 3), (None, dt, torch.float32, dt)[j],
                    seed=j)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
def test_dense_activations(dt, act):
    check_dense(96, 80, 72, dt, False, 0, False, act, True, True, dt)
    check_dense(96, 80, 72, dt, True, 0, False, act, False, False, torch.float32)


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
def test_dense_of_nothing(dt):
    x, _ = make(0, 5, 16, dt)
    w, _ = weight(1, 24, 16, dt, False)
    b, _ = vec(2, 24, dt)
    assert O.dense(x[:0], w, b).shape == (0, 24)
    assert O.dense(x, w[:0]).shape == (5, 0)
    # no inputs: the bias through the activation
    y = O.dense(x[:, :0], w[:, :0], b, act="lrelu", slope=0.5)
    assert torch.equal(y, torch.where(b >= 0, b, 0.5 * b).expand(5, 24))
    dx, dw, db = O.dense_backward(torch.zeros(0, 24, dtype=dt, device="cuda"), x[:0], w)
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == (24, 16)


def test_dense_far_values():
    """Activations at their tails, and infinities and NaN: a row's own, and no
    other row's."""
    z = torch.tensor([-float("inf"), -3e38, -1e9, -100.0, -7.0, -6.0, 0.0, 6.0, 7.0, 100.0, 1e9, 3e38, float("inf"),
                      float("nan")])
    one = torch.ones(1, 1, device="cuda")
    x = z.view(-1, 1).cuda()
    for act in ACTS[1:]:
        got = O.dense(x, one, act=act, slope=SLOPE).view(-1).double().cpu()
        want = act64(z.double(), act)[0]
        if act in ("gelu", "gelu_tanh", "silu"):
            want[0] = 0.0  # their limit
            if act == "gelu_tanh":
                want[1], want[11] = 0.0, 3e38
        assert torch.isnan(got[13]) and torch.equal(got[12:13], want[12:13]), act
        fine = slice(0, 12)
        near(got[fine].clamp(-3.4e38, 3.4e38), want[fine].clamp(-3.4e38, 3.4e38),
             6e-7 * (1 + want[fine].abs().clamp(max=3.4e38)), act)
        # past +-7 a derivative is 0 or 1 (slope, for lrelu) but for the small terms
        _, dw, _ = O.dense_backward(torch.ones(14, 1, device="cuda"), x, one, z=x, act=act, slope=SLOPE, dw=True)
        dx, _, _ = O.dense_backward(torch.ones(14, 1, device="cuda"), torch.zeros(14, 1, device="cuda"), one, z=x,
                                    act=act, slope=SLOPE)
        d = dx.view(-1).double().cpu()
        lim = {"lrelu": (SLOPE, 1.0), "sigmoid": (0.0, 0.0)}.get(act, (0.0, 1.0))
        low, high = d[:4], d[9:13]
        near(low, torch.full((4,), lim[0], dtype=torch.float64), torch.full((4,), 1e-7, dtype=torch.float64), act)
        near(high, torch.full((4,), lim[1], dtype=torch.float64), torch.full((4,), 1e-7, dtype=torch.float64), act)
        assert act == "lrelu" or torch.isnan(d[13])
    for dt in TYPES.values():
        x, _ = make(0, 70, 96, dt)
        w, _ = weight(1, 80, 96, dt, False)
        clean = O.dense(x, w)
        x[11, 5] = float("nan")
        x[40, 95] = float("inf")
        y = O.dense(x, w)
        keep = torch.ones(70, dtype=torch.bool, device="cuda")
        keep[11] = keep[40] = False
        assert torch.isnan(y[11]).all() and not torch.isfinite(y[40]).any()
        assert torch.equal(y[keep], clean[keep])


def check_dense_backward(rows, k, n, dt, planar, pad, wt, act, db_dt, seed=0):
    x, xv = make(seed, rows, k, dt, planar, pad)
    w, wv = weight(seed + 1, n, k, dt, wt)
    dy, dyv = make(seed + 2, rows, n, dt, planar, pad)
    z, zv = make(seed + 3, rows, n, dt, planar, pad) if act else (None, None)
    dx, dw, db = O.dense_backward(dy, x, w, z=z, act=act, slope=SLOPE, planar=planar, db_dtype=db_dt)
    dz = dyv * act64(zv, act)[1] if act else dyv
    dze = dyv.abs() * 6e-7 * (1 + zv.abs()) + U * dz.abs() if act else torch.zeros_like(dz)
    eb = dze.sum(0) + rows * U * dz.abs().sum(0)
    hb = half(db_dt or dt)
    wb = dz.sum(0)
    near(db.double().cpu(), wb, eb + hb * (wb.abs() + eb) + tiny(db_dt or dt), "db")
    if act:
        dze = dze + half(dt) * dz.abs() + tiny(dt)
    for got, want, mag, e, terms in (
            (values(dx, planar), dz @ wv, (dz.abs() + dze) @ wv.abs(), dze @ wv.abs(), n),
            (dw.double().cpu(), dz.t() @ xv, (dz.abs() + dze).t() @ xv.abs(), dze.t() @ xv.abs(), rows)):
        tol = e + (terms + 1) * U * mag
        near(got, want, tol + half(dt) * (want.abs() + tol) + tiny(dt), "dx, dw of %d terms" % terms)
    assert dw.shape == w.shape and dw.stride() == w.stride()


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", DENSE_SHAPES)
def test_dense_backward(rows, k, n, dt, planar):
    i = (rows * 5 + k + n * 3) % 6
    for j, (pad, wt) in enumerate([(0, False), (8, True), (3, False)]):
        check_dense_backward(rows, k, n, dt, planar, pad, wt, ACTS[(i + j) % 6], (None, torch.float32, dt)[j], seed=j)


@pytest.mark.parametrize("act", ACTS)
def test_dense_gradient_against_differences(act):
    """<gradient, v> against central differences of <dy, act(x w^T + b) + r> in
    64 bits along a random direction of x, w and b; the pre-activations keep
    off LeakyReLU's corner. Differences are off by their step squared (1e-10
    of order-one derivatives), the fp32 products by the bounds above: 2e-5 of
    the sum of the terms' magnitudes."""
    rows, k, n = 24, 20, 28
    for planar in (False, True):
        x, xv = make(0, rows, k, torch.float32, planar)
        w, wv = weight(1, n, k, torch.float32, False)
        b, bv = vec(2, n, torch.float32)
        dy, dyv = make(3, rows, n, torch.float32, planar)
        y, z = O.dense(x, w, b, act=act, slope=SLOPE, planar=planar, save=True)
        dx, dw, db = O.dense_backward(dy, x, w, z=z, act=act, slope=SLOPE, planar=planar)
        g = torch.Generator().manual_seed(5)
        vx, vw, vb = (torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (xv, wv, bv))
        t = 1e-5
        z0 = xv @ wv.t() + bv
        slack = 2 * t * ((vx @ wv.t()).abs() + (xv @ vw.t()).abs() + vb.abs())
        keep = (z0.abs() > slack).double() if act == "lrelu" else 1.0
        dyk = dyv * keep
        if act == "lrelu":
            dyd = dyk.float()
            dx, dw, db = O.dense_backward((dyd.t().contiguous() if planar else dyd).cuda(), x, w, z=z, act=act,
                                          slope=SLOPE, planar=planar)
        f = lambda e: (dyk * act64((xv + e * vx) @ (wv + e * vw).t() + bv + e * vb, act)[0]).sum()  # noqa: E731
        want = (f(t) - f(-t)) / (2 * t)
        parts = [values(dx, planar) * vx, dw.double().cpu() * vw, db.double().cpu() * vb]
        got, size = sum(p.sum() for p in parts), sum(p.abs().sum() for p in parts)
        assert abs(got - want) <= 2e-5 * size + 1e-6, (act, planar, float(got), float(want))


# sizes that reach every tile, with and without a cut sum, aligned and not:
# rows, k, n
BIG_SHAPES = [(4096, 256, 4096), (2048, 512, 2048), (2048, 512, 4096), (1024, 512, 1024), (256, 8192, 256),
              (2048, 511, 2047), (4095, 1023, 2049), (1023, 511, 1025), (2048, 1028, 1028), (40000, 64, 96), (16, 4096, 512)]


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", BIG_SHAPES)
def test_products_of_every_tile(rows, k, n, dt, wt, planar):
    """The products alone, in both directions, with the 64-bit products on the
    card. Each of a sum's `terms` roundings is half a step at most of a partial
    sum of random signs, which reaches sqrt(terms) of a product's deviation d:
    together a walk of about terms d u / 2, where S is 0.64 terms d. So 8 u S
    holds for every element with room (and terms u S always)."""
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)

    def rand(a, b, flip, std=1.0):
        t = (torch.randn(b, a, generator=g, device="cuda") if flip else torch.randn(a, b, generator=g, device="cuda"))
        t = (t * std).to(dt)
        return (t, t.t().double()) if flip else (t, t.double())

    x, xv = rand(rows, k, planar)
    dy, dyv = rand(rows, n, planar)
    w, wv = rand(n, k, wt, 1 / math.sqrt(k))
    w = w.t() if wt else w
    y = O.dense(x, w, planar=planar)
    dx, dw, db = O.dense_backward(dy, x, w, planar=planar)
    for got, want, size, terms in (((y.t() if planar else y), xv @ wv.t(), xv.abs() @ wv.abs().t(), k),
                                   ((dx.t() if planar else dx), dyv @ wv, dyv.abs() @ wv.abs(), n),
                                   (dw, dyv.t() @ xv, dyv.abs().t() @ xv.abs(), rows)):
        tol = min(terms, 8) * U * size + half(dt) * want.abs() * 1.01 + tiny(dt)
        off = (got.double() - want).abs() - tol
        assert bool((off <= 0).all()), (terms, float(off.max()))
    eb = rows * U * dyv.abs().sum(0)
    wb = dyv.sum(0)
    assert bool(((db.double() - wb).abs() <= eb + half(dt) * (wb.abs() + eb) + tiny(dt)).all())


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("shape", [(64, 64, 64), (2048, 512, 2048), (1023, 511, 1025)])
def test_fp32_products_of_far_values(shape, planar):
    """fp32 products are formed from three bf16 parts: tiny and huge operands
    keep their bits, and infinities and NaN are what fp32 sums give."""
    rows, k, n = shape
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, k, generator=g, device="cuda")
    w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    put = (lambda t: t.t().contiguous()) if planar else (lambda t: t)
    take = (lambda t: t.t()) if planar else (lambda t: t)
    bound = lambda a, b: 8 * U * (a.abs() @ b.abs().t())  # as above  # noqa: E731
    for sx, sw in ((2.0 ** -100, 1.0), (2.0 ** -120, 2.0 ** 20), (2.0 ** 100, 1.0), (2.0 ** 110, 2.0 ** -110),
                   (2.0 ** 60, 2.0 ** 50)):
        a, b = x * sx, w * sw
        av, bv = a.double(), b.double()
        want = av @ bv.t()
        got = take(O.dense(put(a), b, planar=planar)).double()
        assert bool(((got - want).abs() <= bound(av, bv) + U * want.abs() + 1e-44).all()), (sx, sw)
    x[3, 5], x[7, 9], x[11, 13] = float("inf"), float("nan"), 3e38
    w[:, 13] = w[:, 13].abs() + 2.0  # 3e38 times this leaves the range: infinity
    got, want = take(O.dense(put(x), w, planar=planar)), x.double() @ w.double().t()
    assert torch.isnan(got[7]).all() and torch.isinf(got[3]).all() and torch.equal(got[3].sign(), w[:, 5].sign())
    assert torch.isposinf(got[11]).all()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[3] = keep[7] = keep[11] = False
    # column 13's one large term stays in every later partial sum P, so the
    # roundings are of P and not of a walk's sums: 96 of them at k = 512, rms
    # 0.58 u P each with P = 6 and S = 20, are 1.7 u S rms and 10 u S at six
    # deviations, past the 8 of sums of like terms. k u S bounds any order.
    slack = k * U * (x.double().abs() @ w.double().abs().t()) + U * want.abs()
    assert bool(((got.double() - want).abs()[keep] <= slack[keep]).all())
    x[3] = x[7] = x[11] = 0.0  # the other rows' bits do not depend on these
    assert torch.equal(take(O.dense(put(x), w, planar=planar))[keep], got[keep])


# ------------------------------------------------------ used together


def test_broadcast_inputs_and_writes_beside_slices():
    """An expanded input row, an expanded gradient, and outputs into the
    middle of a wider buffer, whose other elements stay."""
    dt = torch.bfloat16
    row, rv = make(0, 1, 96, dt)
    w, wv = weight(1, 80, 96, dt, False)
    y = O.dense(row.expand(70, 96), w)
    assert torch.equal(y, O.dense(row.expand(70, 96).contiguous(), w))
    d1, _ = make(2, 1, 80, dt)
    x, _ = make(3, 70, 96, dt)
    for a, b in zip(O.dense_backward(d1.expand(70, 80), x, w), O.dense_backward(d1.expand(70, 80).contiguous(), x, w)):
        assert torch.equal(a, b)
    for shape, cut in (((74, 90), (slice(2, 72), slice(5, 85))), ((84, 90), (slice(3, 83), slice(7, 77)))):
        buf = torch.full(shape, 7.0, dtype=dt, device="cuda")
        planar = shape[0] == 84
        xin = x.t().contiguous() if planar else x
        out = O.dense(xin, w, planar=planar, out=buf[cut])
        assert torch.equal(out, O.dense(xin, w, planar=planar))
        rest = torch.ones(shape, dtype=torch.bool, device="cuda")
        rest[cut] = False
        assert torch.all(buf[rest] == 7.0)
    # the residual's own place
    r, _ = make(5, 70, 80, dt)
    want = O.dense(x, w, residual=r)
    assert torch.equal(O.dense(x, w, residual=r, out=r), want)


def block_forward(x, p, planar):
    h, m, r = O.layernorm(x, p["s"], p["b"], planar=planar, stats=True)
    a, z = O.dense(h, p["w1"], p["b1"], act="gelu", planar=planar, save=True)
    y = O.dense(a, p["w2"], p["b2"], residual=x, planar=planar)
    return y, (h, m, r, a, z)


def block_backward(dy, x, p, kept, planar):
    h, m, r, a, z = kept
    da, dw2, db2 = O.dense_backward(dy, a, p["w2"], planar=planar)
    dh, dw1, db1 = O.dense_backward(da, h, p["w1"], z=z, act="gelu", planar=planar)
    dx, ds, db = O.layernorm_backward(dh, x, p["s"], m, r, add=dy, planar=planar)
    return [dx, ds, db, dw1, db1, dw2, db2]


def block_parameters(c, hidden, dt):
    return {"s": vec(1, c, dt, 0.1, 1.0)[0], "b": vec(2, c, dt, 0.1)[0], "w1": weight(3, hidden, c, dt, False)[0],
            "b1": vec(4, hidden, dt, 0.1)[0], "w2": weight(5, c, hidden, dt, False)[0], "b2": vec(6, c, dt, 0.1)[0]}


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
def test_a_block_forward_and_backward(dt, planar):
    """LayerNorm, Dense, GELU, Dense and the residual as a training step uses
    them, against torch's autograd over the formula in 64 bits. Nine stored
    results lie between the input and a gradient, each within a few half steps
    of a value of order one and weights of norm about one: 2-norms agree to
    16 half steps of the type (fp32: to 64, for the sums)."""
    c, hidden, rows = 96, 200, 150
    x, xv = make(0, rows, c, dt, planar)
    dy, dyv = make(9, rows, c, dt, planar)
    p = block_parameters(c, hidden, dt)
    y, kept = block_forward(x, p, planar)
    grads = block_backward(dy, x, p, kept, planar)
    names = ["s", "b", "w1", "b1", "w2", "b2"]
    q = {k: p[k].double().cpu().requires_grad_() for k in names}
    xr = xv.clone().contiguous().requires_grad_()
    h = torch.nn.functional.layer_norm(xr, (c,), q["s"], q["b"], 1e-6)
    yr = act64(h @ q["w1"].t() + q["b1"], "gelu")[0] @ q["w2"].t() + q["b2"] + xr
    want = torch.autograd.grad((yr * dyv).sum(), [xr] + [q[k] for k in names])
    bar = half(dt) * (64 if dt == torch.float32 else 16)
    for got, ref in zip([values(y, planar), values(grads[0], planar)] + [g.double().cpu() for g in grads[1:]],
                        [yr.detach()] + list(want)):
        assert float((got - ref).norm() / ref.norm()) <= bar


def test_captured_and_replayed_on_two_streams():
    """The block's forward and backward captured into two graphs with
    workspaces of their own, replayed in turn on two streams, with eager calls
    in between: the eager call's bits every time."""
    dt = torch.bfloat16
    p = block_parameters(96, 200, dt)
    xs = [make(20 + i, 150, 96, dt)[0] for i in range(2)]
    dys = [make(30 + i, 150, 96, dt)[0] for i in range(2)]

    def step(i):
        y, kept = block_forward(xs[i], p, False)
        return [y] + block_backward(dys[i], xs[i], p, kept, False)

    want = [step(0), step(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for i in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(step(i))
        graphs.append(g)
    for k in range(4):
        for o in outs[0] + outs[1]:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = step(k % 2)
        torch.cuda.synchronize()
        for a, b in zip(outs[0] + outs[1] + eager, want[0] + want[1] + want[k % 2]):
            assert torch.equal(a, b), k


def test_beside_the_executor():
    """An executor's pass and the operators on one card: each keeps its bits."""
    from conftest import smooth_image, weights
    from maxim_amd import hip as H
    plan = P.Plan(weights("S-1"), 64, 64)
    gpu = H.Gpu(plan)
    img = smooth_image(64, 64)
    first = gpu.run(img)
    x, _ = make(0, 64 * 64, 32, torch.float32, True)
    s, _ = vec(1, 32, torch.float32)
    y = O.layernorm(x, s, planar=True)
    assert (gpu.run(img) == first).all()
    assert torch.equal(O.layernorm(x, s, planar=True), y)
    gpu.close()


def test_refusals_on_the_card():
    x, _ = make(0, 8, 16, torch.float32)
    w, _ = weight(1, 24, 16, torch.float32, False)
    with pytest.raises(P.MaximError, match="not on the card"):
        O.dense(x, w.cpu())
    with pytest.raises(P.MaximError, match="not float32"):
        O.dense(x.double(), w)
    with pytest.raises(P.MaximError, match="no one stride"):
        O.dense(x.view(4, 2, 16)[:, :1].expand(4, 3, 16)[:, :, ::1], w)
    with pytest.raises(P.MaximError, match="unknown activation"):
        O.dense(x, w, act="tanh")
    with pytest.raises(P.MaximError, match="requires a gradient"):
        O.dense(x, w.clone().requires_grad_())
    with torch.no_grad():
        O.dense(x, w.clone().requires_grad_())
    with pytest.raises(P.MaximError, match="neither rows nor columns"):
        O.dense(torch.zeros(8, 32, device="cuda")[:, ::2], w)
    with pytest.raises(P.MaximError, match="not a contiguous vector"):
        O.dense(x, w, torch.zeros(48, device="cuda")[::2])
    with pytest.raises(P.MaximError, match="z: missing"):
        O.dense_backward(O.dense(x, w), x, w, act="gelu")
    with pytest.raises(P.MaximError, match="contiguous fp32 value"):
        O.layernorm_backward(x, x, x[0].contiguous(), torch.zeros(7, device="cuda"), torch.zeros(7, device="cuda"))
    with pytest.raises(P.MaximError, match="overlaps"):
        O.layernorm(x[:6], x[0].clone(), out=x[2:])
    d = C.c_int(-1)
    assert O._lib() is not None and torch.cuda.current_device() == 0 and d.value == -1
