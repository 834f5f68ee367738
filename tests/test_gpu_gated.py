"""The gated Dense on device tensors, forward and backward, against its
formulas in 64 bits.

Tolerances as in test_gpu_operators.py (u = 2^-24, h half a step of the
result's type): a sum of k terms in fp32, in any order, is off by k u S at most,
S the sum of the terms' magnitudes; act by 3e-7 (1 + |a|) and its derivative by
6e-7 (1 + |a|); an error e of a moves act(a) by 1.2 e at most. A product of two
values each off by some is off by both, times the other, and one rounding."""

import math

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402
from test_gpu_operators import (ACTS, SLOPE, TYPES, U, act64, act_error, half, make, near, tiny, values, vec,  # noqa: E402
                                weight)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()


SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 257), (2, 33, 5), (3, 128, 48), (7, 777, 130), (16, 512, 640), (17, 96, 100),
          (64, 64, 64), (65, 72, 129), (100, 1, 100), (128, 128, 128), (129, 65, 257), (200, 40, 300), (256, 192, 512),
          (300, 256, 32), (33, 2500, 40), (520, 64, 264), (1030, 32, 96), (40, 96, 12)]


def gated_error(a, c, ae, ce, act, want):
    """How far act(a) c is off for sums off by ae and ce."""
    f = act64(a, act)[0]
    fe = act_error(a, ae, act) + U * f.abs()
    return fe * (c.abs() + ce) + f.abs() * ce + U * want.abs()


def check_gated(rows, k, n, dt, planar, pad, wt, act, save, bias, seed=0):
    x, xv = make(seed, rows, k, dt, planar, pad)
    w, wv = weight(seed + 1, 2 * n, k, dt, wt)
    b, bv = vec(seed + 2, 2 * n, bias) if bias else (None, torch.zeros(2 * n, dtype=torch.float64))
    got = O.gated(x, w, b, act=act, slope=SLOPE, planar=planar, save=save)
    y, z = got if save else (got, None)
    zw = xv @ wv.t() + bv
    ze = (k + 1) * U * (xv.abs() @ wv.abs().t()) + U * (zw.abs() + bv.abs())
    if save:
        near(values(z, planar), zw, ze + half(dt) * (zw.abs() + ze) + tiny(dt), "z")
    a, c, ae, ce = zw[:, :n], zw[:, n:], ze[:, :n], ze[:, n:]
    want = act64(a, act)[0] * c
    err = gated_error(a, c, ae, ce, act, want)
    near(values(y, planar), want, err + half(dt) * (want.abs() + err) + tiny(dt), "y")


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_gated(rows, k, n, dt, planar):
    i = (rows * 7 + k * 3 + n) % 6
    for j, (pad, wt) in enumerate([(0, False), (8, True), (3, False), (0, True)]):
        check_gated(rows, k, n, dt, planar, pad, wt, ACTS[(i + j) % 6], j in (0, 3), (None, dt, torch.float32, dt)[j],
                    seed=j)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
def test_gated_activations(dt, act):
    check_gated(96, 80, 72, dt, False, 0, False, act, True, dt)
    check_gated(96, 80, 72, dt, True, 0, False, act, False, torch.float32)


def check_gated_backward(rows, k, n, dt, planar, pad, wt, act, db_dt, seed=0):
    x, xv = make(seed, rows, k, dt, planar, pad)
    w, wv = weight(seed + 1, 2 * n, k, dt, wt)
    dy, dyv = make(seed + 2, rows, n, dt, planar, pad)
    z, zv = make(seed + 3, rows, 2 * n, dt, planar, pad)
    dx, dw, db = O.gated_backward(dy, x, w, z, act=act, slope=SLOPE, planar=planar, db_dtype=db_dt)
    a, c = zv[:, :n], zv[:, n:]
    f, g = act64(a, act)
    dz = torch.cat([dyv * c * g, dyv * f], 1)
    dze = torch.cat([(dyv * c).abs() * 6e-7 * (1 + a.abs()), dyv.abs() * act_error(a, 0 * a, act)], 1) + 3 * U * dz.abs()
    eb = dze.sum(0) + rows * U * dz.abs().sum(0)
    hb = half(db_dt or dt)
    wb = dz.sum(0)
    near(db.double().cpu(), wb, eb + hb * (wb.abs() + eb) + tiny(db_dt or dt), "db")
    dze = dze + half(dt) * dz.abs() + tiny(dt)
    for got, want, mag, e, terms in (
            (values(dx, planar), dz @ wv, (dz.abs() + dze) @ wv.abs(), dze @ wv.abs(), 2 * n),
            (dw.double().cpu(), dz.t() @ xv, (dz.abs() + dze).t() @ xv.abs(), dze.t() @ xv.abs(), rows)):
        tol = e + (terms + 1) * U * mag
        near(got, want, tol + half(dt) * (want.abs() + tol) + tiny(dt), "dx, dw of %d terms" % terms)
    assert dw.shape == w.shape and dw.stride() == w.stride()


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_gated_backward(rows, k, n, dt, planar):
    i = (rows * 5 + k + n * 3) % 6
    for j, (pad, wt) in enumerate([(0, False), (8, True), (3, False)]):
        check_gated_backward(rows, k, n, dt, planar, pad, wt, ACTS[(i + j) % 6], (None, torch.float32, dt)[j], seed=j)


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
def test_gated_of_nothing(dt):
    x, _ = make(0, 5, 16, dt)
    w, _ = weight(1, 24, 16, dt, False)
    b, bv = vec(2, 24, dt)
    assert O.gated(x[:0], w, b).shape == (0, 12)
    assert O.gated(x, w[:0]).shape == (5, 0)
    # no inputs: the bias's gate and value
    for planar in (False, True):
        xe = x[:, :0].t() if planar else x[:, :0]
        y, z = O.gated(xe, w[:, :0], b, act="lrelu", slope=0.5, planar=planar, save=True)
        a, c = bv[:12], bv[12:]
        want = (torch.where(a >= 0, a, 0.5 * a) * c).expand(5, 12)
        near(values(y, planar), want, half(dt) * want.abs() * 1.01 + 2 * U * want.abs(), "y")
        assert torch.equal(values(z, planar), bv.expand(5, 24))
    dx, dw, db = O.gated_backward(torch.zeros(0, 12, dtype=dt, device="cuda"), x[:0], w, O.gated(x[:0], w, save=True)[1])
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == (24, 16)
    dx, dw, db = O.gated_backward(x[:, :0], x, w[:0], x[:, :0])
    assert not dx.any() and dw.shape == (0, 16) and db.shape == (0,)


def test_gated_backward_of_parts():
    dt = torch.bfloat16
    x, _ = make(0, 70, 96, dt)
    w, _ = weight(1, 2 * 44, 96, dt, False)
    dy, _ = make(2, 70, 44, dt)
    _, z = O.gated(x, w, save=True)
    dx, dw, db = O.gated_backward(dy, x, w, z)
    for which in range(3):
        on = [which == i for i in range(3)]
        got = O.gated_backward(dy, x, w, z, dx=on[0], dw=on[1], db=on[2])
        for i, (g, want) in enumerate(zip(got, (dx, dw, db))):
            assert torch.equal(g, want) if i == which else g is None


def test_gated_far_values():
    """Infinities and NaN keep to their rows, and a gate at minus infinity is
    its activation's limit times the value."""
    for dt in TYPES.values():
        for planar in (False, True):
            x, _ = make(0, 70, 96, dt, planar)
            w, _ = weight(1, 80, 96, dt, False)
            clean = O.gated(x, w, planar=planar)
            xr, cr = (x.t(), clean.t()) if planar else (x, clean)
            xr[11, 5] = float("nan")
            xr[40, 95] = float("inf")
            y = O.gated(x, w, planar=planar)
            y = y.t() if planar else y
            keep = torch.ones(70, dtype=torch.bool, device="cuda")
            keep[11] = keep[40] = False
            assert torch.isnan(y[11]).all() and torch.equal(y[keep], cr[keep])
    one = torch.ones(2, 1, device="cuda")
    z = torch.tensor([-float("inf"), -100.0, -3e4, 100.0], device="cuda")
    x = z[:, None].contiguous()
    for act, want in (("silu", [math.nan, 0.0, 0.0, 1e4]), ("gelu", [math.nan, 0.0, 0.0, 1e4])):
        # limit 0 times minus infinity; the others' tails
        y = O.gated(x, one, act=act).view(-1).cpu()
        assert math.isnan(y[0]) and torch.equal(y[1:3].abs() < 1e-30, torch.ones(2, dtype=torch.bool))
        assert abs(float(y[3]) - want[3]) <= 1e4 * 6e-7


# sizes that reach every tile: rows, k, n
BIG_SHAPES = [(4096, 256, 2048), (2048, 512, 1024), (1024, 512, 512), (256, 8192, 128), (2048, 511, 1023), (4095, 1023, 1025),
              (1023, 511, 513), (2048, 1028, 516), (40000, 64, 48), (16, 4096, 512), (700, 64, 4), (2048, 2048, 4096)]


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", BIG_SHAPES)
def test_gated_products_of_every_tile(rows, k, n, dt, wt, planar):
    """Both sums of every result, through z and through y of no activation,
    against 64-bit products on the card. 8 u S for a sum's roundings, as
    test_products_of_every_tile has it."""
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)

    def rand(a, b, flip, std=1.0):
        t = torch.randn(b, a, generator=g, device="cuda") if flip else torch.randn(a, b, generator=g, device="cuda")
        t = (t * std).to(dt)
        return (t, t.t().double()) if flip else (t, t.double())

    x, xv = rand(rows, k, planar)
    w, wv = rand(2 * n, k, wt, 1 / math.sqrt(k))
    w = w.t() if wt else w
    b = torch.randn(2 * n, generator=g, device="cuda")
    y, z = O.gated(x, w, b, act=None, planar=planar, save=True)
    y, z = (y.t(), z.t()) if planar else (y, z)
    want = xv @ wv.t() + b.double()
    err = min(k, 8) * U * (xv.abs() @ wv.abs().t()) + U * want.abs()
    tol = err + half(dt) * want.abs() * 1.01 + tiny(dt)
    off = (z.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())
    a, c, ae, ce = want[:, :n], want[:, n:], err[:, :n], err[:, n:]
    p = a * c
    pe = ae * (c.abs() + ce) + a.abs() * ce + U * p.abs()
    off = (y.double() - p).abs() - (pe + half(dt) * (p.abs() + pe) * 1.01 + tiny(dt))
    assert bool((off <= 0).all()), float(off.max())
    # the same results where z is not kept
    assert torch.equal(O.gated(x, w, b, act=None, planar=planar), y.t() if planar else y)


@pytest.mark.parametrize("act", ACTS)
def test_gated_gradient_against_differences(act):
    """<gradient, v> against central differences of <dy, act(a) c> in 64 bits
    along a random direction of x, w and b; gates keep off LeakyReLU's corner.
    Differences are off by their step squared (1e-10 of order-one third
    derivatives), the fp32 products by the bounds above: 2e-5 of the sum of the
    terms' magnitudes."""
    rows, k, n = 24, 20, 28
    for planar in (False, True):
        x, xv = make(0, rows, k, torch.float32, planar)
        w, wv = weight(1, 2 * n, k, torch.float32, False)
        b, bv = vec(2, 2 * n, torch.float32)
        dyv = make(3, rows, n, torch.float32)[1]
        _, z = O.gated(x, w, b, act=act, slope=SLOPE, planar=planar, save=True)
        g = torch.Generator().manual_seed(5)
        vx, vw, vb = (torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (xv, wv, bv))
        t = 1e-5
        if act == "lrelu":
            a0 = (xv @ wv.t() + bv)[:, :n]
            slack = 2 * t * ((vx @ wv.t()).abs() + (xv @ vw.t()).abs() + vb.abs())[:, :n]
            dyv = dyv * (a0.abs() > slack)
        dy = dyv.float()
        dx, dw, db = O.gated_backward((dy.t().contiguous() if planar else dy).cuda(), x, w, z, act=act, slope=SLOPE,
                                      planar=planar)

        def f(e):
            q = (xv + e * vx) @ (wv + e * vw).t() + bv + e * vb
            return (dyv * act64(q[:, :n], act)[0] * q[:, n:]).sum()

        want = (f(t) - f(-t)) / (2 * t)
        parts = [values(dx, planar) * vx, dw.double().cpu() * vw, db.double().cpu() * vb]
        got, size = sum(p.sum() for p in parts), sum(p.abs().sum() for p in parts)
        assert abs(got - want) <= 2e-5 * size + 1e-6, (act, planar, float(got), float(want))


def test_gated_slices_and_broadcasts():
    """An expanded input row, results into the middle of wider buffers, whose
    other elements stay, more than two dimensions, another memory order than
    the call's."""
    dt = torch.bfloat16
    row, _ = make(0, 1, 96, dt)
    w, _ = weight(1, 160, 96, dt, False)
    assert torch.equal(O.gated(row.expand(70, 96), w), O.gated(row.expand(70, 96).contiguous(), w))
    x, _ = make(3, 70, 96, dt)
    for planar in (False, True):
        xin = x.t().contiguous() if planar else x
        shape, cut = ((84, 90), (slice(3, 83), slice(7, 77))) if planar else ((74, 90), (slice(2, 72), slice(5, 85)))
        buf = torch.full(shape, 7.0, dtype=dt, device="cuda")
        out = O.gated(xin, w, planar=planar, out=buf[cut])
        assert torch.equal(out, O.gated(xin, w, planar=planar))
        rest = torch.ones(shape, dtype=torch.bool, device="cuda")
        rest[cut] = False
        assert torch.all(buf[rest] == 7.0)
    y, z = O.gated(x.view(7, 10, 96), w, save=True)
    assert y.shape == (7, 10, 80) and z.shape == (7, 10, 160)
    p = x.t().contiguous()
    yp = O.gated(p, w, planar=True)
    assert torch.equal(O.gated(p.t(), w).t(), yp)  # planes seen as rows: x's own order
    d1, _ = make(2, 1, 80, dt)
    for a, b in zip(O.gated_backward(d1.expand(70, 80), x, w, z.view(70, 160)),
                    O.gated_backward(d1.expand(70, 80).contiguous(), x, w, z.view(70, 160))):
        assert torch.equal(a, b)


def test_gated_refusals_on_the_card():
    x, _ = make(0, 8, 16, torch.float32)
    w, _ = weight(1, 24, 16, torch.float32, False)
    with pytest.raises(P.MaximError, match="not on the card"):
        O.gated(x, w.cpu())
    with pytest.raises(P.MaximError, match="no gate's"):
        O.gated(x, w[:23])
    with pytest.raises(P.MaximError, match="memory order"):
        O.gated(x, w, out=torch.empty(12, 8, device="cuda").t())
    with pytest.raises(P.MaximError, match="requires a gradient"):
        O.gated(x, w.clone().requires_grad_())
    with pytest.raises(P.MaximError, match="expected"):
        O.gated_backward(x[:, :12].contiguous(), x, w, x)
