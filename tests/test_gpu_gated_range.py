"""The gated Dense's backward pass in fp16 where dz, a product of three values,
leaves fp16's range and the gradients do not.

dz = (dy c act'(a) | dy act(a)) goes to the products rounded to fp16 as it is
where its largest finite magnitude `top` is between 1 and 65520, and else times
the power of two that takes it into [2^14, 2^15). An element is then off by
half a step, 2^-11 of itself, or by half of fp16's smallest step, 2^-25, which
is 2^-25 / (2^14 / top) = 2^-39 top of the scaled ones at most, and 2^-25 of the
others. The rest as test_gpu_gated.py has it."""

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from test_gpu_operators import ACTS, SLOPE, U, act64, act_error, half, near, tiny, values  # noqa: E402

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()


def make(seed, rows, cols, size, planar=False, flip=False, pad=0):
    """[rows][cols] fp16 values of this size, in planar order a transposed
    view's storage; and the same values in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    v = (torch.randn(rows, cols, generator=g) * size).clamp(-6e4, 6e4).to(F16)
    t = (v.t() if planar or flip else v).contiguous()
    wide = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=F16)
    wide[:, :t.shape[1]] = t
    t = wide.cuda()[:, :t.shape[1]]
    return (t.t() if flip else t), v.double()


def check(rows, k, n, sizes, planar=False, wt=False, act="silu", pad=0, db_dt=torch.float32, mask=None, finite=True):
    """sizes: of dy, x, w and z."""
    dy, dyv = make(0, rows, n, sizes[0], planar, pad=pad)
    x, xv = make(1, rows, k, sizes[1], planar, pad=pad)
    w, wv = make(2, 2 * n, k, sizes[2], flip=wt)
    z, zv = make(3, rows, 2 * n, sizes[3], planar, pad=pad)
    if mask is not None:
        mask(dyv, zv)
        for t, v in ((dy, dyv), (z, zv)):
            t.copy_(v.t() if planar else v)
    a, c = zv[:, :n], zv[:, n:]
    f, g = act64(a, act)
    dz = torch.cat([dyv * c * g, dyv * f], 1)
    top = float(dz.abs()[dz.isfinite()].max())
    dze = torch.cat([(dyv * c).abs() * 6e-7 * (1 + a.abs()), dyv.abs() * act_error(a, 0 * a, act)], 1) + 3 * U * dz.abs()
    eb = dze.sum(0) + rows * U * dz.abs().sum(0)
    dze = dze + half(F16) * dz.abs() + (2 ** -25 if 1 <= top < 65520 else 2 ** -39 * top)
    dx, dw, db = O.gated_backward(dy, x, w, z, act=act, slope=SLOPE, planar=planar, db_dtype=db_dt)
    got = values(dx, planar), dw.double().cpu(), db.double().cpu()
    for i, (want, mag, e, terms) in enumerate(((dz @ wv, (dz.abs() + dze) @ wv.abs(), dze @ wv.abs(), 2 * n),
                                              (dz.t() @ xv, (dz.abs() + dze).t() @ xv.abs(), dze.t() @ xv.abs(), rows))):
        tol = e + (terms + 1) * U * mag
        if finite:
            # what is asked of the call fits fp16, with room for its error
            assert float((want.abs() + 2 * tol).max()) < 65504
        keep = want.isfinite()
        assert bool(keep.all()) or not finite
        assert not got[i][~keep].isfinite().any()
        near(got[i][keep], want[keep], (tol + half(F16) * (want.abs() + tol) + tiny(F16))[keep], ("dx", "dw")[i])
    wb = dz.sum(0)
    if finite:
        near(got[2], wb, eb + half(db_dt or F16) * (wb.abs() + eb) + tiny(db_dt or F16), "db")
    return dx, dw, db, top


# dy, x, w, z: dz past 65504, dz in which most is below fp16's normal range, dz in range
LARGE, SMALL, PLAIN = (3e4, 1e-3, 1e-3, 4.0), (1e-4, 1.0, 30.0, 0.02), (1.0, 1.0, 0.1, 1.0)
SHAPES = [(1, 64, 64), (1, 4096, 512), (3, 33, 5), (17, 96, 100), (130, 64, 64), (129, 65, 257), (300, 256, 32),
          (1030, 32, 96), (64, 520, 300), (512, 512, 512), (4096, 64, 64), (2500, 72, 24)]


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("sizes", [LARGE, SMALL, PLAIN], ids=["large", "small", "plain"])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_gradients_fit_where_dz_does_not(rows, k, n, sizes, planar):
    for j, (wt, pad, act) in enumerate([(False, 0, "silu"), (True, 3, "gelu")]):
        top = check(rows, k, n, sizes, planar, wt, act, pad, (torch.float32, None)[j] if sizes is not LARGE else torch.float32)[3]
        assert top > 65520 if sizes is LARGE else top < 0.01 if sizes is SMALL else 0 < top < 65520


@pytest.mark.parametrize("act", ACTS)
def test_large_dz_of_every_activation(act):
    for planar in (False, True):
        check(96, 80, 72, LARGE, planar, act=act)
        check(96, 80, 72, SMALL, planar, act=act)


@pytest.mark.parametrize("planar", [False, True])
def test_infinities_do_not_choose_the_scale(planar):
    """A row that is infinite or NaN stays so, and the others are as exact as
    without it; where everything else is nothing, that is what it stays."""
    for sizes in (LARGE, SMALL, PLAIN, (0.0, 1.0, 1.0, 1.0)):
        def mask(dyv, zv):
            dyv[5] = float("inf")
            dyv[40] = float("nan")
        check(96, 80, 72, sizes, planar, mask=mask, finite=False)


def test_large_dz_in_a_graph():
    """The scale is the replay's own, not the capture's."""
    rows, k, n = 200, 96, 64
    calls = [[make(i, *s)[0] for i, s in enumerate(((rows, n, z[0]), (rows, k, z[1]), (2 * n, k, z[2]), (rows, 2 * n, z[3])))]
             for z in (LARGE, PLAIN, SMALL)]
    want = [O.gated_backward(*c) for c in calls]
    held = [t.clone() for t in calls[1]]
    O.gated_backward(*held)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = O.gated_backward(*held)
    for i in (0, 1, 2, 0, 0, 2, 1):
        for h, t in zip(held, calls[i]):
            h.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)
        assert all(bool(t.isfinite().all()) for t in got[:2])


def test_many_planes():
    """More blocks in dz's pass than one reads the magnitudes of by itself."""
    check(40, 16, 6000, (3e3, 1e-3, 1e-4, 4.0), True)
    check(40, 16, 6000, (1e-4, 1.0, 3.0, 0.02), True)
