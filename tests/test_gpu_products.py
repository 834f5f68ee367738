"""Dense on device tensors where its kernels' addressing and the choice between
them matter: long lines, operands of different memory orders, few features.
References are 64-bit products on the card."""

import math

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402
from test_gpu_operators import TYPES, U, check_layernorm, check_ln_backward, half, tiny  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()
    yield
    torch.cuda.empty_cache()


def rand(gen, a, b, dt, std=1.0):
    return (torch.randn(a, b, generator=gen, device="cuda") * std).to(dt)


def close(got, want, size, terms, dt, what):
    """Within a result's own rounding and `terms` roundings of its sum. Each of
    those is half a step at most of a partial sum of random signs, which
    reaches sqrt(terms) of a product's deviation d: together a walk of about
    terms d u / 2 where S, the sum of the magnitudes, is 0.64 terms d: 8 u S
    leaves ten deviations (and terms u S holds always).
    But for the fewest terms: of an fp32 product of three bf16 parts (of
    operands in [1, 2) |m| <= 2^-8 and |l| <= 2^-17) m l + l m + l l, up to
    2^-24 of it, is left out, and the matrix cores' last addition may be off by
    a whole step, 2^-23, those before by a 2^-6 of that together: 3.04 u."""
    tol = min(max(terms, 4), 8) * U * size + half(dt) * want.abs() * 1.01 + tiny(dt)
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), (what, float(off.max()))


def long_sum(a, b, step=1 << 21):
    """a b^T and |a| |b|^T over the last axis, in 64 bits and in pieces."""
    want = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device="cuda")
    size = want.clone()
    for i in range(0, a.shape[1], step):
        p, q = a[:, i:i + step].double(), b[:, i:i + step].double()
        want += p @ q.t().contiguous()
        size += p.abs() @ q.abs().t().contiguous()
    return want, size


@pytest.mark.parametrize("dt,k,n,more", [(torch.bfloat16, 128, 136, 8), (torch.float16, 72, 40, 3),
                                         (torch.float32, 40, 72, 8)], ids=["bf16", "f16", "f32"])
def test_planes_of_many_positions(dt, k, n, more):
    """Planes past 2^24 positions, where a tile's lines are further apart than
    31 bits reach: the results at both ends and in between, dw in full."""
    gen = torch.Generator(device="cuda").manual_seed(k)
    rows = (1 << 24) + more
    x, dy = rand(gen, k, rows, dt), rand(gen, n, rows, dt)
    w = rand(gen, n, k, dt, 1 / math.sqrt(k))
    b = rand(gen, 1, n, dt).view(n)
    at = torch.cat([torch.arange(700), torch.arange((1 << 23) - 300, (1 << 23) + 300), torch.arange(rows - 700, rows),
                    torch.randint(0, rows, (500,), generator=torch.Generator().manual_seed(1))]).cuda()
    w64 = w.double()
    y = O.dense(x, w, b, planar=True)
    xs = x[:, at].double()
    close(y[:, at], w64 @ xs + b.double()[:, None], w64.abs() @ xs.abs() + b.double().abs()[:, None], k + 1, dt, "y")
    del y
    dx, dw, db = O.dense_backward(dy, x, w, planar=True)
    ds = dy[:, at].double()
    close(dx[:, at], w64.t().contiguous() @ ds, w64.t().abs().contiguous() @ ds.abs(), n, dt, "dx")
    want, size = long_sum(dy, x)
    close(dw, want, size, rows, dt, "dw")
    close(db, dy.double().sum(1), dy.double().abs().sum(1), rows, dt, "db")


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("n", [1, 3, 8, 16, 17])
def test_few_features_over_many_positions(n, dt):
    """A planar Dense to few features, and from few: sums over every position
    are cut over the card, those over features are not."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    for rows, k in (((1 << 17) + 8, 33), (448 * 640, 32), ((1 << 17) + 3, 64)):
        for a, b in ((k, n), (n, k)):
            x, dy = rand(gen, a, rows, dt), rand(gen, b, rows, dt)
            w = rand(gen, b, a, dt, 1 / math.sqrt(a))
            y = O.dense(x, w, planar=True)
            dx, dw, db = O.dense_backward(dy, x, w, planar=True)
            w64, x64, d64 = w.double(), x.double(), dy.double()
            close(y, w64 @ x64, w64.abs() @ x64.abs(), a, dt, "y")
            close(dx, w64.t().contiguous() @ d64, w64.t().abs().contiguous() @ d64.abs(), b, dt, "dx")
            want, size = long_sum(dy, x)
            close(dw, want, size, rows, dt, "dw")
            close(db, d64.sum(1), d64.abs().sum(1), rows, dt, "db")


def test_one_product_in_fp32():
    """A product of three-part operands alone: within 3.04 u of itself, as
    close() derives it; exact where the parts are."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    for span in (1.0, 0.01):
        x = 1 + span * torch.rand(1 << 18, 1, generator=gen, device="cuda")
        w = 1 + span * torch.rand(256, 1, generator=gen, device="cuda")
        want = x.double() @ w.double().t()
        off = float((O.dense(x, w).double() / want - 1).abs().max())
        assert off <= 3.04 * U * 1.0001 < 1.82e-7, off / U
    x, w = x.bfloat16().float(), w.bfloat16().float()
    assert torch.equal(O.dense(x, w), x @ w.t())


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("k,n", [(1, 7), (1, 1), (7, 1)])
def test_one_feature_forward_and_backward(k, n, planar):
    """What the forward call gives, its backward call takes beside ordinary
    gradients."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    rows, dt = 100, torch.float32
    x, dy = (rand(gen, *((c, rows) if planar else (rows, c)), dt) for c in (k, n))
    w = rand(gen, n, k, dt)
    y, z = O.dense(x, w, act="gelu", planar=planar, save=True)
    assert y.is_contiguous() and z.is_contiguous() and y.shape == dy.shape
    dx, dw, db = O.dense_backward(dy, x, w, z=z, act="gelu", planar=planar)
    x64 = (x.t() if planar else x).double().cpu().requires_grad_()
    w64 = w.double().cpu().requires_grad_()
    z64 = x64 @ w64.t()
    y64 = z64 * 0.5 * torch.special.erfc(-z64 / math.sqrt(2))
    y64.backward((dy.t() if planar else dy).double().cpu())
    # sums of terms + 1 roundings, z's u |z| times a slope below 1.2, and the
    # fits: gelu within 3e-7 (1 + |z|), its derivative within 6e-7 (1 + |z|)
    xa, wa, za = x64.detach().abs(), w64.detach().abs(), z64.detach().abs()
    da = (dy.t() if planar else dy).double().cpu().abs()
    ze = (k + 4) * U * (xa @ wa.t())
    dze = da * (6e-7 * (1 + za) + 0.8 * ze) + 2 * U * da
    for got, want, tol in ((y.t() if planar else y, y64.detach(), 1.2 * ze + 3e-7 * (1 + za) + 2 * U * za),
                           (dx.t() if planar else dx, x64.grad, dze @ wa + (n + 4) * U * 1.2 * (da @ wa)),
                           (dw, w64.grad, dze.t() @ xa + (rows + 4) * U * 1.2 * (da.t() @ xa))):
        assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_relu_at_the_ends(rows, dt):
    """LeakyReLU of slope 0 is ReLU: 0 at minus infinity too, NaN at NaN; any
    other slope keeps the infinity."""
    one = torch.ones(1, 1, dtype=dt, device="cuda")
    z = torch.tensor([-float("inf"), -60000.0, -1.0, -0.0, 0.0, 2.0, float("inf"), float("nan")], dtype=dt, device="cuda")
    x = z.view(-1, 1).repeat(rows, 1)
    want = torch.nn.functional.relu(z.float()).to(dt)
    got = O.dense(x, one, act="lrelu", slope=0.0).view(rows, -1)
    assert torch.equal(got[:, :7], want[:7].expand(rows, 7)) and torch.isnan(got[:, 7]).all()
    got = O.dense(x, one, act="lrelu", slope=0.5).view(rows, -1)
    assert torch.equal(got[:, :7], torch.where(z < 0, 0.5 * z, z)[:7].expand(rows, 7)) and torch.isnan(got[:, 7]).all()
    assert torch.equal(O.dense(x, one, act="lrelu", slope=-0.5).view(rows, -1)[:, 0], z[6].expand(rows))


def test_tangents_are_refused_on_the_card():
    x, w = torch.ones(8, 16, device="cuda"), torch.ones(4, 16, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, x)
        for call in (lambda: O.dense(d, w), lambda: O.dense(w, d), lambda: O.layernorm(d, w[0])):
            with pytest.raises(P.MaximError, match="forward-mode tangent"):
                call()
        assert torch.equal(O.dense(x, w), torch.full((8, 4), 16.0, device="cuda"))


def test_what_out_overwrites_is_known_to_autograd():
    """A result written over a tensor that an earlier operation kept for its
    backward pass: torch says so instead of using the new values."""
    s, w = torch.ones(16, device="cuda"), torch.eye(16, device="cuda")

    def layernorm(t):
        O.layernorm(t, s, out=t)

    def dense(t):
        O.dense(torch.ones_like(t), w, residual=t, out=t)

    def layernorm_backward(t):
        _, m, r = O.layernorm(torch.ones_like(t), s, stats=True)
        O.layernorm_backward(t, torch.ones_like(t), s, m, r, out=t)

    for call in (layernorm, dense, layernorm_backward):
        p = torch.randn(8, 16, device="cuda", requires_grad=True)
        y = p.exp()  # keeps its result
        with torch.no_grad():
            before = y._version
            call(y)
            assert y._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        with torch.inference_mode():
            call(torch.randn(8, 16, device="cuda"))


# sizes that, with x in another memory order than y and dy, reach the tiles that
# matrices of one order do not (test_ops_launches.py holds that every kernel is
# reached); rows, k, n
MIXED_SHAPES = [(100, 40, 72), (4095, 1023, 2049), (2048, 512, 2048), (2048, 512, 4096), (256, 8192, 256), (40000, 64, 96),
                (4287, 6971, 194), (24450, 783, 1028), (612, 2826, 4389), (2284, 633, 7599), (31971, 707, 209)]


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", MIXED_SHAPES)
def test_products_of_mixed_orders(rows, k, n, dt, wt, planar):
    """x in one memory order, y and dy in the other, into and out of buffers
    of their own width and wider."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    for pad in (0, 3):
        # the call's order is y's; x is a view of the other
        x = rand(gen, *((rows, k + pad) if planar else (k, rows + pad)), dt)[:, :k if planar else rows].t()
        dy = rand(gen, *((n, rows + pad) if planar else (rows, n + pad)), dt)[:, :rows if planar else n]
        w = rand(gen, k, n, dt, 1 / math.sqrt(k)).t() if wt else rand(gen, n, k, dt, 1 / math.sqrt(k))
        y = O.dense(x, w, planar=planar, out=torch.empty_like(dy))
        assert y.stride() == dy.stride() or y.is_contiguous()
        dx, dw, db = O.dense_backward(dy, x, w, planar=planar)
        assert dx.shape == x.shape and dx.t().is_contiguous()
        x64, d64, w64 = ((t.t() if planar else t).double().contiguous() for t in (x, dy, w.t() if planar else w))
        for got, a, b, terms, what in ((y.t() if planar else y, x64, w64.t(), k, "y"), (dx.t() if planar else dx, d64, w64, n, "dx"),
                                       (dw, d64.t(), x64, rows, "dw")):
            close(got, a @ b, a.abs() @ b.abs(), terms, dt, (what, pad))
        close(db, d64.sum(0), d64.abs().sum(0), rows, dt, "db")


# planar channels past those that registers hold, positions
LOOP_SHAPES = [(1, 1025), (7, 1025), (100, 1500), (1000, 2049), (64, 3000), (129, 5000)]


@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,cols", LOOP_SHAPES)
def test_layernorm_of_many_planes(rows, cols, dt):
    for pad in (0, 8, 3):
        check_layernorm(rows, cols, dt, True, pad, dt if pad else torch.float32, seed=pad)
        check_ln_backward(rows, cols, dt, True, pad, dt if pad else torch.float32, pad == 8, seed=pad)
    x = torch.randn(cols, rows + 3, device="cuda").to(dt)[:, :rows]
    s = torch.randn(cols, device="cuda").to(dt)
    want = O.layernorm(x, s, planar=True)
    assert torch.equal(O.layernorm(x, s, planar=True, out=x), want)
