"""The 4-bit blocks and the Dense of them on device tensors.

Quantising is exact arithmetic and one rounding that the format defines, so
codes and scales are compared bit for bit with the definition in 64 bits, and
the values that come back with the codes' own. The product's terms are exact in
fp32 (products of two elements have four bits, scales are powers of two), so a
result of k terms is off by k u S at most (u = 2^-24, S the sum of the terms'
magnitudes), and by the activation's and the store's errors of
test_gpu_operators.py."""

import math

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402
from test_gpu_operators import ACTS, SLOPE, TYPES, U, act64, act_error, half, make, near, tiny, values, vec  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()


ELEMENTS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def blocks_of(v):
    """[rows][k] values in 64 bits -> codes [rows][k], scales [rows][blocks], by
    the definition: the nearest element, of two the one of even code."""
    r, k = v.shape
    b = torch.nn.functional.pad(v, (0, -k % 32)).view(r, -1, 32)
    top = b.abs().amax(2)
    bad = ~torch.isfinite(b).all(2)
    top = torch.where(bad, torch.ones_like(top), top)
    # frexp: top = m 2^e with m in [0.5, 1)
    e = torch.where(top > 0, torch.frexp(top).exponent.long() - 1, torch.full_like(top, -1000).long())
    s = torch.clamp(e - 2, min=-127) + 127
    q = torch.ldexp(torch.where(bad[:, :, None], torch.zeros_like(b), b), (127 - s)[:, :, None])
    d = (q.abs()[..., None] - ELEMENTS).abs()
    near_ = d.amin(-1, keepdim=True)
    odd = torch.arange(8) % 2
    code = torch.where(d == near_, odd, 9).argmin(-1)  # even ones first
    code = code + 8 * torch.signbit(torch.where(bad[:, :, None], torch.zeros_like(q), q))
    s = torch.where(bad, torch.full_like(s, 255), s)
    return code.view(r, -1)[:, :k], s


def meant(code, s):
    """The values that they stand for."""
    r, k = code.shape
    v = ELEMENTS[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    scale = torch.where(s == 255, torch.full(s.shape, math.nan, dtype=torch.float64), torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s - 127))
    return v * scale.repeat_interleave(32, 1)[:, :k]


def check_quantize(x, v, planar=False):
    q = O.mx4_quantize(x, planar=planar)
    codes, scales = q.plain()
    code, s = blocks_of(v)
    assert torch.equal(scales.cpu().long(), s)
    got = torch.stack([codes & 15, codes >> 4], -1).view(v.shape[0], -1).cpu().long()
    assert not got[:, v.shape[1]:].any()  # past the last feature
    got = got[:, :v.shape[1]]
    fine = (s != 255).repeat_interleave(32, 1)[:, :v.shape[1]]
    assert torch.equal(got[fine], code[fine])
    want = meant(code, s)
    for dt in TYPES.values():
        y = values(O.mx4_dequantize(q, dtype=dt, planar=planar), planar).reshape(v.shape)
        w = want.to(dt).double()
        assert torch.equal(torch.isnan(y), torch.isnan(w)) and torch.equal(y[fine], w[fine])
    return q, want


SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (5, 255), (64, 256), (65, 257), (63, 1000), (130, 96), (200, 512), (1, 4096),
          (300, 777), (17, 2500)]


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k", SHAPES)
def test_quantize_and_back(rows, k, dt, planar):
    for pad in (0, 3, 8):
        x, v = make(pad, rows, k, dt, planar, pad)
        check_quantize(x, v, planar)


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 63, 64, 97])
@pytest.mark.parametrize("k", [40, 256, 300])
def test_all_bytes_are_written(rows, k):
    # both orders fill the whole storage, and alike: zeros for the rows and
    # features that are not there
    x, _ = make(31, rows, k, torch.bfloat16)
    stored = []
    for t, planar in ((x, False), (x.t().contiguous(), True)):
        q = O.mx4_quantize(t, planar=planar)
        q._data.fill_(0xff)
        O._check(O._L.mxh_mx4_quantize(0, O._stream(0), O._mat(t, "x", 0, planar), q._mat()))
        stored.append(q._data.cpu())
    assert torch.equal(stored[0], stored[1])
    tiles = (k + 255) // 256
    scales = stored[0][q._code_bytes:].view(-1, tiles, 4, 16, 4, 2).permute(0, 4, 3, 1, 5, 2).reshape(-1, tiles * 8)
    assert not scales[rows:].any() and not scales[:, (k + 31) // 32:].any()


def test_every_16_bit_value():
    """Each finite bf16 and fp16 value beside a 6 of every one of some scales,
    so that elements fall on and between all codes, and alone."""
    for dt in (torch.bfloat16, torch.float16):
        every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt)
        every = every[torch.isfinite(every)]
        alone = torch.zeros(every.numel(), 32, dtype=dt)
        alone[:, 5] = every
        check_quantize(alone.cuda(), alone.double())
        x = every[:every.numel() // 31 * 31].view(-1, 31)
        for top in (6.0, 7.5, 4.0, 1.0, 60000.0):
            b = torch.cat([torch.full((x.shape[0], 1), top, dtype=dt), x], 1)
            check_quantize(b.cuda(), b.double())
    # halfway points, and fp32's neighbours of them
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    mid = torch.cat([mid, torch.nextafter(mid, torch.tensor(0.0)), torch.nextafter(mid, torch.tensor(9.0))])
    x = torch.cat([torch.tensor([7.0]), mid, -mid[:4]]).repeat(40, 1) * 2.0 ** torch.arange(-126, 114, 6).float()[:, None]
    check_quantize(x.cuda(), x.double())


def test_far_values():
    """The smallest and largest floats, zeros of both signs, infinities, NaN."""
    x = torch.zeros(12, 96)
    x[0, 3] = 1e-45
    x[1, 40] = -1e-40
    x[2, 7], x[2, 8] = 2.0 ** -126, 2.0 ** -127
    x[3, 9] = 3.4e38
    x[4, 10] = math.inf
    x[5, 70] = -math.inf
    x[6, 33] = math.nan
    x[7] = -0.0
    x[8, :32] = torch.linspace(-3e38, 3e38, 32)
    x[9, 5], x[9, 6] = 2.0 ** -125, 1.75 * 2.0 ** -126
    check_quantize(x.cuda(), x.double())
    check_quantize(x.t().contiguous().cuda(), x.double(), True)


def test_nothing_and_more_dimensions():
    for shape in ((0, 5), (5, 0), (0, 0)):
        x = torch.zeros(shape, device="cuda")
        assert O.mx4_dequantize(O.mx4_quantize(x)).shape == shape
    x = torch.randn(3, 4, 50, device="cuda")
    q = O.mx4_quantize(x)
    assert q.shape == (3, 4, 50)
    y = O.mx4_dequantize(q)
    assert torch.equal(y.view(12, 50), O.mx4_dequantize(O.mx4_quantize(x.view(12, 50))))
    p = x.permute(2, 0, 1)
    assert torch.equal(O.mx4_dequantize(O.mx4_quantize(p, planar=True)), y)
    assert torch.equal(O.mx4_dequantize(O.mx4_quantize(p.contiguous(), planar=True), planar=True), y.permute(2, 0, 1))


# ------------------------------------------------------------- the product


def weights4(seed, n, k):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(n, k, generator=g) / math.sqrt(k)
    q = O.mx4_quantize(w.cuda())
    return q, meant(*blocks_of(w.double()))


def check_dense(rows, k, n, dt, planar, pad, act, residual, bias, seed=0):
    x, xv = make(seed, rows, k, dt, planar, pad)
    q, wv = weights4(seed + 1, n, k)
    b, bv = vec(seed + 2, n, bias) if bias else (None, torch.zeros(n, dtype=torch.float64))
    r, rv = make(seed + 3, rows, n, dt, planar, pad) if residual else (None, 0)
    y = O.mx4_dense(x, q, b, act=act, slope=SLOPE, residual=r, planar=planar)
    xv = meant(*blocks_of(xv))
    zw = xv @ wv.t() + bv
    ze = (k + 1) * U * (xv.abs() @ wv.abs().t()) + U * (zw.abs() + bv.abs())
    want = act64(zw, act)[0] + rv
    err = act_error(zw, ze, act) + 2 * U * want.abs() + (U * rv.abs() if residual else 0)
    near(values(y, planar), want, err + half(dt) * (want.abs() + err) + tiny(dt), "y")


DENSE_SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 257), (2, 33, 5), (3, 128, 48), (7, 777, 130), (16, 512, 640), (1, 4096, 300),
                (17, 96, 100), (64, 64, 64), (65, 72, 129), (100, 1, 100), (128, 256, 128), (129, 257, 257), (200, 40, 300),
                (256, 1024, 512), (300, 2304, 32), (33, 2500, 40), (520, 64, 264), (1030, 32, 96), (16, 8192, 17)]


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", DENSE_SHAPES)
def test_mx4_dense(rows, k, n, dt, planar):
    i = (rows * 7 + k * 3 + n) % 6
    for j, pad in enumerate((0, 8, 3)):
        check_dense(rows, k, n, dt, planar, pad, ACTS[(i + j) % 6], j != 1, (None, dt, torch.float32)[j], seed=j)


BIG_SHAPES = [(2048, 1024, 2048), (1024, 512, 1024), (4095, 777, 1025), (256, 16384, 256), (520, 4096, 4096), (40000, 64, 96),
              (16, 4096, 4096), (17, 4096, 4096), (3000, 256, 3100)]


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("rows,k,n", BIG_SHAPES)
def test_mx4_dense_of_every_tile(rows, k, n, dt, planar):
    """64-bit products of the values that come back, on the card. 8 u S as in
    test_products_of_every_tile."""
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)
    x = torch.randn(*((k, rows) if planar else (rows, k)), generator=g, device="cuda").to(dt)
    w = O.mx4_quantize(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k))
    xv = O.mx4_dequantize(O.mx4_quantize(x, planar=planar), dtype=torch.float32).double()
    wv = O.mx4_dequantize(w).double()
    y = O.mx4_dense(x, w, planar=planar)
    want = xv @ wv.t()
    tol = 8 * U * (xv.abs() @ wv.abs().t()) + half(dt) * want.abs() * 1.01 + tiny(dt)
    off = ((y.t() if planar else y).double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


def test_far_scales_and_rows_of_nan():
    """Blocks near both ends of the scales' range, and rows with NaN and
    infinity, which keep to themselves."""
    for rows in (5, 70):
        x, xv = make(1, rows, 300, torch.float32)
        q, wv = weights4(2, 90, 300)
        for s in (2.0 ** -120, 2.0 ** -100, 2.0 ** 100, 2.0 ** 120):
            want = meant(*blocks_of(xv * s)) @ wv.t()
            size = meant(*blocks_of(xv * s)).abs() @ wv.abs().t()
            near(O.mx4_dense(x * s, q).double().cpu(), want, 301 * U * size + U * want.abs() + 1e-37, "far")
        clean = O.mx4_dense(x, q)
        x[1, 5] = math.nan
        x[3, 299] = -math.inf
        y = O.mx4_dense(x, q)
        keep = [i for i in range(rows) if i not in (1, 3)]
        assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.equal(y[keep], clean[keep])


def test_mx4_dense_of_nothing_slices_and_places():
    q, wv = weights4(1, 24, 16)
    x, _ = make(0, 40, 16, torch.float32)
    b, bv = vec(2, 24, torch.float32)
    assert O.mx4_dense(x[:0], q, b).shape == (0, 24)
    e = O.mx4_quantize(torch.zeros(24, 0, device="cuda"))
    for rows in (3, 40):
        assert torch.equal(O.mx4_dense(x[:rows, :0], e, b), b.expand(rows, 24))
    for rows in (9, 40):
        row = x[:1]
        assert torch.equal(O.mx4_dense(row.expand(rows, 16), q), O.mx4_dense(row.expand(rows, 16).contiguous(), q))
        buf = torch.full((rows + 4, 40), 7.0, device="cuda")
        out = O.mx4_dense(x[:rows], q, out=buf[2:rows + 2, 5:29])
        assert torch.equal(out, O.mx4_dense(x[:rows], q))
        rest = torch.ones_like(buf, dtype=torch.bool)
        rest[2:rows + 2, 5:29] = False
        assert torch.all(buf[rest] == 7.0)
        r = torch.randn(rows, 24, device="cuda")
        want = O.mx4_dense(x[:rows], q, residual=r)
        assert torch.equal(O.mx4_dense(x[:rows], q, residual=r, out=r), want)
    assert O.mx4_dense(x.view(5, 8, 16), q).shape == (5, 8, 24)
    # x in another order than y
    xt = x.t().contiguous()
    assert torch.equal(O.mx4_dense(xt.t(), q).t(), O.mx4_dense(xt, q, planar=True))


@pytest.mark.parametrize("planar", [False, True])
def test_the_longest_lines(planar):
    """As many features as a tile's offsets reach, and one block of 32 past
    them refused: sums of a few powers of two, which are exact."""
    k, at = (1 << 24) - 256, [0, 31, 32, (1 << 23) + 5, (1 << 24) - 300, (1 << 24) - 257]
    w = torch.zeros(4, k, dtype=torch.bfloat16, device="cuda")
    for j, c in enumerate(at):
        w[j % 4, c] = 2.0 ** j
    q = O.mx4_quantize(w)
    for rows in (3, 20):
        x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
        x[:, at] = torch.tensor([2.0 ** (i % 5) for i in range(rows)], dtype=torch.bfloat16, device="cuda")[:, None]
        y = O.mx4_dense(x.t().contiguous() if planar else x, q, planar=planar)
        want = x[:, :1].float() * torch.tensor([1.0 + 16, 2.0 + 32, 4.0, 8.0], device="cuda")
        assert torch.equal((y.t() if planar else y).float(), want)
    with pytest.raises(P.MaximError, match="out of range"):
        O.mx4_quantize(torch.zeros(1, k + 32, dtype=torch.bfloat16, device="cuda"))


def test_captured():
    x = torch.randn(100, 512, device="cuda").bfloat16()
    q = O.mx4_quantize(torch.randn(300, 512, device="cuda"))
    want = [O.mx4_dense(x, q), O.mx4_dense(x[:2], q), O.mx4_dequantize(O.mx4_quantize(x))]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = [O.mx4_dense(x, q), O.mx4_dense(x[:2], q), O.mx4_dequantize(O.mx4_quantize(x))]
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        O.mx4_dense(x, q)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals_on_the_card():
    x = torch.zeros(8, 16, device="cuda")
    q = O.mx4_quantize(torch.zeros(24, 16, device="cuda"))
    for call, match in ((lambda: O.mx4_dense(x, x), "not an Mx4"),
                        (lambda: O.mx4_dequantize(x), "not an Mx4"),
                        (lambda: O.mx4_dense(x[:, :15].contiguous(), q), "expected"),
                        (lambda: O.mx4_quantize(x.cpu()), "not a tensor on the card"),
                        (lambda: O.mx4_quantize(x.double()), "not float32"),
                        (lambda: O.mx4_dense(x, q, act="tanh"), "unknown activation"),
                        (lambda: O.mx4_dense(x, q, torch.zeros(23, device="cuda")), "bias"),
                        (lambda: O.mx4_dense(x, q, out=torch.zeros(8, 16, device="cuda")), "expected")):
        with pytest.raises(P.MaximError, match=match):
            call()
