"""The block operators used together on the card: a gated feed-forward block
trained for a step and served in 4 bits, captured, on several streams, beside
the executor, and with offsets past 32 bits."""

import math

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402
from test_gpu_operators import TYPES, U, act64, half, make, values, vec, weight  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()


NAMES = ["s", "b", "w", "bw", "v", "bv"]


def parameters(c, hidden, dt):
    return {"s": vec(1, c, dt, 0.1, 1.0)[0], "b": vec(2, c, dt, 0.1)[0], "w": weight(3, 2 * hidden, c, dt, False)[0],
            "bw": vec(4, 2 * hidden, dt, 0.1)[0], "v": weight(5, c, hidden, dt, False)[0], "bv": vec(6, c, dt, 0.1)[0]}


def forward(x, p, planar):
    h, m, r = O.layernorm(x, p["s"], p["b"], planar=planar, stats=True)
    a, z = O.gated(h, p["w"], p["bw"], planar=planar, save=True)
    return O.dense(a, p["v"], p["bv"], residual=x, planar=planar), (h, m, r, a, z)


def backward(dy, x, p, kept, planar):
    h, m, r, a, z = kept
    da, dv, dbv = O.dense_backward(dy, a, p["v"], planar=planar)
    dh, dw, dbw = O.gated_backward(da, h, p["w"], z, planar=planar)
    dx, ds, db = O.layernorm_backward(dh, x, p["s"], m, r, add=dy, planar=planar)
    return dx, [ds, db, dw, dbw, dv, dbv]


def step(x, dy, p, planar, max_norm):
    y, kept = forward(x, p, planar)
    dx, grads = backward(dy, x, p, kept, planar)
    norm = O.clip_grads(grads, max_norm)
    return [y, dx, norm] + grads


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("dt", TYPES.values(), ids=TYPES)
def test_a_training_step(dt, planar):
    """LayerNorm, gated Dense, Dense with the residual, their gradients and the
    clipping, against torch's autograd over the formula in 64 bits. About ten
    stored results lie between the input and a gradient, each within a few half
    steps of a value of order one and weights of norm about one: 2-norms agree
    to 24 half steps of the type (fp32: to 64, for the sums), and the norm too."""
    c, hidden, rows = 96, 136, 150
    x, xv = make(0, rows, c, dt, planar)
    dy, dyv = make(9, rows, c, dt, planar)
    p = parameters(c, hidden, dt)
    q = {k: p[k].double().cpu().requires_grad_() for k in NAMES}
    xr = xv.clone().contiguous().requires_grad_()
    h = torch.nn.functional.layer_norm(xr, (c,), q["s"], q["b"], 1e-6)
    z = h @ q["w"].t() + q["bw"]
    yr = (act64(z[:, :hidden], "silu")[0] * z[:, hidden:]) @ q["v"].t() + q["bv"] + xr
    want = torch.autograd.grad((yr * dyv).sum(), [xr] + [q[k] for k in NAMES])
    norm = math.sqrt(sum(float((g ** 2).sum()) for g in want[1:]))
    bar = half(dt) * (64 if dt == torch.float32 else 24)
    y, dx, n, *grads = step(x, dy, p, planar, norm / 4)
    assert abs(float(n) - norm) <= bar * norm
    got = [values(y, planar), values(dx, planar)] + [g.double().cpu() for g in grads]
    for a, b in zip(got, [yr.detach(), want[0]] + [g / 4 for g in want[1:]]):
        assert float((a - b).norm() / b.norm()) <= bar


def test_captured_and_replayed_on_two_streams():
    """The step captured into two graphs with workspaces of their own, replayed
    in turn on two streams, with eager steps in between: the eager step's bits
    every time."""
    dt = torch.bfloat16
    p = parameters(96, 200, dt)
    xs = [make(20 + i, 150, 96, dt)[0] for i in range(2)]
    dys = [make(30 + i, 150, 96, dt)[0] for i in range(2)]
    q = O.mx4_quantize(p["w"])

    def both(i):
        return step(xs[i], dys[i], p, False, 0.5) + [O.mx4_dense(xs[i], q, act="silu")]

    want = [both(0), both(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for i in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(both(i))
        graphs.append(g)
    for k in range(4):
        for o in outs[0] + outs[1]:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = both(k % 2)
        torch.cuda.synchronize()
        for a, b in zip(outs[0] + outs[1] + eager, want[0] + want[1] + want[k % 2]):
            assert torch.equal(a, b), k


def test_on_another_stream_than_the_default():
    dt = torch.float32
    p = parameters(64, 96, dt)
    x, dy = make(1, 70, 64, dt)[0], make(2, 70, 64, dt)[0]
    want = step(x, dy, p, False, 0.5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = step(x, dy, p, False, 0.5)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("planar", [False, True])
def test_served_in_four_bits(planar):
    """The block with its weights in 4-bit blocks, a token and a prompt: each
    product is that of the values that the blocks stand for."""
    dt, c, hidden = torch.bfloat16, 192, 320
    p = parameters(c, hidden, dt)
    w, v = O.mx4_quantize(p["w"]), O.mx4_quantize(p["v"])
    for rows in (1, 40):
        x, xv = make(rows, rows, c, dt, planar)
        h = O.layernorm(x, p["s"], p["b"], planar=planar)
        z = O.mx4_dense(h, w, p["bw"], planar=planar)
        a, b = (z[:hidden], z[hidden:]) if planar else (z[:, :hidden], z[:, hidden:])
        g = (torch.nn.functional.silu(a.float()) * b.float()).to(dt)
        y = O.mx4_dense(g, v, p["bv"], residual=x, planar=planar)
        meant = lambda t: values(O.mx4_dequantize(O.mx4_quantize(t, planar=planar), dtype=torch.float32, planar=planar), planar)  # noqa: E731
        wv, vv = (O.mx4_dequantize(q, dtype=torch.float32).double().cpu() for q in (w, v))
        for got, inp, m, bias, res in ((z, h, wv, p["bw"], 0), (y, g, vv, p["bv"], xv)):
            i = meant(inp)
            want = i @ m.t() + bias.double().cpu() + res
            tol = (i.shape[1] + 3) * U * (i.abs() @ m.abs().t() + want.abs() + 1) + half(dt) * want.abs() * 1.01
            assert bool(((values(got, planar) - want).abs() <= tol).all())


def test_offsets_past_32_bits():
    """Rows and gradients whose elements lie past 2^32 bytes and 2^31 elements
    of their buffers."""
    dt = torch.bfloat16
    n, k, ld, rows = 64, 96, 1 << 15, 70000  # 2.3e9 elements, 4.6 GB
    buf = torch.zeros(rows, ld, dtype=dt, device="cuda")
    x = buf[:, 100:100 + k]
    w, _ = weight(1, 2 * n, k, dt, False)
    ends = torch.tensor([0, 1, 32767, 32768, 65535, 65536, rows - 2, rows - 1], device="cuda")
    x[ends] = torch.randn(8, k, device="cuda").to(dt)
    few = x[ends].contiguous()
    y, z = O.gated(x, w, save=True)
    y8, z8 = O.gated(few, w, save=True)
    out = O.gated(x, w, out=buf[:, 1000:1000 + n])
    wq = O.mx4_quantize(w)
    q8, m8 = O.mx4_dense(few, wq), O.mx4_dequantize(O.mx4_quantize(few))
    m, q = O.mx4_dequantize(O.mx4_quantize(x)), O.mx4_dense(x, wq)
    dy = buf[:, 2000:2000 + n]
    dy[ends] = torch.randn(8, n, device="cuda").to(dt)
    dx, dw, db = O.gated_backward(dy, x, w, z)
    dx8, dw8, db8 = O.gated_backward(dy[ends].contiguous(), few, w, z8)
    # the same sums in other tiles' orders
    for a, b in ((y[ends], y8), (z[ends], z8), (out[ends], y8), (q[ends], q8), (dx[ends], dx8), (dw, dw8), (db, db8)):
        assert float((a.float() - b.float()).norm()) <= 2 * half(dt) * float(b.float().norm())
    assert torch.equal(m[ends], m8)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[ends] = False
    assert not y[rest].any() and not q[rest].any() and not dx[rest].any() and not m[rest].any()
    assert not buf[:, 1000 + n:2000].any() and not buf[:, 200:1000].any()
    del y, z, out, m, q, dy, dx, x
    g = buf.view(-1)[:(1 << 31) + 70001]
    g.zero_()
    g[5], g[-1], g[1 << 31], g[(1 << 31) - 1] = 3.0, 4.0, 12.0, 84.0  # 3, 4, 12, 84: of norm 85
    assert float(O.clip_grads([g], 42.5)) == 85.0
    assert [float(g[i]) for i in (5, -1, 1 << 31, (1 << 31) - 1)] == [1.5, 2.0, 6.0, 42.0]
    assert int((g != 0).sum()) == 4


def test_beside_the_executor():
    from conftest import smooth_image, weights
    from maxim_amd import hip as H
    plan = P.Plan(weights("S-1"), 64, 64)
    gpu = H.Gpu(plan)
    img = smooth_image(64, 64)
    first = gpu.run(img)
    x, _ = make(0, 64 * 64, 32, torch.float32, True)
    w, _ = weight(1, 64, 32, torch.float32, False)
    y = O.gated(x, w, planar=True)
    q = O.mx4_dense(x, O.mx4_quantize(w), planar=True)
    assert (gpu.run(img) == first).all()
    assert torch.equal(O.gated(x, w, planar=True), y) and torch.equal(O.mx4_dense(x, O.mx4_quantize(w), planar=True), q)
    gpu.close()
