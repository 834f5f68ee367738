"""The gradients' global norm and clipping on device tensors against 64 bits.

The norm: squares and sums in 64 bits, whose roundings are 2^-53 of a sum of
positive terms each, far below fp32's half step u = 2^-24; the square root and
the one rounding to fp32 leave u N (1e-12 besides). Clipping multiplies by a
factor that is the fp32 quotient of max_norm and N (off by u, and by N's u)
and rounds once in fp32 and once to the tensor's type: 3 u |g f| + h |g f|."""

import math

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402
from test_gpu_operators import TYPES, U, half, near, tiny  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()


def make(sizes, types, seed=0, std=1.0, shift=0):
    """Tensors of these sizes, `shift` elements into buffers of their own."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = types[i % len(types)]
        v = torch.randn(n + shift, generator=g) * (std * (1 + i % 3))
        out.append(v.to(dt).cuda()[shift:])
    return out


def norm64(grads):
    return math.sqrt(math.fsum(float((g.double().cpu() ** 2).sum()) for g in grads))


def check_clip(grads, max_norm, out=None):
    before = [g.clone() for g in grads]
    want = norm64(before)
    norm = O.clip_grads(grads, max_norm, out=out)
    assert norm.shape == () and norm.dtype == torch.float32
    # a norm past the largest fp32 value (300 elements of 2e37: sqrt(300) 2e37 =
    # 3.464e38, and fp32 ends at 3.403e38) is infinity, and nothing is scaled
    past = want > torch.finfo(torch.float32).max
    assert float(norm) == math.inf if past else abs(float(norm) - want) <= (U + 1e-12) * want
    got = grads if out is None else out
    for b, g in zip(before, got):
        if past or float(norm) <= max_norm:
            assert torch.equal(b.view(torch.uint8), g.view(torch.uint8))
            continue
        w = b.double().cpu() * (max_norm / want)
        near(g.double().cpu(), w, 3 * U * w.abs() + half(b.dtype) * w.abs() * (1 + 4 * U) + tiny(b.dtype), "clipped")
    if out is not None:
        for b, g in zip(before, grads):
            assert torch.equal(b, g)
    return norm


LISTS = [[1], [7], [0, 5, 0], [8192], [8193, 4095, 4097], [64, 64, 8192, 128, 4096, 64], [1] * 300, [100003, 3, 1 << 20],
         list(range(1, 130)), [(1 << 22) + 5, 1, 16384 * 3 + 1] * 3, [513] * 128, [40000] * 129]


@pytest.mark.parametrize("types", [("f32",), ("bf16",), ("f16",), ("bf16", "f32", "f16")], ids="-".join)
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: "%dx%d" % (len(s), max(s)))
def test_norm_and_clip(sizes, types):
    types = [TYPES[t] for t in types]
    for shift in (0, 1, 8):
        grads = make(sizes, types, shift=shift, std=0.5)
        want = norm64(grads)
        assert abs(float(O.grad_norm(grads)) - want) <= (U + 1e-12) * want
        check_clip([g.clone() for g in grads], want * 0.37)
        check_clip([g.clone() for g in grads], want * 2.0)
        check_clip(grads, want * 0.37, out=[torch.empty_like(g) for g in grads])
        check_clip(grads, want * 2.0, out=[torch.empty_like(g) for g in grads])


def test_what_lies_beside_is_not_written():
    buf = torch.ones(100, device="cuda")
    g = buf[3:40]
    O.clip_grads([g], 0.5)
    assert torch.all(buf[:3] == 1) and torch.all(buf[40:] == 1) and torch.all(g < 1)


def test_far_values():
    """Squares beyond fp32's range both ways, infinities and NaN."""
    for dt in (torch.float32, torch.bfloat16):
        for v in (1e-38, 1e-30, 1e25, 2e37):
            g = torch.full((300,), v, dtype=dt, device="cuda")
            check_clip([g], float(norm64([g])) * 0.25)
    g = torch.full((10,), 3e38, device="cuda")  # 9.5e38: past fp32's range
    n = O.clip_grads([g], 1.0)
    assert float(n) == math.inf and torch.all(g == 3e38)
    for bad in (math.inf, -math.inf, math.nan):
        g = torch.ones(5000, device="cuda")
        g[4321] = bad
        h = torch.ones(70, dtype=torch.bfloat16, device="cuda")
        before = g.clone()
        n = O.clip_grads([h, g], 1e-3)
        assert not math.isfinite(float(n)) and math.isnan(float(n)) == math.isnan(bad)
        assert torch.equal(g.view(torch.int32), before.view(torch.int32)) and torch.all(h == 1)
        out = [torch.zeros_like(h), torch.zeros_like(g)]
        O.clip_grads([h, g], 1e-3, out=out)
        assert torch.equal(out[1].view(torch.int32), before.view(torch.int32)) and torch.all(out[0] == 1)
    # a bound of zero, and one that nothing exceeds
    g = torch.randn(100, device="cuda")
    before = g.clone()
    O.clip_grads([g], math.inf)
    assert torch.equal(g, before)
    O.clip_grads([g], 0.0)
    assert not g.any()
    assert float(O.grad_norm([g])) == 0.0 and float(O.clip_grads([g], 0.0)) == 0.0
    assert float(O.grad_norm([g[:0], g[:0]])) == 0.0


def test_shapes_and_orders():
    """Several dimensions, transposed and channels-last storage; a gradient
    into its own place; a norm of the caller's."""
    g = [torch.randn(3, 5, 7, 9, device="cuda").to(memory_format=torch.channels_last), torch.randn(40, 30, device="cuda").t(),
         torch.randn((), device="cuda"), torch.randn(1, 17, device="cuda")[:, :]]
    want = norm64(g)
    assert abs(float(O.grad_norm(g)) - want) <= (U + 1e-12) * want
    out = [torch.empty_like(t, memory_format=torch.preserve_format) for t in g]
    check_clip(g, want / 3, out=out)
    mixed = [g[0], out[1], g[2], out[3]]
    before = [t.clone() for t in g]
    O.clip_grads(g, want / 3, out=mixed)
    for b, t in zip(before, mixed):
        near(t.double().cpu(), b.double().cpu() / 3, 5 * U * b.double().cpu().abs(), "clipped")
    # by a norm twice as large
    t = torch.randn(1000, device="cuda")
    n = O.grad_norm([t])
    o = torch.empty_like(t)
    twice = 2 * n
    assert O.clip_grads([t], float(n), norm=twice, out=[o]) is twice
    near(o.double().cpu(), t.double().cpu() / 2, 5 * U * t.double().cpu().abs(), "by a norm")


def test_the_same_bits_every_time_and_captured():
    grads = make([100003, 64, 1 << 21, 777], [torch.bfloat16, torch.float32], std=2.0)
    out = [torch.empty_like(g) for g in grads]
    n = O.clip_grads(grads, 1.0, out=out)
    want = [n.clone()] + [o.clone() for o in out]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        m = O.clip_grads(grads, 1.0, out=out)
    for _ in range(3):
        for o in out:
            o.zero_()
        m.zero_()
        graph.replay()
        eager = O.grad_norm(grads)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for a, b in zip([m] + out, want):
            assert torch.equal(a, b)


def test_refusals_on_the_card():
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    for call, match in ((lambda: O.clip_grads([], 1.0), "no tensors"),
                        (lambda: O.grad_norm([a, b.cpu()]), r"grads\[1\]: not on the card"),
                        (lambda: O.grad_norm([a.double()]), "not float32"),
                        (lambda: O.grad_norm([a[::2]]), "do not fill"),
                        (lambda: O.grad_norm([a[:1].expand(4)]), "do not fill"),
                        (lambda: O.clip_grads([a, a], 1.0), "there twice"),
                        (lambda: O.clip_grads([a, a[4:]], 1.0), "overlaps"),
                        (lambda: O.clip_grads([a, b], 1.0, out=[b, a]), "overlaps"),
                        (lambda: O.clip_grads([a], 1.0, out=[b, a]), "2 tensors for 1"),
                        (lambda: O.clip_grads([a], 1.0, out=[b[:4]]), "shape and strides"),
                        (lambda: O.clip_grads([a], 1.0, out=[b.half()]), "size and type"),
                        (lambda: O.clip_grads([a], 1.0, norm=a), "one fp32"),
                        (lambda: O.clip_grads([a], -1.0), "max_norm"),
                        (lambda: O.clip_grads([a], math.nan), "max_norm"),
                        (lambda: O.clip_grads([a], 1.0, norm=a[3:4]), "overlaps")):
        with pytest.raises(P.MaximError, match=match):
            call()
    assert torch.all(a == 1) and torch.all(b == 1)
    assert float(O.grad_norm([a, a])) == 4.0  # reading twice is no fault
