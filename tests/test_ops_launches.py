"""What the operators' host side launches, checked without a device: a HIP
runtime that writes the launches down takes calls on made-up addresses
(fake_card.py)."""

import random
import re

import pytest

pytest.importorskip("torch")

import fake_card as F  # noqa: E402

F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def card(tmp_path_factory):
    so = F.library(tmp_path_factory.mktemp("fake"))
    if so is None:
        pytest.skip("no g++")
    return lambda calls: F.run(so, calls)


def dense_calls(rows, k, n, dtype, planar=False, pad=0, wt=False, act=0, x_planar=None):
    """A Dense and its backward pass over [rows][k] -> [rows][n], as the Python
    binding makes them: y in dy's order, dx in x's, dw in w's."""
    xp = planar if x_planar is None else x_planar
    at = [(i + 1) << 52 for i in range(8)]
    x = F.mat(rows, k, at[0], not xp, pad, dtype)
    w = F.mat(n, k, at[1], not wt, 0, dtype)
    y, dy, z = (F.mat(rows, n, a, not planar, p, dtype) for a, p in ((at[2], 0), (at[3], pad), (at[4], pad)))
    dx, dw = F.mat(rows, k, at[5], not xp, 0, dtype), F.mat(n, k, at[6], not wt, 0, dtype)
    return [{"op": "dense", "x": x, "w": w, "y": y, "bias": F.vec(n, at[7], dtype), "act": act},
            {"op": "dense_backward", "dy": dy, "x": x, "w": w, "z": z if act else None, "act": act, "dx": dx, "dw": dw,
             "db": F.vec(n, at[7], dtype)}]


def check_products(call, result):
    """A product's operands as the kernels' addresses need them."""
    assert result["rc"] == 0, (result["error"], call)
    size = F.SIZE[call["x"][5]]
    for l in result["launches"]:
        for i in "01":
            if "dst" + i in l:
                assert F.WORKSPACE <= l["dst" + i] and l["end" + i] <= F.WORKSPACE + result["workspace"], (l, call)
        f = re.match(r"mxo_gemm_\w+?_(\d+)x\d+_([km])([km])_d\d$", l["kernel"])
        if not f:
            continue
        tile, bk = int(f[1]), 128 // size
        for along, ld, p in ((f[2], l["lda"], l["a"]), (f[3], l["ldb"], l["b"])):
            assert p % 16 == 0 and ld * size % 16 == 0, (l, call)
            # a tile's lines, the buffer that bounds them and the step to the
            # next tile are offsets of 31 bits
            assert (tile if along == "k" else bk) * ld * size < 1 << 31, (l, call)


# rows, k, n: planes of 2^24 positions and more, and sums as long
LARGE = [((1 << 24) + d, k, n) for d in (0, 8, 3) for k, n in ((128, 256), (512, 512), (16, 2048), (64, 64))] + [
    (1 << 25, 512, 512), (1 << 26, 64, 256), (1 << 23, 256, 256), (1 << 21, 128, 128), ((1 << 21) + 1, 640, 640),
    (512, (1 << 21) + 3, 512), (512, 1 << 22, 256), (256, 640, (1 << 23) + 1), (300, 1 << 24, 300)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_long_lines_keep_to_31_bits(card, dtype):
    calls = []
    for rows, k, n in LARGE:
        for i in range(16):
            calls += dense_calls(rows, k, n, dtype, bool(i & 1), 3 if i & 2 else 0, bool(i & 4), x_planar=bool(i & 8),
                                 act=int(i % 3 == 0))
    for c, r in zip(calls, card(calls)):
        check_products(c, r)


def test_drawn_products_keep_to_31_bits(card):
    rng = random.Random(5)

    def size(most):
        n = int(2 ** rng.uniform(0, most))
        return n if rng.random() < 0.5 else (n + 63) // 64 * 64

    calls = []
    for _ in range(1500):
        sizes = [size(26), size(11), size(11)]
        rng.shuffle(sizes)
        rows, k, n = sizes[0], min(sizes[1], 1 << 23), min(sizes[2], 1 << 23)
        calls += dense_calls(rows, k, n, rng.choice([F32, F16, BF16]), rng.random() < 0.5, rng.choice([0, 0, 3, 8]),
                             rng.random() < 0.5, rng.choice([0, 1]), rng.random() < 0.5)
    for c, r in zip(calls, card(calls)):
        check_products(c, r)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_few_features_keep_the_card_busy(card, dtype):
    """The gradient of a planar Dense's weights sums over every position: with
    few features too it is spread over the card, 256 CUs. A short sum into few
    columns takes one launch, and many columns need no cut."""
    calls = [dense_calls(448 * 640, k, n, dtype, True)[1] for k in (3, 32, 64, 128) for n in (1, 3, 8, 16, 17)]
    for c, r in zip(calls, card(calls)):
        check_products(c, r)
        dw = [l for l in r["launches"] if "k" in l and l["k"] == 448 * 640]
        assert len(dw) == 1 and dw[0]["gx"] >= 240, (dw, c)
    calls = [dense_calls(rows, k, n, dtype)[0] for rows in (1, 16) for k, n in ((64, 64), (1024, 64), (1024, 4096), (4096, 4096))]
    for c, r in zip(calls, card(calls)):
        assert [l["kernel"][:10] for l in r["launches"]] == ["mxo_skinny"], (r, c)


def test_a_call_too_large_launches_nothing(card):
    """A launch has at most 2^32 threads; a call with one that would not fit is
    refused before any of its launches."""
    at = [(i + 1) << 52 for i in range(8)]
    calls = []
    for dtype in (F32, BF16):
        for planar in (False, True):
            for rows, cols in ((2, 1 << 26), (40, 1 << 24), (3, (1 << 30) + 8), (1, 1 << 27), (1 << 30, 2)):
                x, dy, dx = (F.mat(rows, cols, a, not planar, 8, dtype) for a in at[:3])
                p = [F.vec(cols, a, dtype) for a in at[3:6]]
                calls.append({"op": "layernorm", "x": x, "y": dx, "scale": p[0]})
                calls.append({"op": "layernorm_backward", "dy": dy, "x": x, "dx": dx, "scale": p[0], "dscale": p[1],
                              "dbias": p[2], "mean": at[6], "rstd": at[7]})
            for rows, k, n in ((40, 16, 1 << 24), (8, 16, (1 << 27) + 5), (3, 1 << 27, 8), ((1 << 31) - 2000, 64, 64),
                               (1 << 30, 16, 16), (2, 5, 1 << 30), (1 << 28, 33, 7)):
                for act in (0, 1):
                    calls += dense_calls(rows, k, n, dtype, planar, 3, act=act)
    said = set()
    for c, r in zip(calls, card(calls)):
        assert r["rc"] == 0 or not r["launches"], (r, c)
        assert all(l["gx"] * l["block"] < 1 << 32 for l in r["launches"])
        if r["rc"]:
            assert "one launch" in r["error"], r["error"]
            said.add(c["op"])
    assert said == {"layernorm_backward", "dense", "dense_backward"}


def layernorm_calls(rows, cols, dtype, planar, pad, add=None):
    at = [(i + 1) << 52 for i in range(9)]
    x, dy, a = (F.mat(rows, cols, v, not planar, pad, dtype) for v in at[:3])
    y, dx = (F.mat(rows, cols, v, not planar, 0, dtype) for v in at[3:5])
    p = [F.vec(cols, v, dtype) for v in at[5:8]]
    return [{"op": "layernorm", "x": x, "y": y, "scale": p[0]},
            {"op": "layernorm_backward", "dy": dy, "x": x, "add": a if add else None, "dx": dx, "scale": p[0],
             "dscale": p[1], "dbias": p[2], "mean": at[8], "rstd": at[8] + (1 << 40)}]


def test_the_device_tests_reach_every_kernel(card):
    """Each kernel that the host can choose is one that a test on the device
    runs, by the shapes, orders and paddings that those tests take."""
    import test_gpu_operators as G
    import test_gpu_products as H
    from test_ops_kernels import chosen
    calls = []
    for dtype in (F32, F16, BF16):
        for planar in (False, True):
            for s in G.DENSE_SHAPES:
                for pad, wt in ((0, False), (8, True), (3, False), (0, True)):
                    calls += dense_calls(*s, dtype, planar, pad, wt, act=1)
            for s in G.BIG_SHAPES:
                for wt in (False, True):
                    calls += dense_calls(*s, dtype, planar, 0, wt)
            for s in H.MIXED_SHAPES:
                for wt in (False, True):
                    for pad in (0, 3):
                        calls += dense_calls(*s, dtype, planar, pad, wt, x_planar=not planar)
            for s in G.LN_SHAPES:
                for pad in (0, 8, 3):
                    calls += layernorm_calls(*(s[::-1] if planar else s), dtype, planar, pad)
            for s in G.MANY if planar else G.MANY_ROWS:
                calls += layernorm_calls(*s, dtype, planar, 0)
            for s in H.LOOP_SHAPES:
                calls += layernorm_calls(*s, dtype, planar, 0)
    reached = set()
    for c, r in zip(calls, card(calls)):
        assert r["rc"] == 0, (r["error"], c)
        reached |= {l["kernel"] for l in r["launches"]}
    assert reached == chosen(), sorted(chosen() - reached)


def test_few_rows_and_very_many_columns(card):
    """More columns than the few-rows kernel's grid holds are the tiles'."""
    calls = []
    for n in ((1 << 27) - 16, (1 << 27) - 15, (1 << 27) + 5, (1 << 29) + 1):
        for dtype in (F32, BF16):
            calls.append(dense_calls(8, 16, n, dtype)[0])
    for c, r in zip(calls, card(calls)):
        check_products(c, r)
