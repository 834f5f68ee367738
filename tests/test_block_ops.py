"""The block operators without a device (include/maxim_block_ops.h): what they
refuse, by argument and with a message, before any device work; what their host
side launches, on a HIP runtime that writes the launches down
(fake_block_card.py); the code objects' kernels against the host's choices."""

import ctypes as C
import os
import random
import re
import shutil
import struct
import subprocess

import pytest

torch = pytest.importorskip("torch")

import fake_block_card as F  # noqa: E402
from fake_card import mat as fmat, vec as fvec  # noqa: E402
from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "maxim-rs_amd", "csrc")
READELF = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"
F32, F16, BF16 = 0, 1, 2
SIZE = (4, 2, 2)
BASE = 1 << 40


def mat(rows, cols, at=0, rs=None, cs=1, dtype=BF16):
    return O.Mat(BASE + at, rows, cols, cols if rs is None else rs, cs, dtype, 0)


def vec(n, at=1 << 32, dtype=BF16):
    return O.Vec(BASE + at, n, dtype, 0)


def refused(match, rc):
    assert rc == -1
    assert match in P.last_error(), P.last_error()


# ------------------------------------------------------------- refusals


def test_every_declared_operator_is_exported():
    text = open(os.path.join(ROOT, "include", "maxim_block_ops.h")).read()
    names = re.findall(r"^int (mxh_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S), flags=re.M)
    assert len(names) == 13 and len(set(names)) == 13
    for n in names:
        assert hasattr(O._lib(), n), n


def gated(x, w, b, y, act=3, z=None, ws=None, n=0):
    return O._lib().mxh_gated(0, None, x, w, b, act, 0.0, y, z, ws, n)


def test_gated_refusals():
    x, w, y, b = mat(16, 32), mat(48, 32, 1 << 20), mat(16, 24, 2 << 20), vec(48)
    z = mat(16, 48, 3 << 20)
    refused("x: missing", gated(None, w, b, y))
    refused("w: missing", gated(x, None, b, y))
    refused("y: missing", gated(x, w, b, None))
    refused("w: [48][33]", gated(x, mat(48, 33, 1 << 20), b, y))
    refused("w: 47 rows are no gate's", gated(x, mat(47, 32, 1 << 20), b, y))
    refused("y: [16][25]", gated(x, w, b, mat(16, 25, 2 << 20)))
    refused("z: [16][24]", gated(x, w, b, y, z=mat(16, 24, 3 << 20)))
    refused("bias: 24", gated(x, w, vec(24), y))
    refused("bias: its type", gated(x, w, vec(48, dtype=F16), y))
    refused("w: f16 where x is bf16", gated(x, mat(48, 32, 1 << 20, dtype=F16), b, y))
    refused("z: f32 where x is bf16", gated(x, w, b, y, z=mat(16, 48, 3 << 20, dtype=F32)))
    refused("unknown activation", gated(x, w, b, y, act=6))
    refused("memory order", gated(x, w, b, mat(16, 24, 2 << 20, rs=1, cs=16)))
    refused("memory order", gated(x, w, b, y, z=mat(16, 48, 3 << 20, rs=1, cs=16)))
    refused("share storage", gated(x, w, b, mat(16, 24, 2 << 20, rs=0)))
    refused("share storage", gated(x, w, b, y, z=mat(16, 48, 3 << 20, rs=40)))
    refused("an output overlaps x", gated(x, w, b, mat(16, 24, 32)))
    refused("an output overlaps w", gated(x, w, b, y, z=mat(16, 48, (1 << 20) + 64)))
    refused("an output overlaps bias", gated(x, w, vec(48, 2 << 20), y))
    refused("y overlaps z", gated(x, w, b, y, z=mat(16, 48, 2 << 20)))
    refused("negative stride", gated(mat(16, 32, rs=-32), w, b, y))
    refused("not aligned", gated(mat(16, 32, 1), w, b, y))
    refused("device ordinal", O._lib().mxh_gated(64, None, x, w, b, 3, 0.0, y, z, None, 0))
    size = C.c_uint64()
    refused("bytes: missing", O._lib().mxh_gated_workspace(x, w, y, None, None))
    refused("x: missing", O._lib().mxh_gated_workspace(None, w, y, None, size))
    refused("w: missing", O._lib().mxh_gated_workspace(x, None, y, None, size))
    refused("y: missing", O._lib().mxh_gated_workspace(x, w, None, None, size))
    # a long sum of few results is cut, which takes scratch
    x, w, y = mat(64, 65536), mat(16, 65536, 1 << 24), mat(64, 8, 1 << 26)
    assert O._lib().mxh_gated_workspace(x, w, y, None, size) == 0 and size.value > 0
    refused("bytes of workspace", gated(x, w, None, y))
    refused("bytes of workspace, not", gated(x, w, None, y, ws=BASE + (1 << 36), n=size.value - 1))
    refused("16 bytes", gated(x, w, None, y, ws=BASE + (1 << 36) + 8, n=size.value))


def gated_backward(dy, x, w, z, dx, dw, db, act=3, ws=BASE + (1 << 36), n=1 << 30):
    return O._lib().mxh_gated_backward(0, None, dy, x, w, z, act, 0.0, dx, dw, db, ws, n)


def test_gated_backward_refusals():
    x, w, dy, z = mat(16, 32), mat(48, 32, 1 << 20), mat(16, 24, 2 << 20), mat(16, 48, 3 << 20)
    dx, dw, db = mat(16, 32, 4 << 20), mat(48, 32, 5 << 20), vec(48)
    a = (dy, x, w, z)
    refused("z: missing", gated_backward(dy, x, w, None, dx, dw, db))
    refused("z: [16][24]", gated_backward(dy, x, w, mat(16, 24, 3 << 20), dx, dw, db))
    refused("dy: [16][48]", gated_backward(mat(16, 48, 2 << 20), x, w, z, dx, dw, db))
    refused("dx: [16][31]", gated_backward(*a, mat(16, 31, 4 << 20), dw, db))
    refused("dw: [24][32]", gated_backward(*a, dx, mat(24, 32, 5 << 20), db))
    refused("db: 24", gated_backward(*a, dx, dw, vec(24)))
    refused("memory order", gated_backward(dy, x, w, mat(16, 48, 3 << 20, rs=1, cs=16), dx, dw, db))
    refused("unknown activation", gated_backward(*a, dx, dw, db, act=-1))
    refused("dx overlaps dy", gated_backward(*a, mat(16, 32, 2 << 20), dw, db))
    refused("dx overlaps x", gated_backward(*a, x, dw, db))
    refused("dx overlaps z", gated_backward(*a, mat(16, 32, 3 << 20), dw, db))
    refused("dw overlaps w", gated_backward(*a, dx, w, db))
    refused("dw overlaps dx", gated_backward(*a, dx, mat(48, 32, (4 << 20) + 64), db))
    refused("db overlaps dw", gated_backward(*a, dx, dw, vec(48, 5 << 20)))
    size = C.c_uint64()
    for missing, ops in (("dy", (None, x, w)), ("x", (dy, None, w)), ("w", (dy, x, None))):
        refused(missing + ": missing", O._lib().mxh_gated_backward_workspace(*ops, dx, dw, db, size))
        refused(missing + ": missing", gated_backward(*ops, z, dx, dw, db))
    assert O._lib().mxh_gated_backward_workspace(dy, x, w, dx, dw, db, size) == 0 and size.value
    refused("bytes of workspace, not", gated_backward(*a, dx, dw, db, n=size.value - 1))
    refused("dx: [16][31]", O._lib().mxh_gated_backward_workspace(dy, x, w, mat(16, 31, 4 << 20), dw, db, size))


def vecs(*v):
    return (O.Vec * len(v))(*v)


def test_clip_refusals():
    L = O._lib()
    a, b = vec(100), vec(50, 1 << 33, F32)
    norm, ws, n = BASE + (1 << 34), BASE + (1 << 36), 1 << 20
    size = C.c_uint64()

    def clip(g, out=None, most=1.0, norm=norm, ws=ws, n=n):
        return L.mxh_grad_clip(0, None, g, out, len(g), most, norm, ws, n)

    refused("grads: missing", L.mxh_grad_norm(0, None, None, 2, norm, ws, n))
    refused("grads: -1 tensors", L.mxh_grad_norm(0, None, vecs(a), -1, norm, ws, n))
    refused("norm: missing", L.mxh_grad_norm(0, None, vecs(a), 1, None, ws, n))
    refused("norm: not aligned", L.mxh_grad_norm(0, None, vecs(a), 1, norm + 2, ws, n))
    refused("bytes: missing", L.mxh_grad_norm_workspace(vecs(a), 1, None))
    refused("grads[1]: unknown type", clip(vecs(a, vec(5, 1 << 33, 7))))
    refused("grads[1]: no data", clip(vecs(a, O.Vec(None, 5, F32, 0))))
    refused("grads[0]: not aligned", clip(vecs(vec(5, 1))))
    refused("grads[0]: -5 elements", clip(vecs(vec(-5))))
    refused("elements", clip(vecs(vec(1 << 45))))
    refused("there twice", clip(vecs(a, b, a)))
    refused("overlaps", clip(vecs(a, vec(10, (1 << 32) + 198))))
    refused("overlaps", clip(vecs(a), norm=BASE + (1 << 32) + 4))
    refused("overlaps", L.mxh_grad_norm(0, None, vecs(a), 1, BASE + (1 << 32) + 4, ws, n))
    refused("overlaps", L.mxh_grad_clip_by(0, None, vecs(a), None, 1, 1.0, BASE + (1 << 32) + 4))
    refused("out[0]: not its gradient's", clip(vecs(a), vecs(vec(99, 1 << 35))))
    refused("out[0]: not its gradient's", clip(vecs(a), vecs(vec(100, 1 << 35, F16))))
    refused("overlaps", clip(vecs(a), vecs(vec(100, (1 << 32) + 2))))
    refused("overlaps", clip(vecs(a, b), vecs(vec(100, 1 << 35), vec(50, (1 << 35) + 196, F32))))
    refused("max_norm", clip(vecs(a), most=-1.0))
    refused("max_norm", clip(vecs(a), most=float("nan")))
    big = vecs(vec(1 << 24))
    assert L.mxh_grad_norm_workspace(big, 1, size) == 0 and size.value
    refused("bytes of workspace, not", clip(big, n=size.value - 1))
    refused("bytes of workspace", L.mxh_grad_norm(0, None, big, 1, norm, None, 0))
    refused("device ordinal", L.mxh_grad_norm(64, None, big, 1, norm, ws, 1 << 30))
    # a list that one block takes needs none
    assert L.mxh_grad_norm_workspace(vecs(a, b), 2, size) == 0 and size.value == 0


def mx4(rows, cols, at=1 << 34):
    return O.Mx4Mat(BASE + at, BASE + at + (1 << 33), rows, cols)


def test_mx4_refusals():
    L = O._lib()
    x, q = mat(16, 32), mx4(16, 32)
    c, s = C.c_uint64(), C.c_uint64()
    refused("out of range", L.mxh_mx4_size(-1, 32, c, s))
    refused("out of range", L.mxh_mx4_size(1, 1 << 24, c, s))
    refused("missing", L.mxh_mx4_size(1, 32, c, None))
    assert L.mxh_mx4_size(65, 257, c, s) == 0 and (c.value, s.value) == (65 * 256, 2 * 2 * 512)
    refused("x: missing", L.mxh_mx4_quantize(0, None, None, q))
    refused("q: missing", L.mxh_mx4_quantize(0, None, x, None))
    refused("q: [16][33]", L.mxh_mx4_quantize(0, None, x, mx4(16, 33)))
    refused("q: no data", L.mxh_mx4_quantize(0, None, x, O.Mx4Mat(None, BASE, 16, 32)))
    refused("q: not aligned", L.mxh_mx4_quantize(0, None, x, O.Mx4Mat(BASE + (1 << 34) + 8, BASE + (1 << 35), 16, 32)))
    refused("codes overlaps x", L.mxh_mx4_quantize(0, None, x, O.Mx4Mat(BASE + 1008, BASE + (1 << 35), 16, 32)))
    refused("scales overlaps x", L.mxh_mx4_quantize(0, None, x, O.Mx4Mat(BASE + (1 << 34), BASE + 16, 16, 32)))
    refused("codes overlaps scales", L.mxh_mx4_quantize(0, None, x, O.Mx4Mat(BASE + (1 << 34), BASE + (1 << 34) + 2032, 16, 32)))
    refused("neither rows nor columns", L.mxh_mx4_quantize(0, None, mat(16, 32, rs=70, cs=2), q))
    refused("y: missing", L.mxh_mx4_dequantize(0, None, q, None))
    refused("share storage", L.mxh_mx4_dequantize(0, None, q, mat(16, 32, rs=0)))
    refused("y overlaps codes", L.mxh_mx4_dequantize(0, None, q, mat(16, 32, 1 << 34)))
    refused("y overlaps scales", L.mxh_mx4_dequantize(0, None, q, mat(16, 32, (1 << 34) + (1 << 33) + 4)))

    def dense(x, w, b, y, act=0, res=None, ws=BASE + (1 << 36), n=1 << 30):
        return L.mxh_mx4_dense(0, None, x, w, b, act, 0.0, res, y, ws, n)

    w, y, b = mx4(24, 32), mat(16, 24, 2 << 20), vec(24)
    for missing, ops in (("x", (None, w, None, y)), ("w", (x, None, None, y)), ("y", (x, w, None, None))):
        refused(missing + ": missing", L.mxh_mx4_dense_workspace(*ops, s))
    refused("bytes: missing", L.mxh_mx4_dense_workspace(x, w, None, y, None))
    refused("w: missing", dense(x, None, b, y))
    refused("x: missing", dense(None, w, b, y))
    refused("y: missing", dense(x, w, b, None))
    refused("w: [24][33]", dense(x, mx4(24, 33), b, y))
    refused("y: [16][25]", dense(x, w, b, mat(16, 25, 2 << 20)))
    refused("bias: 23", dense(x, w, vec(23), y))
    refused("unknown activation", dense(x, w, b, y, act=9))
    refused("memory order", dense(x, w, b, y, res=mat(16, 24, 3 << 20, rs=1, cs=16)))
    refused("y overlaps x", dense(x, w, b, mat(16, 24, 32)))
    refused("y overlaps w's codes", dense(x, w, b, mat(16, 24, 1 << 34)))
    refused("y overlaps w's scales", dense(x, w, b, mat(16, 24, (1 << 34) + (1 << 33))))
    refused("y overlaps bias", dense(x, w, vec(24, 2 << 20), y))
    refused("y overlaps the residual", dense(x, w, b, y, res=mat(16, 24, (2 << 20) + 2)))
    size = C.c_uint64()
    x, y = mat(40, 32), mat(40, 24, 2 << 20)
    assert L.mxh_mx4_dense_workspace(x, w, None, y, size) == 0 and size.value
    refused("bytes of workspace, not", dense(x, w, b, y, n=size.value - 1))
    refused("bytes of workspace", dense(x, w, b, y, ws=None))


def test_tensors_of_the_host_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: O.gated(x, x), lambda: O.gated_backward(x, x, x, x), lambda: O.mx4_quantize(x),
                 lambda: O.mx4_dense(x, x)):
        with pytest.raises(P.MaximError, match="x: not a tensor on the card"):
            call()
    for call in (lambda: O.grad_norm([x]), lambda: O.clip_grads([x], 1.0), lambda: O.grad_norm([1.0])):
        with pytest.raises(P.MaximError, match=r"grads\[0\]: not a tensor on the card"):
            call()
    with pytest.raises(P.MaximError, match="not an Mx4"):
        O.mx4_dequantize(x)
    for t in (torch.zeros(4, 6)[:, :3], torch.zeros(8)[::2], torch.zeros(1).expand(5), torch.zeros(2, 3, 4)[:, :2]):
        with pytest.raises(P.MaximError, match="do not fill"):
            O._filled(t, "t")
    for t in (torch.zeros(3, 4).t(), torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last), torch.zeros(()),
              torch.zeros(4, 1, 6)[:, :, :], torch.zeros(6, 9)[2:4]):
        O._filled(t, "t")


# ------------------------------------------------------------- launches


@pytest.fixture(scope="module")
def card(tmp_path_factory):
    so = F.library(tmp_path_factory.mktemp("fake"))
    if so is None:
        pytest.skip("no g++")
    return lambda calls: F.run(so, calls)


AT = [(i + 1) << 52 for i in range(9)]


def gated_calls(rows, k, n, dtype, planar=False, pad=0, wt=False):
    """A gated Dense and its backward pass, as the Python binding makes them."""
    x, w = fmat(rows, k, AT[0], not planar, pad, dtype), fmat(2 * n, k, AT[1], not wt, 0, dtype)
    y, z = fmat(rows, n, AT[2], not planar, 0, dtype), fmat(rows, 2 * n, AT[3], not planar, 0, dtype)
    dy, dx = fmat(rows, n, AT[4], not planar, pad, dtype), fmat(rows, k, AT[5], not planar, 0, dtype)
    return [{"op": "gated", "x": x, "w": w, "y": y, "z": z, "bias": fvec(2 * n, AT[6], dtype)},
            {"op": "gated_backward", "dy": dy, "x": x, "w": w, "z": z, "dx": dx, "dw": fmat(2 * n, k, AT[7], not wt, 0, dtype),
             "db": fvec(2 * n, AT[6], dtype)}]


def check_gated(c, r):
    """Operands as the kernels' addresses need them, workspaces within their
    bytes, tiles for every result."""
    assert r["rc"] == 0, (r["error"], c)
    size, end = SIZE[c["x"][5]], F.WORKSPACE + r["workspace"]
    for l in r["launches"]:
        if l["kernel"].startswith("mxg_dz"):
            rows, n = c["dy"][1], c["dy"][2]
            line, lines = (l["drs"], rows) if "rows" in l["kernel"] else (l["dcs"], 2 * n)
            assert l["dz"] == F.WORKSPACE and l["dz"] + line * lines * size <= end
            assert line * size % 16 == 0 and line >= (2 * n if "rows" in l["kernel"] else rows)
            # a single part is the bias's gradient itself
            assert (l["db"] != 0) == (l["nparts"] == 1) == (l["part"] == 0)
            assert l["part"] + l["nparts"] * 2 * n * 4 <= end or l["db"] == c["db"][0]
        f = re.match(r"mx([og])_gemm_(?:([nm])_)?(bf16|f16|f32)_(\d+)x\d+_([km])([km])(_d\d)?$", l["kernel"])
        if not f:
            continue
        tile, bk, pair = int(f[4]), 128 // size, f[2]
        if l["splits"] > 1:
            assert F.WORKSPACE <= l["part"]
            assert l["part"] + l["splits"] * l["m"] * l["n"] * 4 * (2 if pair else 1) <= end, (l, c)
            assert l["kchunk"] * (l["splits"] - 1) < max(1, l["k"])
        bm, bn = tile // (2 if pair == "m" else 1), tile // (2 if pair == "n" else 1)
        assert (l["tiles_m"] - 1) * bm < l["m"] <= l["tiles_m"] * bm and (l["tiles_n"] - 1) * bn < l["n"] <= l["tiles_n"] * bn
        assert l["gx"] == l["tiles_m"] * l["tiles_n"] * l["splits"]
        assert l["block"] == (512 if tile == 256 else 256)
        if pair:
            # planes or rows, the weights either way
            assert f[5] + f[6] in (("kk", "km") if pair == "n" else ("km", "mm"))
        if not f[7]:
            continue
        for along, ld, p, half in ((f[5], l["lda"], l["a"], l["m"] if pair == "m" else 0),
                                   (f[6], l["ldb"], l["b"], l["n"] if pair == "n" else 0)):
            assert p % 16 == 0 and ld * size % 16 == 0, (l, c)
            assert (tile if along == "k" else bk) * ld * size < 1 << 31, (l, c)
            # the values' half begins at whole chunks
            assert along == "k" or half * size % 16 == 0, (l, c)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gated_launches(card, dtype):
    rng = random.Random(dtype)

    def size(most):
        n = int(2 ** rng.uniform(0, most))
        return n if rng.random() < 0.5 else (n + 63) // 64 * 64

    calls = []
    for _ in range(500):
        calls += gated_calls(size(22), size(11), size(11), dtype, rng.random() < 0.5, rng.choice([0, 0, 3, 8]), rng.random() < 0.5)
    for rows, k, n in ((1 << 24, 64, 64), ((1 << 24) + 3, 128, 32), (512, 1 << 22, 64), (512, (1 << 21) + 3, 256), (1 << 25, 16, 8)):
        for planar in (False, True):
            for wt in (False, True):
                calls += gated_calls(rows, k, n, dtype, planar, 0, wt)
    for c, r in zip(calls, card(calls)):
        check_gated(c, r)


def test_a_tokens_call_needs_no_workspace(card):
    """One row of results lies in both orders: the one that the operands settle
    counts."""
    x, r = fmat(1, 4096, AT[0], True, 0, BF16), fmat(1, 4096, AT[5], True, 0, BF16)
    calls = [gated_calls(1, 2048, 4096, BF16)[0],
             {"op": "mx4_dense", "x": x, "w": [AT[2], AT[3], 4096, 4096], "y": fmat(1, 4096, AT[1], True, 0, BF16), "residual": r},
             {"op": "mx4_dense", "x": x, "w": [AT[2], AT[3], 4096, 4096], "y": [AT[1], 1, 4096, 1, 1, BF16],
              "residual": [AT[5], 1, 4096, 1, 3, BF16]}]
    got = card(calls)
    assert [g["rc"] for g in got] == [0, 0, 0]
    assert [g["workspace"] for g in got[:2]] == [0, 0] and got[2]["workspace"] > 0
    assert [l["kernel"][:10] for g in got for l in g["launches"]][:2] == ["mxg_skinny", "mxq_skinny"]
    assert [l["m"] for l in got[2]["launches"] if "gemm" in l["kernel"]] == [4096]  # a residual of stride 3: planes of one position


def test_gated_forms_of_single_rows_and_columns(card):
    """Axes of one element have any stride: the call's order holds, and only
    kernels that there are take part."""
    calls = []
    for rows, k, n in ((1, 8, 8), (1, 64, 64), (64, 1, 64), (64, 64, 1), (1, 1, 1), (1, 300, 7), (20, 1, 1)):
        for planar in (False, True):
            for wt in (False, True):
                for c in gated_calls(rows, k, n, BF16, planar, 5, wt):
                    calls.append(c)
                    if rows == 1:  # a single position's other stride
                        calls.append(dict(c, x=c["x"][:3] + ([1, 9] if planar else [9, 1]) + c["x"][5:]))
    # an x that lies in both orders with results that have only one
    x, w = [AT[0], 1, 64, 64, 1, BF16], fmat(128, 64, AT[1], True, 0, BF16)
    calls.append({"op": "gated", "x": x, "w": w, "y": [AT[2], 1, 64, 1, 5, BF16]})
    for c, r in zip(calls, card(calls)):
        check_gated(c, r)
    assert r["launches"][0]["kernel"].startswith(("mxg_gemm_m", "mxo_pack"))


def test_a_gated_call_too_large_launches_nothing(card):
    calls = []
    for planar in (False, True):
        for rows, k, n in (((1 << 31) - 2000, 64, 64), (2, 5, 1 << 29), (1 << 28, 33, 700), (1 << 30, 4, 4)):
            calls += gated_calls(rows, k, n, BF16, planar)
    said = 0
    for c, r in zip(calls, card(calls)):
        assert r["rc"] == 0 or not r["launches"], (r, c)
        said += r["rc"] != 0
        assert r["rc"] == 0 or "one launch" in r["error"]
    assert said


def test_clip_launches(card):
    rng = random.Random(3)
    lists = [[0], [0, 0], [1], [8192] * 16, [8192] * 17, [100] * 1000, [1 << 31, 5], [(1 << 33) + 1] * 3, [1 << 30] * 400]
    lists += [[int(2 ** rng.uniform(0, 24)) * rng.choice([0, 1, 1]) for _ in range(rng.randrange(1, 300))] for _ in range(50)]
    calls = []
    for sizes in lists:
        at, grads, out = 1 << 50, [], []
        for n in sizes:
            t = rng.choice([F32, F16, BF16])
            grads.append([at, n, t])
            out.append([at + (1 << 58), n, t])
            at += (n * 4 + 15) // 16 * 16
        calls += [{"op": "norm", "grads": grads}, {"op": "clip", "grads": grads}, {"op": "clip", "grads": grads, "out": out}]
    for c, r in zip(calls, card(calls)):
        assert r["rc"] == 0, (r["error"])
        n = sum(g[1] for g in c["grads"])
        names = [l["kernel"] for l in r["launches"]]
        chunks = sum(-(-g[1] * SIZE[g[2]] // 16384) for g in c["grads"])
        tensors = sum(g[1] > 0 for g in c["grads"])
        if chunks <= 16 and tensors <= 128:
            assert names == ["mxn_small"] and r["workspace"] == 0
            assert r["launches"][0]["elements"] == n and r["launches"][0]["gx"] == 1
            continue
        squares = [l for l in r["launches"] if l["kernel"] == "mxn_squares"]
        clip = [l for l in r["launches"] if l["kernel"] == "mxn_clip"]
        assert names == ["mxn_squares"] * len(squares) + ["mxn_norm"] + ["mxn_clip"] * len(clip)
        assert len(clip) == (len(squares) if c["op"] == "clip" else 0)
        for ls in [squares] + ([clip] if clip else []):
            assert sum(l["elements"] for l in ls) == n and sum(l["chunks"] for l in ls) == chunks
            assert all(0 < l["count"] <= 128 and 0 < l["gx"] <= 2048 and l["chunks"] < 1 << 31 for l in ls)
        at = F.WORKSPACE
        for l in squares:
            assert l["part"] == at
            at += l["gx"] * 8
        join = r["launches"][len(squares)]
        assert join["part"] == F.WORKSPACE and join["nparts"] * 8 == at - F.WORKSPACE == r["workspace"]


def test_mx4_launches(card):
    rng = random.Random(4)
    calls = []
    for _ in range(400):
        rows, k, n = (int(2 ** rng.uniform(0, e)) for e in (18, 15, 13))
        t, planar, xp, pad = rng.choice([F32, F16, BF16]), rng.random() < 0.5, rng.random() < 0.3, rng.choice([0, 3, 8])
        x, y = fmat(rows, k, AT[0], not (planar ^ xp), pad, t), fmat(rows, n, AT[1], not planar, pad, t)
        w = [AT[2], AT[3], n, k]
        calls.append({"op": "mx4_dense", "x": x, "w": w, "y": y, "bias": fvec(n, AT[4], t)})
        calls.append({"op": "quantize", "x": x, "q": [AT[2], AT[3], rows, k]})
        calls.append({"op": "dequantize", "y": y, "q": [AT[2], AT[3], rows, n]})
    calls.append({"op": "mx4_dense", "x": fmat(40, 0, AT[0], True, 0, BF16), "w": [AT[2], AT[3], 7, 0],
                  "y": fmat(40, 7, AT[1], True, 0, BF16)})
    for c, r in zip(calls, card(calls)):
        assert r["rc"] == 0, (r["error"], c)
        if c["op"] != "mx4_dense":
            m = c.get("x") or c["y"]
            l, = r["launches"]
            by_rows = m[4] == 1 and (m[3] != 1 or m[2] == 1 or m[1] == 1)
            assert l["tiles"] == -(-m[2] // 256)
            each = 256 // SIZE[m[5]] if "planar" in l["kernel"] else 64 if "dequantize" in l["kernel"] else 32
            assert l["gx"] == -(-m[1] // each) * l["tiles"]
            assert ("_rows_" in l["kernel"]) == by_rows or m[1] == 1 or m[2] == 1
            continue
        rows, k, n = c["x"][1], c["x"][2], c["y"][2]
        tiles, end = -(-k // 256), F.WORKSPACE + r["workspace"]
        l = [l for l in r["launches"] if l["kernel"].startswith(("mxq_gemm", "mxq_skinny"))]
        assert len(l) == 1
        l = l[0]
        if "skinny" in l["kernel"]:
            assert rows <= 16 and l["k"] == tiles and l["gx"] == -(-n // 16) and r["workspace"] == 0
            continue
        assert {l["m"], l["n"]} == {rows, n} and l["k"] == tiles
        if k:
            code = r["launches"][0]
            assert code["codes"] == F.WORKSPACE and code["scales"] >= code["codes"] + rows * tiles * 128
            assert code["scales"] % 16 == 0 and code["scales"] + -(-rows // 64) * tiles * 512 <= end
            mine, theirs = (l["ca"], l["sa"]), (l["cb"], l["sb"])
            if l["m"] != rows or (rows == n and mine[0] != F.WORKSPACE):
                mine, theirs = theirs, mine
            assert mine == (code["codes"], code["scales"]) and theirs == (AT[2], AT[3])
        tile = int(re.search(r"_(\d+)x", l["kernel"])[1])
        assert l["gx"] == l["tiles_m"] * l["tiles_n"] * l["splits"] and l["tiles_m"] == -(-l["m"] // tile)
        assert tile * tiles * 128 < 1 << 31 and l["block"] == (512 if tile == 256 else 256)
        if l["splits"] > 1:
            assert l["part"] + l["splits"] * rows * n * 4 <= end


def test_ready_loads_every_code_object(card):
    assert card([{"op": "ready"}])[0] == {"rc": 0, "modules": 4}


# ------------------------------------------------------------- code objects


def kernels(name, tmp):
    """{kernel: spilled VGPRs} of a built code object."""
    path = os.path.join(P.LIB_DIR, "maxim_%s.hsaco" % name)
    if not (os.path.exists(READELF) and os.path.exists(path)):
        pytest.skip("no llvm-readelf or no built code object")
    blob = open(path, "rb").read()
    at, elf = 32, tmp / "gfx950.elf"
    for _ in range(struct.unpack_from("<Q", blob, 24)[0]):
        off, size, n = struct.unpack_from("<3Q", blob, at)
        if b"gfx950" in blob[at + 24:at + 24 + n]:
            elf.write_bytes(blob[off:off + size])
        at += 24 + n
    notes = subprocess.run([READELF, "--notes", str(elf)], capture_output=True, text=True, check=True).stdout
    out = {}
    for k in notes.split("- .agpr_count:")[1:]:
        f = dict(re.findall(r"\.(name|vgpr_spill_count):\s+(\S+)", re.sub(r"\n {6,}.*", "", k)))
        out[f["name"]] = int(f["vgpr_spill_count"])
    return out


def tiles(path, table):
    body = re.search(r"%s\[\] = \{(.*?)\};" % table, open(os.path.join(SRC, "exec", path)).read(), re.S).group(1)
    return [x.split(", ")[:2] for x in re.findall(r"\{([\d., ]+)\}", body)]


def chosen(name):
    out = set()
    for t in ("bf16", "f16", "f32"):
        if name == "gated":
            for b, stages in tiles("ops.cpp", "kTiles32" if t == "f32" else "kTiles16"):
                if stages == "0" and b != "64":
                    continue
                out |= {"mxg_gemm_%s_%s_%sx%s_%s%s" % (a, t, b, b, o, "" if stages == "0" else "_d" + stages)
                        for a, o in (("n", "kk"), ("n", "km"), ("m", "km"), ("m", "mm"))}
            out |= {"mxg_%s_%s_%s" % (j, a, t) for j in ("join", "join8") for a in "nm"}
            out |= {"mxg_skinny_" + t, "mxg_dz_rows_" + t, "mxg_dz_planar_" + t, "mxg_grad_join_" + t}
        elif name == "mx4":
            out |= {"mxq_gemm_%s_%sx%s_d%s" % (t, b, b, stages) for b, stages in tiles("mx4.cpp", "kTilesMx4")}
            out |= {"mxq_%s_%s_%s" % (w, o, t) for w in ("quantize", "dequantize") for o in ("rows", "planar")}
            out |= {"mxq_skinny_" + t}
    return out or {"mxn_squares", "mxn_norm", "mxn_clip", "mxn_small"}


@pytest.mark.parametrize("name", ["gated", "mx4", "grads"])
def test_the_code_object_holds_what_the_host_chooses_from(name, tmp_path):
    got = kernels(name, tmp_path)
    assert set(got) == chosen(name)
    assert not any(got.values()), {k: v for k, v in got.items() if v}
