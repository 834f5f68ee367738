"""What the operators refuse (include/maxim_ops.h), by argument and with a
message, before any device work: the calls here carry made-up addresses, and
none of them gets as far as the runtime."""

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from maxim_amd import plan as P  # noqa: E402

F32, F16, BF16 = 0, 1, 2
BASE = 1 << 40


def mat(rows, cols, at=0, rs=None, cs=1, dtype=BF16):
    return O.Mat(BASE + at, rows, cols, cols if rs is None else rs, cs, dtype, 0)


def vec(n, at=1 << 32, dtype=BF16):
    return O.Vec(BASE + at, n, dtype, 0)


def refused(match, rc):
    assert rc == -1
    assert match in P.last_error(), P.last_error()


def ln(x, scale, bias, y, eps=1e-6, mean=None, rstd=None):
    return O._lib().mxh_layernorm(0, None, x, scale, bias, eps, y, mean, rstd)


def test_layernorm_refusals():
    x, y, s, b = mat(4, 8), mat(4, 8, 1 << 20), vec(8), vec(8, 1 << 33)
    refused("x: missing", ln(None, s, b, y))
    refused("y: missing", ln(x, s, b, None))
    refused("scale: missing", ln(x, None, b, y))
    refused("unknown type", ln(mat(4, 8, dtype=7), s, b, y))
    refused("y: f32 where x is bf16", ln(x, s, b, mat(4, 8, 1 << 20, dtype=F32)))
    refused("expected [4][8]", ln(x, s, b, mat(4, 9, 1 << 20)))
    refused("no columns", ln(mat(4, 0), vec(0), None, mat(4, 0)))
    refused("scale: 7 elements", ln(x, vec(7), b, y))
    refused("scale: its type", ln(x, vec(8, dtype=F16), b, y))
    refused("differ in type", ln(x, vec(8, dtype=F32), b, y))
    refused("eps", ln(x, s, b, y, eps=-1.0))
    refused("eps", ln(x, s, b, y, eps=float("nan")))
    refused("neither rows nor columns", ln(mat(4, 8, rs=20, cs=2), s, b, y))
    refused("negative stride", ln(mat(4, 8, rs=-8), s, b, y))
    refused("out of range", ln(mat(1 << 31, 8), s, b, mat(1 << 31, 8, 1 << 40)))
    refused("strides out of range", ln(mat(4, 8, rs=1 << 62), s, b, y))
    refused("share storage", ln(x, s, b, mat(4, 8, 1 << 20, rs=0)))
    refused("share storage", ln(x, s, b, mat(4, 8, 1 << 20, rs=7)))
    refused("differ in memory order", ln(x, s, b, mat(4, 8, 1 << 20, rs=1, cs=4)))
    refused("not aligned", ln(mat(4, 8, 1), s, b, y))
    refused("no data", ln(O.Mat(None, 4, 8, 8, 1, BF16, 0), s, b, y))
    # one row on: y's first rows are x's last
    refused("y overlaps x", ln(x, s, b, mat(4, 8, 16)))
    # a slice whose columns reach into x's
    refused("y overlaps x", ln(mat(4, 8, rs=16), s, b, mat(4, 8, 14, rs=16)))
    # and one that runs over the line's end into x's next row
    refused("y overlaps x", ln(mat(4, 8, rs=16), s, b, mat(4, 8, 18, rs=16)))
    refused("scale", ln(x, vec(8, 1 << 20), b, y))
    refused("a statistic overlaps y", ln(x, s, b, y, mean=BASE + (1 << 20), rstd=BASE + (1 << 22)))
    refused("mean overlaps rstd", ln(x, s, b, y, mean=BASE + (1 << 22), rstd=BASE + (1 << 22) + 8))
    refused("device ordinal", O._lib().mxh_layernorm(64, None, x, s, b, 1e-6, y, None, None))
    refused("device ordinal", O._lib().mxh_ops_ready(-1))


def lnb(dy, x, s, mean, rstd, add, dx, ds, db, ws=BASE + (1 << 36), n=1 << 30):
    return O._lib().mxh_layernorm_backward(0, None, dy, x, s, mean, rstd, add, dx, ds, db, ws, n)


def test_layernorm_backward_refusals():
    x, dy, dx, add = mat(100, 8), mat(100, 8, 1 << 20), mat(100, 8, 2 << 20), mat(100, 8, 3 << 20)
    s, ds, db = vec(8), vec(8, 1 << 33), vec(8, 1 << 34)
    m, r = BASE + (1 << 28), BASE + (1 << 29)
    refused("mean, rstd", lnb(dy, x, s, None, r, None, dx, ds, db))
    refused("dscale and dbias", lnb(dy, x, s, m, r, None, dx, ds, None))
    refused("add without dx", lnb(dy, x, s, m, r, add, None, ds, db))
    refused("scale's type", lnb(dy, x, s, m, r, None, dx, vec(8, 1 << 33, F32), db))
    refused("dx overlaps x", lnb(dy, x, s, m, r, None, x, ds, db))
    refused("dx overlaps dy", lnb(dy, x, s, m, r, None, mat(100, 8, (1 << 20) + 16), ds, db))
    refused("dx overlaps add", lnb(dy, x, s, m, r, add, mat(100, 8, (3 << 20) + 16), ds, db))
    refused("dx overlaps the statistics", lnb(dy, x, s, m, r, None, mat(100, 8, 1 << 28), ds, db))
    refused("gradient overlaps", lnb(dy, x, s, m, r, None, dx, vec(8, 1 << 20), db))
    refused("dscale overlaps dbias", lnb(dy, x, s, m, r, None, dx, ds, vec(8, (1 << 33) + 4)))
    size = C.c_uint64()
    assert O._lib().mxh_layernorm_backward_workspace(x, size) == 0
    refused("bytes of workspace", lnb(dy, x, s, m, r, None, dx, ds, db, None))
    refused("bytes of workspace, not", lnb(dy, x, s, m, r, None, dx, ds, db, n=size.value - 1))
    refused("16 bytes", lnb(dy, x, s, m, r, None, dx, ds, db, ws=BASE + (1 << 36) + 8))
    refused("bytes: missing", O._lib().mxh_layernorm_backward_workspace(x, None))


def dn(x, w, b, y, act=0, res=None, z=None, ws=None, n=0):
    return O._lib().mxh_dense(0, None, x, w, b, act, 0.0, res, y, z, ws, n)


def test_dense_refusals():
    x, w, y, b = mat(16, 32), mat(24, 32, 1 << 20), mat(16, 24, 2 << 20), vec(24)
    refused("w: [24][33]", dn(x, mat(24, 33, 1 << 20), b, y))
    refused("y: [16][25]", dn(x, w, b, mat(16, 25, 2 << 20)))
    refused("bias: 23", dn(x, w, vec(23), y))
    refused("w: f16 where x is bf16", dn(x, mat(24, 32, 1 << 20, dtype=F16), b, y))
    refused("unknown activation", dn(x, w, b, y, act=6))
    refused("unknown activation", dn(x, w, b, y, act=-1))
    refused("memory order", dn(x, w, b, y, res=mat(16, 24, 3 << 20, rs=1, cs=16)))
    refused("memory order", dn(x, w, b, y, z=mat(16, 24, 3 << 20, rs=1, cs=16)))
    refused("an output overlaps x", dn(x, w, b, mat(16, 24, 32)))
    refused("an output overlaps w", dn(x, w, b, mat(16, 24, 1 << 20)))
    refused("an output overlaps bias", dn(x, w, vec(24, 2 << 20), y))
    refused("an output overlaps the residual", dn(x, w, b, y, res=mat(16, 24, (2 << 20) + 2)))
    refused("an output overlaps the residual", dn(x, w, b, y, res=mat(16, 24, 3 << 20), z=mat(16, 24, 3 << 20)))
    refused("y overlaps z", dn(x, w, b, y, z=y))
    # few outputs and a long sum are split over the card, which takes scratch
    x, w, y = mat(64, 65536), mat(8, 65536, 1 << 24), mat(64, 8, 1 << 26)
    size = C.c_uint64()
    assert O._lib().mxh_dense_workspace(x, w, y, size) == 0 and size.value > 0
    refused("bytes of workspace", dn(x, w, vec(8), y))


def test_dense_backward_refusals():
    L = O._lib()
    x, w, dy, z = mat(16, 32), mat(24, 32, 1 << 20), mat(16, 24, 2 << 20), mat(16, 24, 3 << 20)
    dx, dw, db = mat(16, 32, 4 << 20), mat(24, 32, 5 << 20), vec(24)

    def call(dy=dy, x=x, w=w, z=z, act=1, dx=dx, dw=dw, db=db, ws=BASE + (1 << 36), n=1 << 30):
        return L.mxh_dense_backward(0, None, dy, x, w, z, act, 0.0, dx, dw, db, ws, n)

    refused("z: missing", call(z=None))
    refused("unknown activation", call(act=9))
    refused("z: [16][23]", call(z=mat(16, 23, 3 << 20)))
    refused("memory order", call(z=mat(16, 24, 3 << 20, rs=1, cs=16)))
    refused("dx: [16][31]", call(dx=mat(16, 31, 4 << 20)))
    refused("dw: [24][31]", call(dw=mat(24, 31, 5 << 20)))
    refused("db: 25", call(db=vec(25)))
    refused("db: its type", call(db=vec(24, dtype=F16)))
    refused("dx overlaps x", call(dx=x))
    refused("dx overlaps dy", call(dx=mat(16, 32, 2 << 20)))
    refused("dw overlaps w", call(dw=w))
    refused("dw overlaps dx", call(dw=mat(24, 32, 4 << 20)))
    refused("db overlaps z", call(db=vec(24, 3 << 20)))
    refused("share storage", call(dw=mat(24, 32, 5 << 20, rs=0)))
    refused("bytes of workspace", call(ws=None))


def test_python_refusals():
    """The binding's own checks: tensors that are not the card's."""
    x = torch.zeros(4, 8)
    for call in (lambda: O.layernorm(x, x[0]), lambda: O.dense(x, x), lambda: O.layernorm([1.0], x[0]),
                 lambda: O.dense_backward(x, x, x), lambda: O.layernorm_backward(x, x, x[0], x[0], x[0])):
        with pytest.raises(P.MaximError, match="x: not a tensor on the card"):
            call()


def test_a_second_hip_runtime_is_refused():
    """A runtime that the executor loaded before torch brought its own."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import ctypes, sys\n"
            "sys.path.insert(0, %r)\n"
            "try:\n    ctypes.CDLL('/opt/rocm/lib/libamdhip64.so')\n"
            "except OSError:\n    sys.exit(7)\n"
            "from maxim_amd import ops, plan\n"
            "try:\n    ops._lib()\n"
            "except plan.MaximError as e:\n    sys.exit(0 if 'two HIP runtimes' in str(e) else 1)\n"
            "sys.exit(0 if len(ops._runtimes()) == 1 else 2)\n" % os.path.join(root, "maxim-rs_amd"))
    rc = subprocess.run([sys.executable, "-c", code]).returncode
    if rc == 7:
        pytest.skip("no HIP runtime outside torch")
    assert rc == 0


def test_every_declared_operator_is_exported():
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                             "maxim_ops.h")).read()
    names = re.findall(r"^int (mxh_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S), flags=re.M)
    assert len(names) == 8
    for n in names:
        assert hasattr(O._lib(), n), n


def test_tangents_are_refused():
    """A call would drop a forward-mode tangent: tensors that carry one are
    refused, but inside an autograd.Function, which sees none."""
    from torch.autograd import forward_ad

    class Card:
        """A CPU tensor that says that it is the card's."""
        dtype, is_cuda, requires_grad = torch.float32, True, False

        def __init__(self, t):
            self.t = t

        def get_device(self):
            return 0

    O._lib()
    tell = forward_ad.unpack_dual
    x = torch.zeros(3)
    try:
        forward_ad.unpack_dual = lambda t: tell(t.t)
        assert O._tensor(Card(x), "x", 0) == 0
        with forward_ad.dual_level():
            d = forward_ad.make_dual(x, torch.ones(3))
            assert O._tensor(Card(x), "x", 0) == 0
            with pytest.raises(P.MaximError, match="x carries a forward-mode tangent"):
                O._tensor(Card(d), "x", 0)

            class Twice(torch.autograd.Function):
                @staticmethod
                def forward(v):
                    assert O._tensor(Card(v), "x", 0) == 0
                    return 2 * v

                @staticmethod
                def setup_context(ctx, inputs, output):
                    pass

                @staticmethod
                def jvp(ctx, t):
                    return 2 * t

            assert torch.equal(tell(Twice.apply(d)).tangent, torch.full((3,), 2.0))
        assert O._tensor(Card(x), "x", 0) == 0
    finally:
        forward_ad.unpack_dual = tell
