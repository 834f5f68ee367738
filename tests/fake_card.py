"""The operators' host side against a HIP runtime that launches nothing
(fake_hip.cpp): run(calls) gives, for each call, its status, its message, the
launches it made and its workspace's bytes. A process of its own, since a
process keeps the runtime it first loads."""

import ctypes as C
import json
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "maxim-rs_amd")
WORKSPACE = 1 << 60
SIZE = (4, 2, 2)


def mat(rows, cols, at, by_cols=True, pad=0, dtype=2):
    """A matrix operand: [rows][cols] with columns contiguous, or in planar
    order, in a buffer `pad` elements wider, at address `at`."""
    ld = (cols if by_cols else rows) + pad
    return [at, rows, cols, ld if by_cols else 1, 1 if by_cols else ld, dtype]


def vec(n, at, dtype=2):
    return [at, n, dtype]


def library(folder):
    """The fake runtime, built in `folder`; None without a compiler."""
    cxx = shutil.which("g++")
    if cxx is None:
        return None
    objs = []
    for i, flags in enumerate(([], ["-DDEFAULTS"])):
        objs.append(os.path.join(str(folder), "fake%d.o" % i))
        subprocess.run([cxx, "-std=c++17", "-O1", "-fPIC", "-I" + os.path.join(PKG, "csrc", "exec"),
                        "-c", os.path.join(HERE, "fake_hip.cpp"), "-o", objs[-1]] + flags, check=True)
    so = os.path.join(str(folder), "libfakehip.so")
    subprocess.run([cxx, "-shared", "-o", so] + objs, check=True)
    return so


def run(so, calls):
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], input=json.dumps(calls), text=True,
                       stdout=subprocess.PIPE, env=dict(os.environ, MAXIM_HIP_LIB=so))
    assert r.returncode == 0, r.returncode
    return json.loads(r.stdout)


def main():
    sys.path.insert(0, PKG)
    from maxim_amd import ops as O
    from maxim_amd import plan as P
    fake = C.CDLL(os.environ["MAXIM_HIP_LIB"])
    fake.fake_launches.restype = C.c_char_p
    L = O._lib()

    def m(v):
        return None if v is None else O.Mat(v[0], v[1], v[2], v[3], v[4], v[5], 0)

    def w(v):
        return None if v is None else O.Vec(v[0], v[1], v[2], 0)

    def call(c):
        g, n = c.get, C.c_uint64()
        rc = 0
        if c["op"] == "dense":
            x, wt, y = m(c["x"]), m(c["w"]), m(c["y"])
            rc = L.mxh_dense_workspace(x, wt, y, n)
            rc = rc or L.mxh_dense(0, None, x, wt, w(g("bias")), g("act", 0), 0.2, m(g("residual")), y, m(g("z")),
                                   WORKSPACE, n.value)
        elif c["op"] == "dense_backward":
            a = [m(c["dy"]), m(c["x"]), m(c["w"])]
            outs = [m(g("dx")), m(g("dw")), w(g("db"))]
            rc = L.mxh_dense_backward_workspace(*a, g("act", 0), *outs, n)
            rc = rc or L.mxh_dense_backward(0, None, *a, m(g("z")), g("act", 0), 0.2, *outs, WORKSPACE, n.value)
        elif c["op"] == "layernorm":
            rc = L.mxh_layernorm(0, None, m(c["x"]), w(c["scale"]), None, 1e-6, m(c["y"]), None, None)
        else:
            x, ds = m(c["x"]), w(g("dscale"))
            rc = L.mxh_layernorm_backward_workspace(x, n)
            rc = rc or L.mxh_layernorm_backward(0, None, m(c["dy"]), x, w(c["scale"]), c["mean"], c["rstd"],
                                                m(g("add")), m(g("dx")), ds, w(g("dbias")), WORKSPACE, n.value)
        return {"rc": rc, "error": P.last_error() if rc else "", "workspace": n.value,
                "launches": json.loads(fake.fake_launches())}

    print(json.dumps([call(c) for c in json.load(sys.stdin)]))


if __name__ == "__main__":
    main()
