"""The block operators' host side against a HIP runtime that launches nothing
(fake_block_hip.cpp): run(calls) gives, for each call, its status, its message,
the launches it made and its workspace's bytes. A process of its own, since a
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


def library(folder):
    """The fake runtime, built in `folder`; None without a compiler."""
    cxx = shutil.which("g++")
    if cxx is None:
        return None
    objs = []
    for i, flags in enumerate(([], ["-DDEFAULTS"])):
        objs.append(os.path.join(str(folder), "fake%d.o" % i))
        subprocess.run([cxx, "-std=c++17", "-O1", "-fPIC", "-I" + os.path.join(PKG, "csrc", "exec"),
                        "-c", os.path.join(HERE, "fake_block_hip.cpp"), "-o", objs[-1]] + flags, check=True)
    so = os.path.join(str(folder), "libfakeblockhip.so")
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

    def vs(v):
        return None if v is None else (O.Vec * len(v))(*[O.Vec(*t, 0) for t in v])

    def q(v):
        return O.Mx4Mat(*v)

    def call(c):
        g, n = c.get, C.c_uint64()
        op = c["op"]
        if op == "ready":
            rc = L.mxh_ops_ready(0)
            return {"rc": rc, "modules": fake.fake_modules()}
        if op == "gated":
            x, wt, y = m(c["x"]), m(c["w"]), m(c["y"])
            z = m(g("z"))
            rc = L.mxh_gated_workspace(x, wt, y, z, n)
            rc = rc or L.mxh_gated(0, None, x, wt, w(g("bias")), g("act", 3), 0.2, y, z, WORKSPACE, n.value)
        elif op == "gated_backward":
            a = [m(c["dy"]), m(c["x"]), m(c["w"])]
            outs = [m(g("dx")), m(g("dw")), w(g("db"))]
            rc = L.mxh_gated_backward_workspace(*a, *outs, n)
            rc = rc or L.mxh_gated_backward(0, None, *a, m(c["z"]), g("act", 3), 0.2, *outs, WORKSPACE, n.value)
        elif op == "norm":
            a = vs(c["grads"])
            rc = L.mxh_grad_norm_workspace(a, len(a), n)
            rc = rc or L.mxh_grad_norm(0, None, a, len(a), 1 << 59, WORKSPACE, n.value)
        elif op == "clip":
            a, o = vs(c["grads"]), vs(g("out"))
            rc = L.mxh_grad_norm_workspace(a, len(a), n)
            rc = rc or L.mxh_grad_clip(0, None, a, o, len(a), 1.0, 1 << 59, WORKSPACE, n.value)
        elif op == "quantize":
            rc = L.mxh_mx4_quantize(0, None, m(c["x"]), q(c["q"]))
        elif op == "dequantize":
            rc = L.mxh_mx4_dequantize(0, None, q(c["q"]), m(c["y"]))
        else:
            x, wt, y = m(c["x"]), q(c["w"]), m(c["y"])
            res = m(g("residual"))
            rc = L.mxh_mx4_dense_workspace(x, wt, res, y, n)
            rc = rc or L.mxh_mx4_dense(0, None, x, wt, w(g("bias")), g("act", 0), 0.2, res, y, WORKSPACE, n.value)
        return {"rc": rc, "error": P.last_error() if rc else "", "workspace": n.value,
                "launches": json.loads(fake.fake_launches())}

    print(json.dumps([call(c) for c in json.load(sys.stdin)]))


if __name__ == "__main__":
    main()
