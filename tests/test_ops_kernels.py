"""The operators' kernels: each that the host can choose is in the code object
and each in it can be chosen (the reference checks its kernel list both ways
at startup, src/cuda.rs:76-85); none spills but where it is known; the GELU
fit they share."""

import math
import os
import re
import shutil
import struct
import subprocess

import numpy as np
import pytest

from maxim_amd import plan as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "maxim-rs_amd", "csrc")
READELF = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{kernel: spilled VGPRs}"""
    path = os.path.join(P.LIB_DIR, "maxim_ops.hsaco")
    if not (os.path.exists(READELF) and os.path.exists(path)):
        pytest.skip("no llvm-readelf or no built code object")
    blob = open(path, "rb").read()
    at, elf = 32, tmp_path_factory.mktemp("co") / "gfx950.elf"
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


def chosen():
    src = open(os.path.join(SRC, "exec", "ops.cpp")).read()

    def table(name):
        body = re.search(r"%s(?:\[\](?:\[2\])?)? = \{(.*?)\};" % name, src, re.S).group(1)
        return [x.split(", ") for x in re.findall(r"\{([\d., ]+)\}", body)]

    out = {"mxo_join_parts", "mxo_pack_16", "mxo_pack_32"}
    for t in ("bf16", "f16", "f32"):
        bits = "32" if t == "f32" else "16"
        for d in ("", "bwd_"):
            out |= {"mxo_ln_%srows_%s_%s" % (d, t, "x".join(f)) for f in table("kForms")}
            out |= {"mxo_ln_%splanar_%s_%s" % (d, t, "x".join(f))
                    for f in table(("kBackward" if d else "kForward") + bits)}
            out |= {"mxo_ln_%s%s_%s_%s" % (d, o, t, k) for o, k in (("rows", "long"), ("planar", "loop"))}
        out |= {"mxo_%s_%s_%s" % (a, o, t) for a in ("ln_param", "dz") for o in ("rows", "planar")}
        out |= {"mxo_%s_%s" % (a, t) for a in ("skinny", "join", "join8")}
        for f in table("kTiles" + bits):
            out |= {"mxo_gemm_%s_%sx%s_%s%s" % (t, f[0], f[0], o, "" if f[1] == "0" else "_d" + f[1])
                    for o in ("kk", "km", "mk", "mm")}
    return out


def test_the_code_object_holds_what_the_host_chooses_from(kernels):
    assert set(kernels) == chosen()


def test_spills(kernels):
    """Only forms with eight waves a SIMD or two vectors a thread, outside
    their loops over rows, spill a few registers."""
    spilled = {k: v for k, v in kernels.items() if v}
    assert all(re.match(r"mxo_ln_rows_b?f16_(128|512|1024)x1$|mxo_ln_bwd_planar_f32_512x\d+x8$", k) for k in spilled), spilled
    assert all(v <= 16 for v in spilled.values()), spilled


def test_phi_fit():
    """phi_tail's polynomial in fp32, as the kernels evaluate it: within 1.4e-7
    of Phi(-x) for x from 0 to 6, and monotone enough that past 6 zero is 1e-9
    off at most."""
    text = open(os.path.join(SRC, "ops", "ops_common.h")).read()
    body = text[text.index("float phi_tail"):]
    c = [np.float32(v) for v in re.findall(r"(-?\d\.\d+e[+-]\d\d)f", body[:body.index("return ax")])]
    assert len(c) == 8
    x = np.linspace(0, 6, 60001).astype(np.float32)
    q = np.full(x.shape, c[0], np.float32)
    for k in c[1:]:  # fma: one rounding a step
        q = (q.astype(np.float64) * x + k).astype(np.float32)
    got = np.exp2(q.astype(np.float64)).astype(np.float32).astype(np.float64)
    want = np.array([0.5 * math.erfc(v / math.sqrt(2)) for v in x.astype(np.float64)])
    # the hardware's exp2 is off by one ulp: 6e-8 of 0.5 at most
    assert np.abs(got - want).max() <= 1.4e-7 - 6e-8
    assert 0.5 * math.erfc(6 / math.sqrt(2)) < 1e-9
