"""The memory order of the gated Dense's results from Python, where axes of one
element leave it open: the Python call itself, on tensors of the host and a HIP
runtime that runs nothing (fake_block_card.py)."""

import json
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

import fake_block_card as F  # noqa: E402

SCRIPT = r"""
import json, sys
sys.path.insert(0, sys.argv[1])
import torch
from maxim_amd import ops as O

O._lib()
O._device = lambda x: 0
O._tensor = lambda t, what, device: O._types[t.dtype]
O._stream = lambda device: None
out = []
for rows, k, n, planar, mine, save, given in json.load(sys.stdin):
    # the call's own order, or the other one seen through a transpose
    a, b = (k, rows) if planar else (rows, k)
    x = torch.zeros(a, b) if mine else torch.zeros(b, a).t()
    w = torch.zeros(2 * n, k)
    y0 = None
    if given:
        a = n if planar else rows, rows if planar else n
        y0 = torch.zeros(a) if mine else torch.zeros(a[::-1]).t()
    try:
        got = O.gated(x, w, planar=planar, save=save, out=y0)
        y, z = got if save else (got, None)
        good = tuple(y.shape) == ((n, rows) if planar else (rows, n)) and (not given or y is y0)
        good = good and (z is None or tuple(z.shape) == ((2 * n, rows) if planar else (rows, 2 * n)))
        if z is not None and rows > 1 and k > 1:
            # z's order is x's: features side by side or positions
            by_rows = x.stride(1 if planar else 0) == 1
            good = good and z.stride() == ((rows, 1) if planar else (1, rows)) if by_rows else \
                z.stride() == ((1, 2 * n) if planar else (2 * n, 1))
        out.append("" if good else "y %s z %s" % (y.stride(), z is None or z.stride()))
    except Exception as e:
        out.append(str(e))
print(json.dumps(out))
"""


def test_one_feature_or_position_leaves_no_order_open(tmp_path):
    so = F.library(tmp_path)
    if so is None:
        pytest.skip("no g++")
    calls = [[rows, k, n, planar, mine, save, given]
             for rows in (1, 2, 70) for k in (1, 3, 64) for n in (1, 2, 5) for planar in (False, True)
             for mine in (True, False) for save in (True, False) for given in (False, True)]
    r = subprocess.run([sys.executable, "-c", SCRIPT, F.PKG], input=json.dumps(calls), text=True,
                       stdout=subprocess.PIPE, env=dict(os.environ, MAXIM_HIP_LIB=so))
    assert r.returncode == 0
    bad = {str(c): e for c, e in zip(calls, json.loads(r.stdout)) if e}
    assert not bad


@pytest.mark.gpu
@pytest.mark.parametrize("mine", [True, False])
@pytest.mark.parametrize("planar", [True, False])
def test_one_feature_of_either_order(gpu_ok, planar, mine):
    """With z kept the same y as without, z against 64 bits: 96 products of fp32
    off by 97 u of the terms' magnitudes, u = 2^-24."""
    from maxim_amd import ops as O
    g = torch.Generator().manual_seed(3)
    v, w = torch.randn(70, 96, generator=g), torch.randn(2, 96, generator=g)
    x = v.cuda() if planar != mine else v.t().contiguous().cuda()
    x = x if mine else x.t()
    y, z = O.gated(x, w.cuda(), planar=planar, save=True)
    assert torch.equal(y, O.gated(x, w.cuda(), planar=planar))
    zv = (z.t() if planar else z).double().cpu()
    want = v.double() @ w.double().t()
    assert zv.shape == want.shape
    assert bool(((zv - want).abs() <= 97 * 2.0 ** -24 * (v.double().abs() @ w.double().abs().t())).all())
    d = [torch.ones_like(y) for _ in range(2)]
    one, two = O.gated_backward(d[0], x, w.cuda(), z, planar=planar), O.gated_backward(d[1], x, w.cuda(), z.clone(), planar=planar)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
