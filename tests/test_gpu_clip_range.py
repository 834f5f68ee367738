"""Clipping where the factor max_norm / N is below fp32's normal range, 2^-126,
and the results are not. Tolerance as in test_gpu_grads.py: the factor is off by
u and by N's u, and a product rounds once to fp32 and once to the tensor's type:
3 u |g f| + h |g f|, and half of fp32's smallest step for a result below its
normal range. max_norm is a power of two, which fp32 has exactly."""

import math

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402
from test_gpu_operators import U, half, near  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def named(request, gpu_ok):
    print(request.node.name, flush=True)
    O.ready()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [300, 70001, 3000001], ids=["one_launch", "chunks", "many"])
@pytest.mark.parametrize("power", [-1, -13, -20, -60, -100, -130])
def test_factors_below_the_normal_range(dt, size, power):
    g = torch.Generator().manual_seed(size)
    v = torch.rand(size, generator=g, dtype=torch.float64) * 2 - 1
    v *= 2.9e38 / float((v * v).sum().sqrt())
    v[7] = 1e-3  # and one that goes to nothing
    t = v.to(dt).cuda()
    want = t.double().cpu()
    norm = math.sqrt(math.fsum((want * want).tolist()))
    most = 2.0 ** power
    assert most / norm < 2.0 ** -126 and norm < 3.4e38
    w = want * (most / norm)
    tol = (3 * U + half(dt) * (1 + 4 * U)) * w.abs() + 2.0 ** (-150 if dt == torch.float32 else -134)
    out = [torch.empty_like(t)]
    got = O.clip_grads([t], most, out=out)
    assert abs(float(got) - norm) <= (U + 1e-12) * norm
    near(out[0].double().cpu(), w, tol, "out of place")
    kept = t.clone()
    O.clip_grads([kept], most, norm=got)
    assert torch.equal(kept.view(torch.uint8), out[0].view(torch.uint8))
    O.clip_grads([t], most)
    assert torch.equal(t.view(torch.uint8), out[0].view(torch.uint8))


def test_factors_at_the_border():
    """Both ways of multiplying give the same where both are exact: powers of
    two, with the factor just above, at and below 2^-126."""
    g = torch.zeros(64, device="cuda")
    g[0] = 2.0 ** 127
    for power in (2, 1, 0, -1, -2, -5):
        out = [torch.empty_like(g)]
        O.clip_grads([g], 2.0 ** power, out=out)
        assert float(out[0][0]) == 2.0 ** power and not out[0][1:].any()
    # a bound that is nothing
    O.clip_grads([g], 0.0)
    assert not g.any()
