"""The launches of the gated Dense's backward pass in fp16, which forms dz again
where it left fp16's range (include/maxim_block_ops.h), on a HIP runtime that
writes them down (fake_block_card.py)."""

import pytest

torch = pytest.importorskip("torch")

import fake_block_card as F  # noqa: E402
from test_block_ops import AT, BF16, F16, F32, check_gated, gated_calls  # noqa: E402


@pytest.fixture(scope="module")
def card(tmp_path_factory):
    so = F.library(tmp_path_factory.mktemp("fake"))
    if so is None:
        pytest.skip("no g++")
    return lambda calls: F.run(so, calls)


SHAPES = [(1, 64, 64), (40, 300, 77), (4096, 1024, 2048), (71680, 64, 64), (33, 8, 9000), (5, 16, 1 << 20)]


@pytest.mark.parametrize("planar", [False, True])
def test_fp16_forms_dz_where_its_range_holds_it(card, planar):
    calls = [gated_calls(*s, t, planar)[1] for s in SHAPES for t in (F32, F16, BF16)]
    calls += [dict(c, dx=None, dw=None) for c in calls]
    for c, r in zip(calls, card(calls)):
        check_gated(c, r) if c["dx"] else None
        assert r["rc"] == 0
        dz = [l for l in r["launches"] if l["kernel"].startswith("mxg_dz")]
        assert r["launches"][:len(dz)] == dz and len({l["kernel"] for l in dz}) == 1
        if c["x"][5] != F16 or not c["dx"]:
            assert len(dz) == 1
            continue
        blocks = dz[0]["gx"] * dz[0]["gy"]
        # once more, in runs as long or longer; many blocks' magnitudes by one between
        assert dz[-1]["gx"] == dz[0]["gx"] and 1 <= dz[-1]["gy"] <= dz[0]["gy"]
        assert len(dz) == (3 if blocks > 4096 else 2)
        assert len(dz) == 2 or (dz[1]["gx"], dz[1]["gy"]) == (1, 1)
        # room for a magnitude a block, the largest, and the products' factor,
        # behind dz and the bias's sums and before the products' scratch
        size, n = 2, c["dy"][2]
        used = (dz[0]["drs"] * c["dy"][1] if not planar else dz[0]["dcs"] * 2 * n) * size
        if dz[0]["part"]:
            used += dz[0]["nparts"] * 2 * n * 4
        assert r["workspace"] >= used + (blocks + 2) * 4
        for l in r["launches"][len(dz):]:
            if l.get("splits", 1) > 1:
                assert l["part"] >= F.WORKSPACE + used + (blocks + 2) * 4


def test_fp16_of_no_rows_or_features(card):
    """Nothing to form dz from: the products' factor is not read either."""
    calls = [gated_calls(*s, F16, p)[1] for s in ((0, 8, 8), (8, 0, 8), (8, 8, 0)) for p in (False, True)]
    for c, r in zip(calls, card(calls)):
        assert r["rc"] == 0, r["error"]
        dz = [l for l in r["launches"] if l["kernel"].startswith("mxg_dz")]
        assert len(dz) == (2 if c["dy"][1] and c["dy"][2] else 0)
