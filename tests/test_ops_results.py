"""The tensors that the Python binding makes for results: shapes and memory
orders, which need no device."""

import pytest

torch = pytest.importorskip("torch")

from maxim_amd import ops as O  # noqa: E402


def result(x, n, planar):
    """_new's tensor for an x given as the binding would describe it."""
    O._lib()
    rows, cols = (x.shape[1], x.shape[0]) if planar else (x.shape[0], x.shape[1])
    rs, cs = (x.stride(1), x.stride(0)) if planar else x.stride()
    t, m = O._new(x, O.Mat(x.data_ptr(), rows, cols, rs, cs, 0, 0), n, planar)
    assert t.data_ptr() == m.data and (m.rows, m.cols) == (rows, n)
    # the matrix describes the tensor
    want = (t.stride(1), t.stride(0)) if planar else t.stride()
    assert m.rows <= 1 or m.row_stride == want[0]
    assert m.cols <= 1 or m.col_stride == want[1]
    return t


@pytest.mark.parametrize("n", [1, 2, 7])
def test_one_feature_has_its_calls_order(n):
    """An x of one feature (or one position) lies in both orders: results have
    the one that the call names, as an ordinary tensor has, unless x's strides
    are the other one's."""
    for x in (torch.zeros(6, 1), torch.zeros(6, 4)[:, :1], torch.zeros(6, 1, 1).view(6, 1), torch.zeros(6)[:, None]):
        assert result(x, n, False).is_contiguous() and result(x, n, False).shape == (6, n)
    for x in (torch.zeros(1, 6), torch.zeros(4, 6)[:1], torch.zeros(6, 1).t()):
        assert result(x, n, True).is_contiguous() and result(x, n, True).shape == (n, 6)
    assert result(torch.zeros(4, 6)[:1].t(), n, False).t().is_contiguous()
    assert result(torch.zeros(1, 6), n, False).is_contiguous()
    assert result(torch.zeros(6, 1), n, True).is_contiguous()


@pytest.mark.parametrize("n", [1, 6, 7])
def test_results_keep_the_order_of_wider_inputs(n):
    t = torch.zeros(5, 6)
    assert result(t, n, False).is_contiguous() and result(t, n, True).is_contiguous()
    # the other order than the call's, as it lies
    assert result(t.t(), n, False).t().is_contiguous() and result(t.t(), n, True).t().is_contiguous()
    # a row for all positions, a position for all features
    assert result(t[:1].expand(5, 6), n, False).shape == (5, n)
    assert result(t[:, :1].expand(5, 6), n, True).shape == (n, 6)
