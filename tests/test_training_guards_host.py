"""The host side of the training operators where a call could go wrong unseen: nothing here reaches a GPU."""
import pytest
import torch

import nestedtensor_b200 as nt
from nestedtensor_b200 import _cabi
from nestedtensor_b200.nn import training


def _nested(shapes, **kw):
    sizes = torch.tensor(shapes, dtype=torch.int64)
    return nt.NestedTensor(torch.zeros(int(sizes.prod(1).sum()), **kw), sizes)


# rows of one width, of several widths, of none; dimensions that differ while their product does not
@pytest.mark.parametrize("shapes", [[(3, 5), (4, 5)], [(3, 5), (4, 7)], [(4, 7), (3, 5)], [(3, 0), (4, 7)], [(3, 5), (0, 0), (2, 5)],
                                    [(2, 0), (5, 0)], [(0, 4), (6, 9), (1, 1)], [(2, 3, 4), (5, 4, 3)], [(2, 3, 4), (5, 3, 4)],
                                    [(2, 3, 0), (5, 4, 0)], [(3,), (0,), (2,)]], ids=str)
def test_row_offsets_follow_the_lengths(native_libs, shapes):
    """with_values() takes any constituents (L_i, ...): whatever their other dimensions, sequence i of the result begins at row
    L_0 + ... + L_(i-1)."""
    lengths = [s[0] for s in shapes]
    starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    for b in (_nested(shapes).with_values(torch.zeros(sum(lengths), 6)), _nested(shapes).with_values(torch.zeros(sum(lengths), 6)).to(torch.float16)):
        offsets, row = b._row_offsets()
        offsets = offsets[:len(lengths) + 1]
        assert row >= 1 and offsets.dtype == torch.int64
        assert (offsets % row == 0).all() and (offsets // row).tolist() == starts
        assert b.nested_size() == tuple(torch.Size([n, 6]) for n in lengths)
        assert b._record()[2][:len(lengths) + 1].tolist() == [6 * n for n in starts]


def test_structure_and_record_share_their_offsets(native_libs):
    """One copy of the offsets, whichever operator asked first."""
    for first in ("rows", "record"):
        a = _nested([(3, 5), (4, 5)])
        b = a.with_values(torch.zeros(7, 2))
        assert a._meta is None
        if first == "rows":
            rows = a._row_offsets()[0]
            assert a._meta is rows
            meta = a._record()[2]
        else:
            meta = a._record()[2]
            rows = a._row_offsets()[0]
        assert rows is meta and b._row_offsets()[0] is meta and a._meta is meta
        assert b._meta is None and b._record()[2].tolist() == [0, 6, 14, 3, 2, 4, 2]  # (its own sizes)
    given = torch.tensor([0, 15, 35, 3, 5, 4, 5])
    a = nt.NestedTensor(torch.zeros(35), torch.tensor([[3, 5], [4, 5]]), given)
    assert a._meta is given and a._record()[2] is given and a._row_offsets() == (given, 5)
    odd = _nested([(3, 5), (4, 7)])  # the record counts elements, the structure rows
    assert odd._record()[2].tolist() == [0, 15, 43, 3, 5, 4, 7]
    offsets, row = odd._row_offsets()
    assert row == 1 and offsets[:3].tolist() == [0, 3, 7] and odd._record()[2].tolist() == [0, 15, 43, 3, 5, 4, 7]


def test_the_tracked_rows_are_the_callers_own_tensor():
    """No base of a view in its place: that would pass by its hooks, and lead gradients around a no_grad block."""
    x = torch.randn(7, 5, requires_grad=True)
    sizes = torch.tensor([[3, 5], [4, 5]])
    buf = x.view(-1)
    assert nt.NestedTensor(buf, sizes)._tracked()[0] is buf
    with torch.no_grad():
        cut = x.view(-1)
    assert nt.NestedTensor(cut, sizes)._tracked()[0] is cut


def test_a_tracked_buffer_is_known_as_one():
    x = torch.randn(7, 5, requires_grad=True)
    a = nt.NestedTensor(x.view(-1), torch.tensor([[3, 5], [4, 5]]))
    assert a.requires_grad and a.values().requires_grad and a.with_values(x * 1).requires_grad
    assert not a.with_values(x.detach()).requires_grad and not nt.NestedTensor(x.detach().view(-1), a._sizes).requires_grad
    for t in (a, a.with_values(x * 1)):
        with pytest.raises(RuntimeError, match="does not track gradients"):
            t._record()
        assert t._layout()[1].tolist() == [0, 15, 35, 3, 5, 4, 5]
        with torch.no_grad():
            assert t._record()[0].numel() == 35


@pytest.mark.parametrize("scaling", [float("nan"), float("inf"), -float("inf"), 1e39, 3e38])
def test_attention_refuses_scalings_that_are_not_finite(native_libs, scaling):
    """Times log2(e), as the kernels hold it in 32 bits."""
    lib = _cabi.load()
    for path in (0, 1, 2, 3):
        assert lib.ntb200_varlen_attention_train(16, 64, 16, 64, 16, 64, 32, 16, 16, 64, 16, 64, 1, 4, 4, 1, 64, 4, scaling, 2, path, 16, 1 << 20,
                                                 None) == -1
        assert lib.ntb200_varlen_attention_backward(16, 16, 64, 16, 64, 16, 64, 16, 16, 16, 64, 16, 64, 16, 64, 16, 64, 16, 64, 1, 4, 4, 1, 64, 4, 4,
                                                    scaling, 2, path, 16, 1 << 20, None) == -1


def test_tensor_core_kernels_refuse_scalings_that_are_not_positive(native_libs):
    lib = _cabi.load()
    for scaling in (0.0, -0.125, 2.0 ** -130):
        for path in (2, 3):
            assert lib.ntb200_varlen_attention_train(16, 64, 16, 64, 16, 64, 32, 16, 16, 64, 16, 64, 1, 4, 4, 1, 64, 4, scaling, 2, path, 16, 1 << 20,
                                                     None) == -7
            assert lib.ntb200_varlen_cross_attention_ws(16, 64, 16, 64, 16, 64, 32, 16, 16, 1, 4, 4, 1, 64, 4, scaling, 2, path, 16, 1 << 20,
                                                        None) == -7
        for path in (2, 3, 4):
            assert lib.ntb200_varlen_attention(16, 32, 16, 1, 4, 1, 64, 4, scaling, 2, path, 16, 1 << 20, None) == -7
        assert lib.ntb200_varlen_cross_attention(16, 64, 16, 64, 16, 64, 32, 16, 16, 1, 4, 1, 64, 4, scaling, 2, 2, None) == -7


def test_a_pass_without_gradients_leaves_the_graph_alone():
    """What an operator under no_grad looked at is not kept: gradients flow through the constituents afterwards."""
    x = torch.randn(7, 5, requires_grad=True)
    a = _nested([(3, 5), (4, 5)])
    for rows in (x, x * 1):
        b = a.with_values(rows)
        with torch.no_grad():
            b._record()
            assert b.numel() == 35
        x.grad = None
        b.unbind()[1].sum().backward()
        assert torch.equal(x.grad, torch.cat([torch.zeros(3, 5), torch.ones(4, 5)]))
    later = torch.randn(7, 5)
    b = a.with_values(later)
    b._record()
    later.requires_grad_()
    b.unbind()[0].sum().backward()
    assert torch.equal(later.grad, torch.cat([torch.ones(3, 5), torch.zeros(4, 5)]))
