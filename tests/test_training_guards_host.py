"""The host side of the training operators where a call could go wrong unseen: nothing here reaches a GPU."""
import pytest
import torch

import nestedtensor_b200 as nt


def _nested(shapes, **kw):
    sizes = torch.tensor(shapes, dtype=torch.int64)
    return nt.NestedTensor(torch.zeros(int(sizes.prod(1).sum()), **kw), sizes)


# rows of one width, of several widths, of none; dimensions that differ while their product does not
@pytest.mark.parametrize("shapes", [[(3, 5), (4, 5)], [(3, 5), (4, 7)], [(4, 7), (3, 5)], [(3, 0), (4, 7)], [(3, 5), (0, 0), (2, 5)],
                                    [(2, 0), (5, 0)], [(0, 4), (6, 9), (1, 1)], [(2, 3, 4), (5, 4, 3)], [(2, 3, 4), (5, 3, 4)],
                                    [(2, 3, 0), (5, 4, 0)], [(3,), (0,), (2,)]], ids=str)
def test_row_offsets_follow_the_lengths(shapes):
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
