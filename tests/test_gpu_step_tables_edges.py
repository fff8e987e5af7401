"""Block bookkeeping at the edges of its sizes, strides and lengths."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def test_table_rows_that_overlap_are_refused(cuda):
    """The table is written in place: one row expanded over the requests has no room of its own for each."""
    from smaq_b200 import ops
    row = ints([5, -1, -1], cuda)
    for shared in (row[None].expand(2, -1), row.as_strided((2, 2), (1, 1))):
        with pytest.raises(ValueError, match="rows of their own"):
            ops.step_tables(ints([1, 2, 3], cuda), ints([3], cuda), ints([0, 0], cuda), ints([4, 4], cuda), shared, block_size=16, num_tokens=8)
    assert row.tolist() == [5, -1, -1]
    t = ops.step_tables(ints([1, 2, 3], cuda), ints([3], cuda), ints([0], cuda), ints([4], cuda), row[None].expand(1, -1), block_size=16, num_tokens=4)
    assert t.slots.tolist() == [48, 49, 50, 51] and row.tolist() == [3, -1, -1]
