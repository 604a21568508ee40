"""Arguments of the paged key/value cache that have to be refused before any
kernel sees them, and what a call asks for: no GPU needed."""

from __future__ import annotations

import pytest
import torch

import awa_b200

INTS = dict(dtype=torch.int32)


@pytest.mark.parametrize("table", [
    torch.zeros(4, **INTS).expand(3, -1),                       # one row for all: stride 0
    torch.zeros(6, **INTS).as_strided((3, 4), (1, 1)),          # rows that overlap
    torch.zeros(9, **INTS).as_strided((3, 4), (2, 1)),
], ids=["expanded", "stride1", "stride2"])
def test_page_tables_whose_rows_overlap(table):
    """Passed on with a stride of the width, such a table would be read behind its storage."""
    with pytest.raises(ValueError, match="page_table"):
        awa_b200.CacheBatch(torch.zeros(4, **INTS), torch.zeros(3, **INTS), table, 3, 1)


def test_strides_of_page_tables_that_are_taken():
    starts, past = torch.zeros(4, **INTS), torch.zeros(3, **INTS)
    wide = torch.zeros(3, 9, **INTS)
    assert awa_b200.CacheBatch(starts, past, wide[:, 2:6], 3, 1).c.table_stride == 9
    assert awa_b200.CacheBatch(starts, past, wide, 3, 1).c.table_stride == 9
    # the stride of a single row is never used
    one = torch.zeros(4, **INTS).expand(1, -1).as_strided((1, 4), (0, 1))
    assert awa_b200.CacheBatch(starts[:2], past[:1], one, 3, 1).c.table_stride == 4
