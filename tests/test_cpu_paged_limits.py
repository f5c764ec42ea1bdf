"""Limits of the paged KV cache that are refused or said on tensors without a GPU."""
import pytest
import torch

import penny_b200.ops as P

ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def test_longest_row_below_zero():
    for longest, said in ((-1, "max_len"), (0, "CUDA"), (1 << 40, "CUDA")):
        with pytest.raises(RuntimeError, match=said):
            P.page_tables(ints(3, 4), ints(3), ints(10), ints(1), ints(3), 16, 8, max_len=longest)


def test_rows_of_more_than_a_row_has():
    """Positions past the table, or on no page, are an IndexError here; on the device an index past the end would stop the context."""
    c = P.PagedKVCache(1, 2, 40, 2, head_dim=64, page_size=16, device="cpu")
    c.table[1] = torch.tensor([4, 0, 5], dtype=torch.int32)
    assert [t.shape for t in c.rows_of(0, 1, 48)] == [(2, 48, 64)] * 2 and c.rows_of(0, 1, 0)[0].shape == (2, 0, 64)
    for row, length in ((1, 49), (1, 1000), (1, -1), (0, 1)):
        with pytest.raises(IndexError):
            c.rows_of(0, row, length)
    for bad in (6, 1 << 30, -3):
        c.table[1, 1] = bad
        with pytest.raises(IndexError):
            c.rows_of(0, 1, 17)
        c.rows_of(0, 1, 16)
