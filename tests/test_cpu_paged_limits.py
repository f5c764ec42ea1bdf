"""Limits of the paged KV cache that are refused or said on tensors without a GPU."""
import pytest
import torch

import penny_b200.ops as P

ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def test_longest_row_below_zero():
    for longest, said in ((-1, "max_len"), (0, "CUDA"), (1 << 40, "CUDA")):
        with pytest.raises(RuntimeError, match=said):
            P.page_tables(ints(3, 4), ints(3), ints(10), ints(1), ints(3), 16, 8, max_len=longest)
