"""Attention over shared pages with a window, for rows that were cut back since their groups were found."""
import pytest
import torch

from test_gpu_paged_shared import BF, F8, HALF
from test_gpu_paged_shared_wide import Wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim,shared,rows,cache", [(32, 8, 128, 2048, 72, BF), (32, 8, 128, 2048, 140, F8), (20, 20, 64, 2048, 64, HALF), (4, 1, 256, 4096, 160, BF)])
def test_rows_that_end_with_what_they_share(heads, kv_heads, dim, shared, rows, cache):
    """Rows cut back to what they share, or near to it, under windows of about as many positions; others that are longer.  (So many that the
    kernel for shared pages is what runs.)"""
    case = Wide([(0, shared, 16 + 40 * (i % 30)) for i in range(rows)] + [(None, 0, 200)], heads, kv_heads, dim, 16, cache, seed=shared, spread=0.5)
    groups, full = case.groups(), case.lengths.clone()
    case.table = torch.cat([case.table, torch.full((len(full), 200), -1, device="cuda", dtype=torch.int32)], 1)
    kind = torch.arange(len(full), device="cuda") % 3
    case.lengths = torch.where(groups.shared > 0, torch.where(kind == 0, shared, torch.where(kind == 1, shared + 5, full)), full).int()
    for window in (shared - 1, shared, shared + 1, shared + 16, 0):
        out = case.check(groups=groups, window=window)
        assert not (out == 0).all(-1).any()
