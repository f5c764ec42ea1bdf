"""Attention with groups for tables that the kernel for shared pages cannot take."""
import pytest
import torch

import penny_b200.ops as P
from penny_b200._ext import ops
from penny_b200.parallel import schedule

pytestmark = pytest.mark.gpu


def test_long_tables_of_many_rows():
    """1024 rows, 32 heads, 2^20 positions a row: read each row by itself, as without groups."""
    rows, heads, page = 1024, 32, 64
    width = (1 << 20) // page
    assert not schedule.shared_fits(rows, heads, 1, width * page, 128)
    k, v = (torch.randn(6, page, heads, 128, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(rows, heads, 128, device="cuda").bfloat16()
    table = torch.full((rows, width), -1, device="cuda", dtype=torch.int32)
    table[:, 0] = 1
    table[:, 1] = torch.arange(rows, device="cuda") % 4 + 2
    lengths = (torch.arange(rows, device="cuda") % 130).int()
    groups = P.page_groups(table, lengths, page)
    assert int(groups.shared.max()) == page
    space = torch.empty(P.paged_attention_workspace_bytes(rows, heads, heads, 128, width * page, groups=True), dtype=torch.uint8, device="cuda")
    got = P.paged_attention(q, k, v, table, lengths, groups=groups, workspace=space)
    assert torch.equal(got, P.paged_attention(q, k, v, table, lengths)) and ops.gemm_error() == 0
