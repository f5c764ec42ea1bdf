"""The longest a row can be: max_len of the page tables, the cache and the decoder."""
import pytest
import torch

import penny_b200.ops as P
from penny_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder

pytestmark = pytest.mark.gpu


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page", [1, 7, 16, 50, 64])
def test_rows_end_at_max_len(page):
    """A row gets max_len positions and no more, whether or not whole pages hold them; one that is refused stays as it is."""
    c = P.PagedKVCache(1, 3, 50, 1, 64, page_size=page)
    assert c.advance(_ints(50, 49, 51), 200).granted.tolist() == [True, True, False]
    assert c.lengths.tolist() == [50, 49, 0]
    assert c.advance(_ints(1, 1, 50), 200).granted.tolist() == [False, True, True]
    step = c.advance(_ints(-1, 1, 0), 4)
    assert step.granted.tolist() == [True, False, True] and step.slots.tolist() == [-1] * 4 and c.lengths.tolist() == [49, 50, 50]
    assert c.advance(_ints(1, 0, -50), 1).granted.all() and c.lengths.tolist() == [50, 50, 0]


def test_page_tables_with_a_longest_row():
    for longest, granted in ((None, True), (48, True), (40, True), (39, False), (1 << 40, True)):
        table, lengths, free, count = torch.zeros(1, 3, dtype=torch.int32, device="cuda"), _ints(30), _ints(5, 6, 7), _ints(3)
        assert P.page_tables(table, lengths, free, count, _ints(10), 16, 16, max_len=longest).granted.tolist() == [granted]
        assert lengths.tolist() == [40 if granted else 30]
    # a row that is longer already keeps what it has, may shrink, and gets nothing
    table, lengths, free, count = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), _ints(45, 48), _ints(5, 6, 7), _ints(1)
    assert P.page_tables(table, lengths, free, count, _ints(1, -20), 16, 16, max_len=40).granted.tolist() == [False, True]
    assert lengths.tolist() == [45, 28] and int(count) == 2


def test_decoder_ends_at_max_len():
    m = LlamaTPDecoder(LlamaConfig.tiny(), world=1, max_batch=2, max_len=50, full_init=True, page_size=16)
    m.fill_synthetic_kv(49)
    m.capture()
    m.step(torch.tensor([1, 2]))
    with pytest.raises(RuntimeError, match="50 positions"):
        m.step(torch.tensor([1, 2]))
    assert m.paged.lengths.tolist() == [50, 50]


def test_tables_past_two_to_the_31_positions():
    """A workspace for a table that could hold more positions than a row can have, and the attention with it and without."""
    c = P.PagedKVCache(1, 1, 2 ** 31, 1, 64, page_size=1 << 16, pages=2)
    assert c.table.shape[1] * c.page_size == 2 ** 31
    step = c.advance(_ints(70000), 70000)
    qkv = torch.randn(70000, 6 * 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    c.append(0, qkv, step, 4, 1e4)
    q = qkv[-1:, :256].unflatten(1, (4, 64))
    ws = c.workspace(4)
    assert ws.numel() == P.paged_attention_workspace_bytes(1, 4, 1, 64, 2 ** 31) == P.paged_attention_workspace_bytes(1, 4, 1, 64, 2 ** 40) > 0
    out = c.attend(0, q, workspace=ws)
    assert torch.equal(out, c.attend(0, q))
    k, v = (t[0].double() for t in c.rows_of(0, 0, 70000))
    p = (q[0].double() @ k.t() / 8).softmax(-1)
    want, size = p @ v, p @ v.abs()
    assert ((out[0].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -12) * size + 2.0 ** -8 * want.abs()).all()  # (a weight and the output rounded)
