"""Calls of the paged KV cache that are refused, on tensors without a GPU."""
import pytest
import torch

import penny_b200.ops as P

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def _tables(**over):
    a = dict(table=ints(3, 4), lengths=ints(3), free=ints(10), free_count=ints(1), new=ints(3), page_size=16, tokens=8, out=None) | over
    return P.page_tables(**a)


def _step(tokens=8, rows=3):
    return (torch.zeros(tokens, dtype=torch.int64), ints(tokens), ints(rows + 1), torch.zeros(rows, dtype=torch.bool))


@pytest.mark.parametrize("over,said", [
    (dict(table=torch.zeros(3, 4)), "int32"), (dict(table=ints(3)), "int32"), (dict(table=ints(0, 4)), "int32"), (dict(table=ints(4, 3).t()), "contiguous rows"),
    (dict(table=ints(1, 4).expand(3, 4)), "do not overlap"), (dict(lengths=ints(4)), "lengths"), (dict(lengths=ints(6)[::2]), "lengths"),
    (dict(new=torch.zeros(3, dtype=torch.int64)), "new tokens"), (dict(free=ints(0)), "free"), (dict(free_count=ints(2)), "free_count"),
    (dict(page_size=0), "page size"), (dict(page_size=-16), "page size"), (dict(tokens=-1), "tokens"), (dict(tokens=2 ** 31), "tokens"),
    (dict(table=ints(8193, 1), lengths=ints(8193), new=ints(8193)), "PAGED_MAX_ROWS"), (dict(out=_step(9)), "out is"), (dict(out=_step(8, 4)), "out is"),
    (dict(out=_step(8)[:1] + (ints(12)[1:9],) + _step(8)[2:]), "aligned"), (dict(), "CUDA"),
])
def test_page_tables(over, said):
    with pytest.raises(RuntimeError, match=said):
        _tables(**over)


def test_page_tables_new_is_no_state():
    lengths = ints(3)
    with pytest.raises(RuntimeError, match="of their own"):
        _tables(lengths=lengths, new=lengths)


def _append(**over):
    a = dict(qkv=torch.zeros(5, 12 * 64, dtype=BF), k=torch.zeros(6, 16, 2, 64, dtype=BF), slots=torch.zeros(5, dtype=torch.int64), positions=ints(5),
             heads=8, theta=1e4) | over
    a.setdefault("v", torch.zeros_like(a["k"]))
    return P.paged_append(**a)


@pytest.mark.parametrize("over,said", [
    (dict(qkv=torch.zeros(5, 768)), "bf16 or fp16"), (dict(qkv=torch.zeros(5, 768, dtype=F8)), "bf16 or fp16"), (dict(qkv=torch.zeros(5, 760, dtype=BF)), "qkv must be"),
    (dict(qkv=torch.zeros(768, dtype=BF)), "qkv must be"), (dict(heads=7), "qkv must be"), (dict(qkv=torch.zeros(768, 5, dtype=BF).t()), "contiguous"),
    (dict(qkv=torch.zeros(5 * 768 + 1, dtype=BF)[1:].view(5, 768)), "aligned"), (dict(qkv=torch.zeros(1, 768, dtype=BF).expand(5, 768)), "contiguous"),
    (dict(k=torch.zeros(6, 16, 2, 64, dtype=torch.float16)), "projection's type"), (dict(k=torch.zeros(6, 16, 2, 64)), "bf16, fp16 or e4m3"),
    (dict(v=torch.zeros(6, 16, 2, 64, dtype=torch.float16)), "one type"), (dict(v=torch.zeros(6, 2, 16, 64, dtype=BF).transpose(1, 2)), "strides"),
    (dict(k=torch.zeros(6, 16, 128, dtype=BF)), "kv_heads, dim"), (dict(k=torch.zeros(1, 16, 2, 64, dtype=BF).expand(6, 16, 2, 64), v=torch.zeros(1, 16, 2, 64, dtype=BF).expand(6, 16, 2, 64)), "overlap"),
    (dict(k=torch.zeros(6, 16, 64, 2, dtype=BF).transpose(2, 3)), "contiguous in dim"),
    (dict(k=torch.zeros(6, 16, 2, 72, dtype=BF)[..., :64], v=torch.zeros(6, 16, 2, 72, dtype=BF)[..., 4:68]), "aligned"),
    (dict(k=torch.zeros(6, 16, 2, 8, dtype=BF), qkv=torch.zeros(5, 96, dtype=BF)), "multiple of 16"),
    (dict(k=torch.zeros(6, 16, 2, 272, dtype=BF), qkv=torch.zeros(5, 12 * 272, dtype=BF)), "multiple of 16"),
    (dict(k=torch.zeros(6, 16, 2, 64, dtype=F8)), "beside e4m3"), (dict(k_scale=torch.ones(2), v_scale=torch.ones(2)), "beside e4m3"),
    (dict(k=torch.zeros(6, 16, 2, 64, dtype=F8), k_scale=torch.ones(2), v_scale=torch.ones(3)), "kv_heads. fp32"),
    (dict(slots=ints(5)), "slots"), (dict(slots=torch.zeros(4, dtype=torch.int64)), "slots"), (dict(positions=torch.zeros(5, dtype=torch.int64)), "positions"),
    (dict(theta=0.0), "theta"), (dict(theta=float("inf")), "theta"), (dict(theta=float("nan")), "theta"), (dict(out=torch.zeros(5, 768, dtype=BF)), "out must"),
    (dict(out=torch.zeros(5, 640)), "out must"), (dict(qkv=torch.zeros(5, 768, dtype=BF, requires_grad=True)), "gradients"), (dict(), "CUDA"),
])
def test_paged_append(over, said):
    with pytest.raises(RuntimeError, match=said):
        _append(**over)


def _attend(**over):
    a = dict(q=torch.zeros(3, 8, 64, dtype=BF), k=torch.zeros(6, 16, 2, 64, dtype=BF), table=ints(3, 4), lengths=ints(3)) | over
    a.setdefault("v", torch.zeros_like(a["k"]))
    return P.paged_attention(**a)


@pytest.mark.parametrize("over,said", [
    (dict(q=torch.zeros(3, 8, 64)), "bf16 or fp16"), (dict(q=torch.zeros(3, 512, dtype=BF)), "rows, heads, dim"), (dict(q=torch.zeros(3, 8, 128, dtype=BF)), "rows, heads, dim"),
    (dict(q=torch.zeros(3, 7, 64, dtype=BF)), "multiple of the caches"), (dict(q=torch.zeros(3, 0, 64, dtype=BF)), "multiple of the caches"),
    (dict(q=torch.zeros(3, 64, 8, dtype=BF).transpose(1, 2)), "contiguous"), (dict(q=torch.zeros(3, 8, 68, dtype=BF)[..., :64]), "aligned"),
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.float16)), "projection's type"),
    (dict(q=torch.zeros(3, 8, 96, dtype=BF), k=torch.zeros(6, 16, 2, 96, dtype=BF)), "dim 64, 128 or 256"), (dict(table=ints(2, 4)), "table"),
    (dict(table=ints(3, 0)), "table"), (dict(table=torch.zeros(3, 4, dtype=torch.int64)), "table"), (dict(table=ints(4, 3).t()), "table"), (dict(lengths=ints(2)), "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), "lengths"), (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"), (dict(out=torch.zeros(3, 8, 64)), "out like q"),
    (dict(out=torch.zeros(1, 8, 64, dtype=BF).expand(3, 8, 64)), "out like q"), (dict(out=torch.zeros(10 * 64, dtype=BF).as_strided((3, 8, 64), (64, 64, 1))), "apart"),
    (dict(out=torch.zeros(4000, dtype=BF).as_strided((3, 8, 64), (64 * 7, 64, 1))), "apart"), (dict(scale=1e300), "scale"),
    (dict(k=torch.zeros(6, 16, 2, 64, dtype=BF, requires_grad=True)), "gradients"), (dict(out=torch.zeros(8, 3, 64, dtype=BF).transpose(0, 1)), "CUDA"),
    (dict(out=torch.zeros(3, 9, 72, dtype=BF)[:, 1:, :64]), "CUDA"), (dict(lse=torch.zeros(3, 8, dtype=BF)), "lse"), (dict(lse=torch.zeros(8, 3).t()), "lse"),
    (dict(k=torch.zeros(0, 16, 2, 64, dtype=BF)), "pages"), (dict(k=torch.zeros(6, 16, 2, 64, dtype=F8), k_scale=torch.ones(2)), "beside e4m3"),
    (dict(workspace=torch.zeros(65, dtype=torch.uint8)[1:]), "aligned"), (dict(q=torch.zeros(3, 8, 64, dtype=BF, requires_grad=True)), "gradients"), (dict(), "CUDA"),
])
def test_paged_attention(over, said):
    with pytest.raises(RuntimeError, match=said):
        _attend(**over)


def test_cache():
    for over in (dict(rows=0), dict(page_size=0), dict(pages=0), dict(max_len=0), dict(rows=8193), dict(dtype=torch.float32), dict(k_scale=torch.ones(2)),
                 dict(dtype=F8, k_scale=[torch.ones(2)] * 3)):
        with pytest.raises(ValueError):
            P.PagedKVCache(**(dict(layers=2, rows=2, max_len=40, kv_heads=2, head_dim=64, device="cpu") | over))
    c = P.PagedKVCache(2, 3, 40, 2, head_dim=64, page_size=16, device="cpu", dtype=F8)
    assert c.pages == 9 and c.table.shape == (3, 3) and c.k[1].shape == (9, 16, 2, 64) and int(c.free[int(c.free_count) - 1]) == 0
    assert c.k_scale[1].tolist() == [1, 1]
