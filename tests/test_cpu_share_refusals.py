"""Calls of the operators on shared pages and of the log probabilities that are refused, on tensors without a GPU."""
import pytest
import torch

import penny_b200.ops as P

BF = torch.bfloat16
ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def _state(**over):
    return dict(table=ints(3, 4), lengths=ints(3), free=ints(10), free_count=ints(1), refs=ints(10)) | over


STATE = [(dict(table=torch.zeros(3, 4)), "int32"), (dict(table=ints(3)), "int32"), (dict(table=ints(4, 3).t()), "contiguous rows"), (dict(table=ints(0, 4)), "int32"),
         (dict(table=ints(1, 4).expand(3, 4)), "do not overlap"), (dict(lengths=ints(4)), "lengths"), (dict(free=ints(0)), "free"), (dict(free_count=ints(2)), "free_count"),
         (dict(refs=ints(9)), "refs"), (dict(refs=torch.zeros(10)), "refs"), (dict(table=ints(8193, 1), lengths=ints(8193)), "PAGED_MAX_ROWS"), (dict(page_size=0), "page size"),
         (dict(), "CUDA")]


@pytest.mark.parametrize("over,said", STATE + [(dict(source=ints(3)), "forks"), (dict(source=ints(2).long(), target=ints(2).long()), "forks"),
                                               (dict(source=ints(8193), target=ints(8193)), "forks"), (dict(source=ints(4)[::2]), "forks")])
def test_fork(over, said):
    with pytest.raises(RuntimeError, match=said):
        P.page_fork(**(_state(source=ints(2), target=ints(2), page_size=16) | over))


@pytest.mark.parametrize("over,said", STATE)
def test_compact(over, said):
    with pytest.raises(RuntimeError, match=said):
        P.page_compact(**(_state(page_size=16) | over))


def test_state_that_shares_memory():
    both = ints(20)
    for call in (lambda **a: P.page_fork(**a, source=ints(2), target=ints(2), page_size=16), lambda **a: P.page_compact(**a, page_size=16),
                 lambda **a: P.page_tables(**a, new=ints(3), page_size=16, tokens=0)):
        with pytest.raises(RuntimeError, match="of their own"):
            call(**_state(free=both[:10], refs=both[9:19]))
    with pytest.raises(RuntimeError, match="of their own"):
        P.page_fork(**_state(lengths=both[:3]), source=both[2:4], target=ints(2), page_size=16)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.page_fork(**_state(), source=both[:2], target=both[:2], page_size=16)  # (rows onto themselves: nothing is granted)
    with pytest.raises(RuntimeError, match="refs"):
        P.page_tables(**_state(refs=ints(11)), new=ints(3), page_size=16, tokens=0)


pool = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)  # noqa: E731
ONE = pool(6, 4, 2, 64)


@pytest.mark.parametrize("pools,lists,said", [
    ([pool(6, 4, 64)], None, "kv_heads, dim"), ([pool(0, 4, 2, 64)], None, "kv_heads, dim"), ([pool(6, 4, 2, 4)], None, "16 bytes"),
    ([pool(6, 4, 64, 2).transpose(2, 3)], None, "contiguous in dim"), ([pool(6, 4, 2, 68)[..., :64]], None, "16 bytes"), ([pool(6, 4, 2, 72)[..., 4:68]], None, "aligned"),
    ([pool(1, 4, 2, 64).expand(6, 4, 2, 64)], None, "overlap"), ([pool(6, 1, 2, 64).expand(6, 4, 2, 64)], None, "overlap"),
    ([pool(5000).as_strided((6, 4, 2, 64), (256, 128, 64, 1))], None, "overlap"), ([ONE, pool(6, 4, 3, 64)], None, "one shape"), ([ONE, pool(6, 4, 2, 64, dtype=torch.uint8)], None, "size of values"),
    ([ONE, pool(6, 2, 4, 64).transpose(1, 2)], None, "strides"), ([ONE, ONE], None, "apart"), ([pool(6, 4, 2, 64).requires_grad_()], None, "gradients"),
    ([ONE], (ints(3), ints(2)), "copies"), ([ONE], (ints(3).long(), ints(3).long()), "copies"), ([ONE], (ints(6)[::2], ints(3)), "copies"),
    ([ONE.view(torch.int32)], (ONE.view(torch.int32).view(-1)[:8], ints(8)), "apart"), ([ONE], None, "CUDA"),
    ([pool(12, 4, 2, 64)[:6], pool(12, 4, 2, 64)[6:]], None, "CUDA"), ([(b := pool(6, 2, 4, 2, 64))[:, 0], b[:, 1]], None, "CUDA"),
    ([pool(4, 6, 2, 64).transpose(0, 1)], None, "CUDA"), ([pool(2, 6, 4, 64).permute(1, 2, 0, 3)], None, "CUDA"), ([pool(2, 4, 6, 64).permute(2, 1, 0, 3)], None, "CUDA")])
def test_copy(pools, lists, said):
    with pytest.raises(RuntimeError, match=said):
        P.page_copy(pools, *(lists or (ints(3), ints(3))))


@pytest.mark.parametrize("over,said", [(dict(table=torch.zeros(3, 4)), "int32"), (dict(table=ints(4, 3).t()), "contiguous rows"), (dict(lengths=ints(2)), "lengths"),
                                       (dict(lengths=ints(3).long()), "lengths"), (dict(page_size=0), "page size"), (dict(table=ints(8193, 1), lengths=ints(8193)), "PAGED_MAX_ROWS"),
                                       (dict(), "CUDA")])
def test_groups(over, said):
    with pytest.raises(RuntimeError, match=said):
        P.page_groups(**(dict(table=ints(3, 4), lengths=ints(3), page_size=16) | over))


def _groups(order=3, starts=4, shared=3):
    return P.PageGroups(ints(order), ints(starts), ints(shared))


@pytest.mark.parametrize("over,said", [
    (dict(groups=_groups(order=2)), "groups are"), (dict(groups=_groups(starts=3)), "groups are"), (dict(groups=_groups(shared=4)), "groups are"),
    (dict(groups=(ints(3), ints(4).long(), ints(3))), "groups are"), (dict(groups=(ints(6)[::2], ints(4), ints(3))), "groups are"),
    (dict(groups=_groups(8193, 8194, 8193), q=torch.zeros(8193, 8, 64, dtype=BF), table=ints(8193, 1), lengths=ints(8193)), "PAGED_MAX_ROWS"),
    (dict(groups=_groups(), window=-1), "window"), (dict(groups=_groups()), "CUDA")])
def test_attention_with_groups(over, said):
    with pytest.raises(RuntimeError, match=said):
        P.paged_attention(**(dict(q=torch.zeros(3, 8, 64, dtype=BF), k=torch.zeros(6, 16, 2, 64, dtype=BF), v=torch.zeros(6, 16, 2, 64, dtype=BF), table=ints(3, 4),
                                  lengths=ints(3)) | over))


def test_cache_without_sharing():
    c = P.PagedKVCache(2, 3, 40, 2, head_dim=64, page_size=16, device="cpu")
    for call in (lambda: c.fork(ints(1), ints(1)), c.compact):
        with pytest.raises(ValueError, match="sharing"):
            call()
    c = P.PagedKVCache(2, 3, 40, 2, head_dim=64, page_size=16, device="cpu", sharing=True)
    assert c.refs.tolist() == [0] * 9 and len(c.snapshot()) == 5


@pytest.mark.parametrize("over,said", [
    (dict(logits=torch.zeros(3, 50, dtype=torch.float64)), "bf16, fp16 or fp32"), (dict(logits=torch.zeros(50)), "rows, vocab"), (dict(logits=torch.zeros(3, 0)), "rows, vocab"),
    (dict(logits=torch.zeros(50, 3).t()), "contiguous rows"), (dict(tokens=torch.zeros(2, dtype=torch.int64)), "tokens"), (dict(tokens=ints(3)), "tokens"),
    (dict(tokens=torch.zeros(6, dtype=torch.int64)[::2]), "tokens"), (dict(top=-1), "top"), (dict(top=33), "top"), (dict(logits=torch.zeros(3, 5), top=6), "top"),
    (dict(logits=torch.zeros(3, 50, requires_grad=True)), "gradients"), (dict(), "CUDA")])
def test_logprobs(over, said):
    with pytest.raises(RuntimeError, match=said):
        P.token_logprobs(**(dict(logits=torch.zeros(3, 50), tokens=torch.zeros(3, dtype=torch.int64), top=2) | over))
