"""A decoder whose rows are forked: continuations of one prompt, with their log probabilities, against rows that share nothing."""
import pytest
import torch

import penny_b200.ops as P
from penny_b200._ext import ops
from penny_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder

pytestmark = pytest.mark.gpu


def _model(**more):
    return LlamaTPDecoder(LlamaConfig.tiny(), max_batch=8, page_size=16, full_init=True, **(dict(max_len=80000, pages=400) | more))


def _prompts(model, lengths):
    """Rows 0, 1, ... with that many cached positions, the others empty."""
    model.fill_synthetic_kv(max(lengths))
    model.release(range(len(lengths), 8))
    leave = torch.tensor([n - max(lengths) for n in lengths] + [0] * (8 - len(lengths)), dtype=torch.int32, device="cuda")
    model.paged.advance(leave, 0)


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_forks_go_on_as_rows_of_their_own(use_graph, cache_dtype):
    scales = {} if cache_dtype == torch.bfloat16 else dict(cache_scales=tuple(torch.full((2,), 0.05, device="cuda") for _ in range(2)))
    model = _model(sharing=True, use_graph=use_graph, cache_dtype=cache_dtype, **scales)
    if use_graph:
        model.fill_synthetic_kv(20)
        model.capture()
    _prompts(model, [300, 75])
    free = int(model.paged.free_count)
    model.fork([0, 0, 0, 1, 1, 0], [2, 3, 4, 5, 6, 7])
    # whole pages are shared (18 of 300 positions, 4 of 75), one each is copied
    assert int(model.paged.free_count) == free - 6
    assert model.paged.lengths.tolist() == [300, 75, 300, 300, 300, 75, 75, 300]
    # the same cached positions in rows of their own
    plain = _model(use_graph=False, cache_dtype=cache_dtype, **scales)
    plain.paged.advance(model.paged.lengths.clone(), 8 * 300)
    for i in range(2):
        for pools, mine in ((model.paged.k, plain.paged.k), (model.paged.v, plain.paged.v)):
            for r, n in enumerate(model.paged.lengths.tolist()):
                at = torch.arange(n, device="cuda")
                a, b = model.paged.table[r, at // 16].long(), plain.paged.table[r, at // 16].long()
                mine[i].view(torch.uint8)[b, at % 16] = pools[i].view(torch.uint8)[a, at % 16]
    g = torch.Generator().manual_seed(3)
    for step in range(20):  # (over the end of a page)
        tokens = torch.randint(0, 2048, (8,), generator=g)
        model.step(tokens)
        plain.step(tokens)
        a, b = model.logits.float(), plain.logits.float()
        # two ways to add up the attention, each rounded to bf16 (2^-9 of it), through two layers
        assert (a - b).norm() < 0.02 * b.norm(), step
        if step == 0:
            assert model.paged.groups().shared.tolist() == [288, 64, 288, 288, 288, 64, 64, 288]
        got = model.logprobs(top=5)
        want = torch.log_softmax(a.double(), -1)
        assert torch.equal(got.top_ids[:, 0], model.next_tokens) and torch.equal(got.logprobs, got.top_logprobs[:, 0])
        assert (got.logprobs.double() - want.gather(1, model.next_tokens[:, None])[:, 0]).abs().max() < 1e-5
        assert (got.entropy.double() + (want.exp() * want).sum(-1)).abs().max() < 1e-5
    assert ops.gemm_error() == 0 and model.paged.lengths.tolist() == plain.paged.lengths.tolist()
    # the prompts leave, their forks go on
    model.release([0, 1])
    tokens = torch.randint(0, 2048, (8,), generator=g)
    plain.release([0, 1])
    model.step(tokens)
    plain.step(tokens)
    assert (model.logits[2:].float() - plain.logits[2:].float()).norm() < 0.02 * plain.logits[2:].float().norm()
    model.release(range(8))
    assert int(model.paged.free_count) == model.paged.pages and not model.paged.refs.any()


def test_greedy_forks_are_alike():
    model = _model(sharing=True)
    _prompts(model, [130])
    model.tokens.fill_(17)
    model.fork([0] * 7, range(1, 8))
    model.capture()
    got = model.decode(12)
    assert (got == got[:, :1]).all()
    moves = model.paged.compact()
    assert moves.copy_from.numel() == model.paged.pages // 2
    more = model.decode(3)
    assert (more == more[:, :1]).all()


def test_forks_that_are_refused():
    model = _model(sharing=True, pages=12)
    model.release(range(8))
    model.paged.advance(torch.tensor([100, 8, 0, 0, 0, 0, 0, 0], dtype=torch.int32, device="cuda"), 108)
    with pytest.raises(P.OutOfPages) as e:
        model.fork([0, 0, 0, 0, 1, 0], [2, 1, 3, 4, 5, 6])
    assert e.value.rows == [1, 6]  # (not empty; four pages for five forks)
    assert model.paged.lengths.tolist() == [100, 8, 100, 100, 100, 8, 0, 0]
    with pytest.raises(IndexError):
        model.fork([0], [8])
    with pytest.raises(ValueError, match="sharing"):
        _model().fork([0], [1])
    with pytest.raises(ValueError, match="page_size above 0"):
        LlamaTPDecoder(LlamaConfig.tiny(), max_batch=2, max_len=64, sharing=True)
