"""Log probabilities of a decoder's rows between a fork and the next step."""
import pytest
import torch

from test_gpu_shared_decoder import _model, _prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("use_graph", [False, True])
def test_forked_rows_have_their_sources_logits(use_graph):
    model = _model(sharing=True, use_graph=use_graph)
    if use_graph:
        model.fill_synthetic_kv(20)
        model.capture()
    _prompts(model, [90, 33, 47])
    model.step(torch.arange(8) * 5)
    model.release([3, 4, 5, 6, 7])
    of = {3: 1, 5: 0, 4: 1, 7: 2}
    before = model.logprobs(top=6)
    model.fork(list(of.values()), list(of))
    got = model.logprobs(top=6)
    for t, s in of.items():
        assert all(torch.equal(a[t], b[s]) for a, b in zip(got, before)), t
    rest = [0, 1, 2, 6]
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got, before))


def test_tokens_of_the_caller():
    """Continuations that take different tokens from the same logits."""
    model = _model(sharing=True)
    _prompts(model, [90, 33])
    model.step(torch.arange(8) * 5)
    model.release(range(1, 8))
    model.fork([0] * 7, range(1, 8))
    greedy = model.logprobs(top=8)
    tokens = greedy.top_ids[0].cpu()
    got = model.logprobs(top=8, tokens=tokens)
    assert torch.equal(got.logprobs, greedy.top_logprobs[0]) and torch.equal(got.entropy, greedy.entropy) and torch.equal(got.top_ids, greedy.top_ids)
    assert all(torch.equal(a, b) for a, b in zip(model.logprobs(8, tokens.cuda()), got))
    assert all(torch.equal(a, b) for a, b in zip(model.logprobs(8, tokens.cuda().repeat_interleave(2)[::2]), got))
    model.step(tokens)
    want = torch.log_softmax(model.logits.double(), -1).gather(1, tokens.cuda()[:, None])[:, 0]
    assert (model.logprobs(tokens=tokens).logprobs.double() - want).abs().max() < 1e-5
    for bad in (tokens[:7], tokens.int(), tokens[None]):
        with pytest.raises(ValueError, match="tokens"):
            model.logprobs(tokens=bad)
