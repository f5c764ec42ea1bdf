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
