"""Log probabilities are not above zero and entropies not below, wherever a row's largest logits stand."""
import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (40, 32001), (600, 20000)])
def test_a_logit_that_dominates(dtype, rows, vocab):
    """One logit stands by 0.1 to 40 above another that is met first (by up to 8 it does not become what the sums count from), all others far
    below; and among plain ones."""
    for below in (-200.0, -12.0, 0.0):
        x = torch.full((rows, vocab), below, device="cuda")
        at = (torch.arange(rows, device="cuda") * 7919) % vocab
        x[torch.arange(rows), (at + vocab // 2) % vocab] = torch.linspace(0.1, 40, rows, device="cuda")
        x[torch.arange(rows), at] = 0.0
        for offset in (0.0, 300.0):
            y = (x + offset).to(dtype)
            tokens = y.argmax(-1)
            got = P.token_logprobs(y, tokens, 4)
            assert (got.logprobs <= 0).all() and (got.top_logprobs <= 0).all() and (got.entropy >= 0).all()
            want = torch.log_softmax(y.double(), -1)
            entropy = -torch.where(want > -700, want.exp() * want, 0).sum(-1)
            # (differences of fp32 numbers of up to 8 beside the base, and of sums of up to 2^17 terms)
            assert (got.logprobs.double() - want.gather(1, tokens[:, None])[:, 0]).abs().max() < 2e-5
            assert (got.entropy.double() - entropy).abs().max() < 2e-4
