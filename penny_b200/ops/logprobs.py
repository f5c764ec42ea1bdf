"""Log probabilities of the tokens of a step or of a text, with the entropy and the likeliest alternatives.

    import penny_b200.ops as P
    got = P.token_logprobs(logits, tokens, top=20)    # logits [rows, vocab], tokens [rows] int64
    got.logprobs, got.entropy, got.top_logprobs, got.top_ids

One pass over the logits, nothing waits for the device, the call may be captured in a CUDA graph.  The reference has no sampling: it
serves that of vLLM and SGLang (README.md:20-33).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .._ext import ops


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # [rows] fp32: of the given tokens
    entropy: torch.Tensor       # [rows] fp32, in nats
    top_logprobs: torch.Tensor  # [rows, top] fp32: of the likeliest tokens, descending
    top_ids: torch.Tensor       # [rows, top] int64: of equal logits the lowest id first


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Under softmax(logits[r]): the log probability of token tokens[r], the entropy, and the `top` likeliest tokens.

    logits [rows, vocab]: bf16, fp16 or fp32, rows contiguous, any stride and alignment; tokens [rows] int64; top: 0 to 32, no more than the
    vocabulary.  A logit of minus infinity is a token that cannot come: log probability minus infinity, nothing in the entropy.  A row
    of nothing else has log probabilities of minus infinity and entropy 0; one with NaN or plus infinity NaN throughout (its top_ids say
    nothing).  A token that the vocabulary does not have (-1: a row that is padding) has NaN."""
    return TokenLogprobs._make(ops.token_logprobs(logits, tokens, top))
