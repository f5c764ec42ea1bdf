"""Tensors of the paged operators that ask for gradients, which these calls do not have: refused, but for calls without gradients."""
import pytest
import torch

import penny_b200.ops as P

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def _call(attend, **over):
    k = torch.zeros(6, 16, 2, 64, dtype=F8)
    a = dict(k_scale=torch.ones(2), v_scale=torch.ones(2)) | over
    if attend:
        return P.paged_attention(torch.zeros(3, 8, 64, dtype=BF), k, k.clone(), ints(3, 4), ints(3), **a)
    return P.paged_append(torch.zeros(5, 768, dtype=BF), k, k.clone(), torch.zeros(5, dtype=torch.int64), ints(5), 8, 1e4, **a)


@pytest.mark.parametrize("attend,name,like", [
    (True, "k_scale", torch.ones(2)), (True, "v_scale", torch.ones(2)), (True, "out", torch.zeros(3, 8, 64, dtype=BF)), (True, "lse", torch.zeros(3, 8)),
    (False, "k_scale", torch.ones(2)), (False, "v_scale", torch.ones(2)), (False, "out", torch.zeros(5, 640, dtype=BF))])
def test_gradients(attend, name, like):
    leaf = like.clone().requires_grad_()
    for t in (leaf, leaf * 1):
        with pytest.raises(RuntimeError, match="gradients"):
            _call(attend, **{name: t})
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            _call(attend, **{name: t})
