"""Paged attention where the scores are large."""
import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu
BF, HF, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
STEP = {BF: 2.0 ** -8, HF: 2.0 ** -11}


@pytest.mark.parametrize("dtype,cache", [(HF, HF), (HF, E4M3), (BF, E4M3), (BF, BF)])
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 30, 2.0 ** 60])
def test_scores_too_large_for_their_fractions(dtype, cache, size):
    """Scores whose neighbours in fp32 are further apart than the type of the weights is wide: numbers, and those of the largest."""
    dim, n = 64, 333
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(6, 64, 1, dim, device="cuda", generator=g).to(cache) for _ in range(2))
    q = torch.randn(1, 8, dim, device="cuda", generator=g).to(dtype)
    one = torch.ones(1, device="cuda")
    scales = dict(k_scale=one, v_scale=one) if cache == E4M3 else {}
    table = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    out = P.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=size, **scales)
    s = torch.einsum("hd,td->ht", q[0].double(), k.double().view(-1, dim)[:n])
    # (64 products of values up to 5 in any order: scores apart by more than 2 ** -10 keep their order in fp32)
    top = s.topk(2, -1)
    assert out.isfinite().all()
    for h in range(8):
        if top.values[h, 0] - top.values[h, 1] > 2.0 ** -10:
            want = v.view(-1, dim)[top.indices[h, 0]].double()  # (the weight and the output rounded)
            assert ((out[0, h].double() - want).abs() <= ((STEP[BF] if cache == BF else STEP[HF]) + STEP[dtype]) * (1 + 2.0 ** -6) * want.abs()).all(), h
