"""Attention over shared pages where the base of the weights moves in the middle of a tile of positions."""
import math

import pytest
import torch

from test_gpu_paged_shared import BF, F8, HALF
from test_gpu_paged_shared_wide import Wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [BF, HALF, F8])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 2, 64), (300, 1, 64)])
def test_base_that_moves_behind_half_a_tile(cache, heads, kv_heads, dim):
    """In every tile of 128 positions the second half has a score so far above all in front of it that their weights are scaled; the values
    of the first half are larger, so that what was scaled counts beside what was not."""
    case = Wide([(0, 512, n) for n in (1, 100, 400)] + [(None, 0, 500)], heads, kv_heads, dim, 16, cache, seed=dim, spread=1.0)
    g = torch.Generator(device="cuda").manual_seed(dim)
    unit = 0.02 if cache == F8 else 1.0
    if cache == F8:
        case.scales = [torch.full((kv_heads,), unit, device="cuda") for _ in range(2)]
    sign = torch.where(case.q[:1, :1] < 0, -1.0, 1.0)  # one direction for all queries
    case.q = (0.8 * sign).expand_as(case.q).to(case.q.dtype).contiguous()
    # a key of c times that direction scores 0.8 c sqrt(dim): 2^11 (fp16 weights 2^16) more in every tile than in the one before
    step = (11 if cache == BF else 16) * math.log(2) / (0.8 * math.sqrt(dim))
    pos = torch.full(case.k.shape[:2], -1, device="cuda")  # which position lies where
    for r, n in enumerate(case.lengths.tolist()):
        at = torch.arange(n, device="cuda")
        pos[case.table[r, at // 16].long(), at % 16] = at
    pos = pos[..., None, None]
    k = 0.02 * torch.randn(case.k.shape, device="cuda", generator=g) + (pos % 128 == 100) * step * (pos // 128 + 1).clamp(max=5) * sign[0, 0]
    v = torch.randn(case.v.shape, device="cuda", generator=g) * torch.where(pos % 128 < 64, 256.0, 1.0) * (0.005 if cache == F8 else 1.0)
    nan = torch.full((), math.nan, device="cuda")
    case.k, case.v = ((torch.where(pos < 0, nan, t / unit)).to(cache) for t in (k, v))
    first = case.check()
    for _ in range(4):
        assert torch.equal(case.check(), first)
