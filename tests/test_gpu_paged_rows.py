"""Paged attention of large batches, every row against fp64, into outputs that hold something else before."""
import math
import random

import pytest
import torch

import penny_b200.ops as P
from test_gpu_paged_attention import BF, E4M3, HF, STEP, _case

pytestmark = pytest.mark.gpu


def _spread(rows, top):
    """Lengths of every size up to `top`, short ones and empty rows most often."""
    rng = random.Random(rows)
    return [rng.choice([0, 1, rng.randrange(17), rng.randrange(100), rng.randrange(top + 1)]) for _ in range(rows)]


def _check_all(c, out, lse, window=0):
    """The bounds of the other attention tests, for all rows at once."""
    q, k, v = c["q"], c["k"], c["v"]
    B, H, dim = q.shape
    page, Hkv = k.shape[1:3]
    n, G, bf = c["lengths"].clamp(min=0).long(), H // Hkv, k.dtype == BF
    first = (n - window).clamp(min=0) if window else torch.zeros_like(n)
    longest = int((n - first).max())
    at = first[:, None] + torch.arange(longest, device="cuda")
    there = at < n[:, None]
    at = torch.where(there, at, 0)
    ids = torch.where(there, c["table"].long().gather(1, at // page), 0)
    rows = lambda p: (p.view(torch.uint8)[ids, at % page].view(E4M3) if p.dtype == E4M3 else p[ids, at % page])  # noqa: E731
    for kh in range(Hkv):
        keys, vals = (rows(p[:, :, kh]).double().masked_fill(~there[..., None], 0) for p in (k, v))
        if k.dtype == E4M3:
            keys, vals = keys * c["k_scale"][kh].double(), vals * c["v_scale"][kh].double()
        qh, scale = q[:, kh * G:kh * G + G].double(), 1 / math.sqrt(dim)
        s = (qh @ keys.transpose(1, 2) * scale).masked_fill(~there[:, None], -math.inf)
        off = dim * 2.0 ** -23 * scale * (qh.abs() @ keys.abs().transpose(1, 2)).amax(-1, keepdim=True) + 2.0 ** -20
        true = s.logsumexp(-1)
        p = (s - true.masked_fill(true == -math.inf, 0)[..., None]).exp()
        want, size = p @ vals, p @ vals.abs()
        floor = 0 if bf else (n[:, None, None] - first[:, None, None]) * 2.0 ** (-32 if q.dtype == BF else -40) * vals.abs().amax((1, 2))[:, None, None]
        bound = ((STEP[BF] if bf else STEP[HF]) + 2 * off) * size * (1 + 2.0 ** -6) + STEP[q.dtype] * want.abs() * (1 + 2.0 ** -6) + floor
        bound = bound + (2.0 ** -25 if q.dtype == HF else 0)
        got, got_lse = out[:, kh * G:kh * G + G].double(), lse[:, kh * G:kh * G + G].double()
        wrong = ((got - want).abs() <= bound).logical_not().flatten(1).any(1)  # (NaN too)
        assert not wrong.any(), (kh, wrong.nonzero().flatten().tolist()[:20])
        empty = n == 0
        assert (got_lse[empty] == -math.inf).all()
        wrong = ((got_lse - true).abs() <= off[..., 0] + 2.0 ** -22 * true.abs()).logical_not().any(1) & ~empty
        assert not wrong.any(), (kh, wrong.nonzero().flatten().tolist()[:20])


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, HF), (BF, E4M3), (HF, E4M3)])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,window", [
    ([1, 7000] + [40] * 130, 8, 2, 128, 0), ([600] * 300, 8, 8, 128, 0), ([7, 0, 30] * 1500, 2, 1, 128, 0), (_spread(999, 700), 8, 2, 64, 0),
    (_spread(3001, 90), 3, 1, 256, 0), (_spread(130, 3000), 18, 1, 128, 700), (_spread(64, 4000), 4, 4, 64, 0), (_spread(33, 300) * 31, 1, 1, 64, 20),
    ([0] * 31 + [333] + [0] * 32 + [444] + [0] * 63 + [1], 16, 2, 128, 0)])
def test_every_row(dtype, cache, lengths, heads, kv_heads, dim, window):
    c = _case(lengths, heads, kv_heads, dim, 16, dtype, cache, seed=21)
    out = torch.full_like(c["q"], float("nan"), memory_format=torch.contiguous_format)
    lse = torch.full(c["q"].shape[:2], float("nan"), device="cuda")
    P.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lengths"], out=out, lse=lse, window=window, **{s: c[s] for s in ("k_scale", "v_scale") if s in c})
    _check_all(c, out, lse, window)
