"""Paged attention where the weights of a long row are far below its largest one, and where its scores are large."""
import math

import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu
BF, HF, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
STEP = {BF: 2.0 ** -8, HF: 2.0 ** -11}


def _dominated(dtype, cache, n, at, gap, dim=64, page=64, heads=296):
    """One row of n positions for `heads` KV heads (so few CTAs have each that a warp walks a quarter of the row): all scores zero but
    that of position `at`, about `gap`; its values are zero, the others' two.  Every page but that position's is the same one."""
    width = -(-n // page)
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    table[0, at // page] = 1
    k, v = torch.zeros(2, page, 1, dim, device="cuda"), torch.full((2, page, 1, dim), 2.0, device="cuda")
    k[1, at % page, 0, 0], v[1, at % page] = 448 if cache == E4M3 else gap, 0
    scales = {} if cache != E4M3 else dict(k_scale=torch.full((heads,), gap / 448, device="cuda"), v_scale=torch.ones(heads, device="cuda"))
    k, v = (t.to(cache).expand(-1, -1, heads, -1) for t in (k, v))
    q = torch.zeros(1, heads, dim, dtype=dtype, device="cuda")
    q[..., 0] = 1
    score = float(k[1, at % page, 0, 0].float()) * (float(scales["k_scale"][0]) if scales else 1.0)
    lse = torch.zeros(1, heads, device="cuda")
    out = P.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), lse=lse, scale=1.0, **scales)
    tail = (n - 1) * math.exp(-score)
    return out, lse, 2 * tail / (1 + tail), score + math.log1p(tail)


@pytest.mark.parametrize("dtype,cache", [(HF, HF), (HF, E4M3), (BF, E4M3), (BF, BF)])
@pytest.mark.parametrize("n", [100003, 1600000])
@pytest.mark.parametrize("where", ["first", "early", "last"])
@pytest.mark.parametrize("gap", [17.4, 19.0, 12.0])
def test_one_key_far_above_the_others(dtype, cache, n, where, gap):
    """A weight is off by half a step of the type that meets V where that type holds it in full; an fp16 one also by 2 ** -25 of what the
    largest is multiplied by, 2 ** 15, or 2 ** 7 at least where the base lags (bf16 q of an e4m3 cache).  fp32's part: a score's base-2
    exponent (up to 32) to 2 ** -20, weights and outputs to 2 ** -17.  A warp walks n / 4 positions at most; a lane adds an eighth of
    their weights one after another to its sum (2 ** -24 of it each: n * 2 ** -29), and each position adds a product to the output
    (2 ** -23 of it each, for matrix instructions may cut off: n * 2 ** -25)."""
    at = {"first": 0, "early": n // 8, "last": n - 1}[where]
    out, lse, want, true = _dominated(dtype, cache, n, at, gap)
    floor = 0.0 if cache == BF else 2 * n * 2.0 ** (-32 if dtype == BF else -40)
    bound = (STEP[BF] if cache == BF else STEP[HF]) * want + STEP[dtype] * want + floor + 2.0 ** -25 + (2.0 ** -17 + n * (2.0 ** -29 + 2.0 ** -25)) * want
    err = (out.double() - want).abs().max().item()
    assert err <= bound, (err, bound)
    assert (lse.double() - true).abs().max().item() <= 2.0 ** -16 + n * 2.0 ** -29


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


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("top", [1.0, 1.9921875, 2.0 ** -12, 60000.0])
def test_small_values_of_q_beside_a_large_one(dtype, top):
    """q of an 8-bit cache whose score comes from values far under its largest one, which meets a key of zero: what fp16 holds beside the
    largest is not lost (values down to 2 ** -29 of it; scores to 2 ** -20, sums and logarithm to as much)."""
    dim, page = 64, 16
    small = top * (2.0 ** -20 if dtype == BF else 2.0 ** -9) * (1 + 2.0 ** -7)
    q = torch.zeros(1, 4, dim, dtype=dtype, device="cuda")
    q[..., 0], q[0, :, 1] = top, torch.tensor([1.0, 0.5, -0.25, 2.0 ** -8], device="cuda").to(dtype) * torch.tensor(small, device="cuda").to(dtype)
    k, v = torch.zeros(1, page, 1, dim, device="cuda"), torch.zeros(1, page, 1, dim, device="cuda")
    k[0, 1, 0, 1] = 448
    v[0, 1] = 1
    one, scale = torch.ones(1, device="cuda"), 1.75 / (448 * small)
    lse = torch.zeros(1, 4, device="cuda")
    out = P.paged_attention(q, k.to(E4M3), v.to(E4M3), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda"),
                            lse=lse, scale=scale, k_scale=one, v_scale=one)
    s = q[0, :, 1].double() * 448 * float(torch.tensor(scale, dtype=torch.float32))
    true = torch.log1p(s.exp())
    assert ((lse[0].double() - true).abs() <= 2.0 ** -18).all(), (lse, true)
    want = torch.sigmoid(s)[:, None]
    assert ((out[0].double() - want).abs() <= (STEP[HF] + STEP[dtype] + 2.0 ** -17) * want).all()
