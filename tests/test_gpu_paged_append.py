"""Rotary positions and stores into pages, against fp64."""
import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step of a value's own size
E4M3 = torch.float8_e4m3fn


def _pool(pages, page, heads, dim, dtype, by_head, gen):
    shape = (pages, heads, page, dim) if by_head else (pages, page, heads, dim)
    x = torch.randn(*shape, device="cuda", generator=gen).to(dtype)
    return x.transpose(1, 2) if by_head else x


def _check(got, want, size, step, msg):
    """Half a step of the value's type and of its smallest values, and what fp32 makes of the angle's fraction (2 ** -24 of a turn
    is 2 ** -21.3 rad) and of two products, of the values that were turned (`size`)."""
    small = {2.0 ** -8: 0.0, 2.0 ** -11: 2.0 ** -25, 2.0 ** -4: 2.0 ** -10}[step]
    err = (got.double() - want).abs()
    assert (err <= (step + 1e-6) * want.abs() + size * 2.0 ** -20 + small).all(), (msg, float(err.max()))


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,page,pad", [
    (1, 4, 1, 128, 16, 0), (7, 3, 3, 16, 1, 2), (64, 32, 8, 128, 16, 8), (33, 20, 20, 64, 24, 1), (130, 8, 1, 256, 5, 0), (50, 0, 2, 48, 64, 3),
    (4737, 4, 2, 64, 16, 3), (9001, 2, 1, 128, 33, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_append(tokens, heads, kv_heads, dim, page, pad, dtype, cache):
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    kind, by_head, n = dtype if cache == "same" else E4M3, tokens % 2 == 0, tokens + pad
    pages = -(-tokens // page) + 3
    k, v = (_pool(pages, page, kv_heads, dim, kind, by_head, g) for _ in range(2))
    scales = {} if cache == "same" else {s: 0.02 + 0.01 * torch.rand(kv_heads, device="cuda", generator=g) for s in ("k_scale", "v_scale")}
    width = (heads + 2 * kv_heads) * dim
    wide = torch.randn(n, width + 8, device="cuda", generator=g).to(dtype)
    wide[min(2, tokens - 1), heads * dim:width] *= 40  # (some past what e4m3 holds)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:n]
    slots[tokens:] = -1
    if tokens > 5:
        slots[4], slots[5] = pages * page, 2 ** 40  # no slots of the pool
    real = (slots >= 0) & (slots < pages * page)
    positions = torch.randint(0, 130000, (n,), device="cuda", generator=g, dtype=torch.int32)
    positions[0] = 0
    x = wide[:, :width].double().view(n, -1, 2, dim // 2)
    ang = positions.double()[:, None] * 5e5 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float64) * 2 / dim)
    a, b = x[:, :heads + kv_heads].unbind(2)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    size = torch.cat([a.abs() + b.abs()] * 2, -1)
    value = x[:, heads + kv_heads:].flatten(2)
    for out in (None, torch.full((n, (heads + kv_heads) * dim + 16), 7.0, dtype=dtype, device="cuda")):
        qkv, k1, v1 = wide.clone()[:, :width], k.clone(), v.clone()
        k1, v1 = (torch.empty_strided(t.shape, k.stride(), dtype=kind, device="cuda").copy_(t) for t in (k1, v1))
        rot = None if out is None else out[:, :(heads + kv_heads) * dim]
        P.paged_append(qkv, k1, v1, slots, positions, heads, 5e5, out=rot, **scales)
        got = (qkv[:, :(heads + kv_heads) * dim] if rot is None else rot).unflatten(1, (-1, dim))
        _check(got[real], turned[real], size[real], STEP[dtype], "turned")
        # rows without a slot, values, what lies behind the rows: as they were
        if rot is None:
            assert torch.equal(got[~real], wide[:, :(heads + kv_heads) * dim].unflatten(1, (-1, dim))[~real])
            assert torch.equal(qkv[:, (heads + kv_heads) * dim:], wide[:, (heads + kv_heads) * dim:width])
        else:
            assert torch.equal(qkv, wide[:, :width]) and (out[~real] == 7).all() and (out[:, (heads + kv_heads) * dim:] == 7).all()
        for pool, old, new, most, sc in ((k1, k, turned[:, heads:], size[:, heads:], "k_scale"), (v1, v, value, value.abs(), "v_scale")):
            rows = slots[real]
            there = pool.reshape(-1, kv_heads, dim)[rows]
            if cache == "e4m3":
                by = scales[sc].double()[:, None]
                _check(there, (new[real] / by).clamp(-448, 448), most[real] / by, 2.0 ** -4, sc)
            else:
                _check(there, new[real], most[real] if sc == "k_scale" else 0 * most[real], STEP[dtype], sc)
                if sc == "v_scale":
                    assert torch.equal(there, wide[:, :width].view(n, -1, dim)[:, heads + kv_heads:][real])
            rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
            rest[rows] = False
            assert torch.equal(pool.reshape(-1, kv_heads, dim).view(torch.uint8)[rest], old.reshape(-1, kv_heads, dim).view(torch.uint8)[rest])


def test_values_without_a_number():
    """Infinities and NaN go where they belong; e4m3 keeps NaN and holds infinities at its largest value."""
    qkv = torch.zeros(2, 3 * 64, dtype=torch.bfloat16, device="cuda")
    qkv[0, 64], qkv[0, 128], qkv[1, 129], qkv[1, 130] = float("nan"), float("inf"), float("-inf"), float("nan")
    slots, positions = torch.tensor([3, 1], device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for dtype in (torch.bfloat16, E4M3):
        k, v = (torch.zeros(1, 4, 1, 64, device="cuda").to(dtype) for _ in range(2))
        sc = dict(k_scale=torch.ones(1, device="cuda"), v_scale=torch.ones(1, device="cuda")) if dtype == E4M3 else {}
        P.paged_append(qkv.clone(), k, v, slots, positions, 1, 1e4, **sc)
        kf, vf, top = k.float()[0, :, 0], v.float()[0, :, 0], 448.0 if dtype == E4M3 else float("inf")
        assert kf[3, 0].isnan() and kf[3, 32].isnan() and not kf[3, 1:32].isnan().any() and not kf[:3].isnan().any()
        assert vf[3, 0] == top and vf[1, 1] == -top and vf[1, 2].isnan()


def test_no_tokens():
    k = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    P.paged_append(torch.zeros(0, 192, dtype=torch.bfloat16, device="cuda"), k, k.clone(), torch.zeros(0, dtype=torch.int64, device="cuda"),
                   torch.zeros(0, dtype=torch.int32, device="cuda"), 1, 1e4)


def test_far_places():
    """A pool whose rows lie past 32 bits of elements."""
    pages, page, heads, dim = 2 ** 18 + 2, 16, 8, 128  # 2 ** 32 values and two pages
    if torch.cuda.mem_get_info()[0] < 22 << 30:
        pytest.skip("needs 22 GB")
    k, v = (torch.zeros(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    qkv = torch.randn(3, (8 + 16) * dim, device="cuda").bfloat16()
    slots = torch.tensor([pages * page - 1, 5, (pages - 2) * page], device="cuda")
    P.paged_append(qkv, k, v, slots, torch.zeros(3, dtype=torch.int32, device="cuda"), 8, 1e4)
    want = qkv.view(3, 24, dim)
    for i, s in enumerate(slots.tolist()):  # (position 0: nothing is turned)
        assert torch.equal(k.view(-1, heads, dim)[s], want[i, 8:16]) and torch.equal(v.view(-1, heads, dim)[s], want[i, 16:])
    q = qkv.view(3, 24, dim)[:, :8]
    table = torch.tensor([[pages - 1], [0], [pages - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([16, 6, 1], dtype=torch.int32, device="cuda")
    out = P.paged_attention(q, k, v, table, lengths)
    assert torch.equal(out[2], want[2, 16:])  # a single position: its value
    for b, (n, pg) in enumerate(((16, pages - 1), (6, 0))):
        s = torch.einsum("hd,thd->ht", q[b].double(), k[pg, :n].double()) / dim ** 0.5
        o = torch.einsum("ht,thd->hd", s.softmax(-1), v[pg, :n].double())
        # one value in a row of zeros: its weight and the output are rounded
        assert ((out[b].double() - o).abs() <= 2.0 ** -7 * o.abs() + 1e-6).all()
