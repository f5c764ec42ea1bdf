"""Attention of one new token per sequence over pages, against fp64."""
import math

import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu
BF, HF, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
STEP = {BF: 2.0 ** -8, HF: 2.0 ** -11}  # half a step of a value's own size


def _case(lengths, heads, kv_heads, dim, page, dtype, cache, by_head=False, seed=0, stale=float("nan")):
    """A pool in which everything that no row has, and every position behind a row's end, is `stale`."""
    g = torch.Generator(device="cuda").manual_seed(seed + dim + page)
    B, width = len(lengths), max(1, -(-max(lengths + [1]) // page)) + 1
    held = [-(-max(0, n) // page) for n in lengths]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.full((B, width), -1, dtype=torch.int32), 0
    shape = (pages, kv_heads, page, dim) if by_head else (pages, page, kv_heads, dim)
    pools = [torch.randn(*shape, device="cuda", generator=g) * (60 if cache == E4M3 else 1) for _ in range(2)]
    pools = [p.transpose(1, 2) if by_head else p for p in pools]
    live = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
        for i in range(held[b]):
            live[table[b, i], :min(page, n - i * page)] = True
    pools = [p.masked_fill_(~live.cuda()[:, :, None, None], stale).to(cache) for p in pools]
    q = (torch.randn(B, heads + 2, dim, device="cuda", generator=g) * 2).to(dtype)[:, 1:heads + 1]
    scales = {s: 0.01 + 0.01 * torch.rand(kv_heads, device="cuda", generator=g) for s in ("k_scale", "v_scale")} if cache == E4M3 else {}
    return dict(q=q, k=pools[0], v=pools[1], table=table.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), **scales)


def _check(c, out, lse, window=0, scale=None, rows=None):
    """A weight is off by half a step of the type that meets V (bf16, else fp16: 2 ** -25 at least) and by what fp32 makes of its
    score: dim products and sums, 2 ** -23 of the products' sizes each; the output by half a step more."""
    q, k, v = c["q"], c["k"], c["v"]
    dim, G, page = q.shape[2], q.shape[1] // k.shape[2], k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    for b in range(q.shape[0]) if rows is None else rows:
        n = max(0, int(c["lengths"][b]))
        at = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
        ids = c["table"][b, at // page]
        at, ids = at[(ids >= 0) & (ids < k.shape[0])], ids[(ids >= 0) & (ids < k.shape[0])]
        if at.numel() == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all(), b
            continue
        keys, vals = (p.view(torch.uint8)[ids, at % page].view(E4M3).double() if p.dtype == E4M3 else p[ids, at % page].double() for p in (k, v))
        if k.dtype == E4M3:
            keys, vals = keys * c["k_scale"].double()[:, None], vals * c["v_scale"].double()[:, None]
        keys, vals = keys.repeat_interleave(G, 1), vals.repeat_interleave(G, 1)
        s = torch.einsum("hd,thd->ht", q[b].double(), keys) * scale
        off = dim * 2.0 ** -23 * abs(scale) * torch.einsum("hd,thd->ht", q[b].double().abs(), keys.abs()).amax(-1, keepdim=True) + 2.0 ** -20
        p = s.softmax(-1)
        want, size = torch.einsum("ht,thd->hd", p, vals), torch.einsum("ht,thd->hd", p, vals.abs())
        bf = k.dtype == BF
        step = STEP[BF] if bf else STEP[HF]
        floor = 0 if bf else at.numel() * 2.0 ** -25 * vals.abs().amax()
        bound = (step + 2 * off) * size * (1 + 2.0 ** -6) + STEP[q.dtype] * want.abs() * (1 + 2.0 ** -6) + floor + (2.0 ** -25 if q.dtype == HF else 0)
        err = (out[b].double() - want).abs()
        assert (err <= bound).all(), (b, n, float((err - bound).max()), float(err.max()))
        true = s.logsumexp(-1)
        assert ((lse[b].double() - true).abs() <= off[:, 0] + 2.0 ** -22 * true.abs()).all(), (b, n)


def _workspace_bytes(*a):
    from penny_b200._ext import ops
    return ops.paged_attention_workspace_bytes(*a)


def _run(c, **kw):
    lse = torch.full(c["q"].shape[:2], 5.0, device="cuda")
    out = P.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lengths"], lse=lse, **{s: c[s] for s in ("k_scale", "v_scale") if s in c}, **kw)
    return out, lse


TYPES = [(BF, BF), (HF, HF), (BF, E4M3), (HF, E4M3)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,page", [(4, 1, 16), (20, 20, 24), (15, 5, 1), (28, 2, 5), (32, 2, 64), (34, 2, 128), (8, 1, 7)])
def test_lengths(dtype, cache, dim, heads, kv_heads, page):
    """Rows of no positions, of one, at the ends of pages, tiles and pieces, in one batch with long ones; stale NaN everywhere else."""
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, page, page + 1, 255, 511, 513, 0, 1300]
    for by_head in (False, True):
        c = _case(lengths, heads, kv_heads, dim, page, dtype, cache, by_head)
        _check(c, *_run(c))


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, E4M3)])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([20000], 4, 1), ([4111, 9], 8, 2), ([70001], 2, 1), ([255, 256, 511, 512, 0, 2600], 16, 1),
                                                    ([1, 7000] + [40] * 130, 8, 2), ([600] * 300, 8, 8), ([0, 0], 4, 2), ([7, 0, 30] * 1500, 2, 1)])
def test_pieces(dtype, cache, lengths, heads, kv_heads):
    """Rows that are cut into many pieces, one long row among short ones, more rows than a block has threads, whole rows."""
    c = _case(lengths, heads, kv_heads, 128, 16, dtype, cache, seed=1)
    out, lse = _run(c)
    _check(c, out, lse, rows=range(min(8, len(lengths))))
    ws = torch.full((_workspace_bytes(len(lengths), heads, kv_heads, 128, c["table"].shape[1] * 16),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):  # a workspace's contents mean nothing
        again, lse2 = _run(c, workspace=ws)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    if ws.numel():
        with pytest.raises(RuntimeError, match="workspace too small"):
            _run(c, workspace=ws[:-16])


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, E4M3)])
@pytest.mark.parametrize("heads,kv_heads,dim,window", [(4, 1, 128, 0), (3, 1, 64, 5000), (34, 2, 64, 0), (8, 1, 256, 0), (32, 2, 256, 700)])
@pytest.mark.parametrize("lengths", [[0, 30011], [1, 9000, 0, 20, 5001, 0, 0], [7001, 0, 1, 16] * 5, [2000, 1, 0] * 16 + [4999], [800, 0] * 60])
def test_join(dtype, cache, heads, kv_heads, dim, window, lengths):
    """Rows in hundreds of parts, in a few and in one, empty rows among them: every way in which the joining kernel shares them out."""
    c = _case(lengths, heads, kv_heads, dim, 16, dtype, cache, seed=9)
    out, lse = _run(c, window=window)
    _check(c, out, lse, window=window, rows=range(min(8, len(lengths))))
    _check(c, out, lse, window=window, rows=range(max(0, len(lengths) - 8), len(lengths)))


@pytest.mark.parametrize("window", [1, 16, 17, 300, 100000])
@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, HF), (BF, E4M3)])
def test_window(window, dtype, cache):
    c = _case([0, 1, 16, 17, 33, 301, 900, 3000], 8, 2, 64, 24, dtype, cache, seed=2)
    for b, n in enumerate(c["lengths"].tolist()):  # what lies before the window is as stale as what lies behind the end
        gone = c["table"][b, :max(0, n - window) // 24].long()
        c["k"].view(torch.uint8)[gone] = 0x7f
        c["v"].view(torch.uint8)[gone] = 0x7f
    _check(c, *_run(c, window=window), window=window)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scale(scale):
    c = _case([40, 700], 8, 2, 128, 16, BF, BF, seed=3)
    _check(c, *_run(c, scale=scale), scale=scale)


def test_lengths_and_pages_that_the_pool_does_not_have():
    """Lengths below zero and past the table, pages outside the pool in the middle of a row, all over it, a table that repeats a page."""
    c = _case([100, 200, 300, 400, 50], 8, 2, 128, 16, BF, BF, seed=4)
    c["table"][1, 3], c["table"][1, 11] = -1, 2 ** 31 - 1
    c["table"][2, :] = c["k"].shape[0]
    c["table"][3, 5:8] = c["table"][0, 0]
    c["lengths"][4] = -7
    _check(c, *_run(c))
    c = _case([64, 64], 4, 1, 64, 16, HF, HF, seed=5)
    c["table"] = c["table"][:, :4].contiguous()
    c["lengths"] += 2 ** 31 - 65
    out, lse = _run(c)
    c["lengths"].fill_(64)
    _check(c, out, lse)


def test_values_without_a_number():
    """NaN and infinities among a row's own positions give what softmax gives; other rows do not see them."""
    for cache in (BF, E4M3):
        c = _case([50, 50, 600, 50], 8, 2, 64, 16, BF, cache, seed=6, stale=0.0)
        nan = torch.full((64,), float("nan"), device="cuda").to(cache)
        t = c["table"]
        c["k"][t[0, 1], 3, 0] = nan            # a score of NaN: the KV head's rows are NaN
        c["v"][t[1, 2], 5, 1] = nan            # a value of NaN
        c["v"][t[2, 30], 5, 1] = nan           # in a row that may be cut
        out, lse = _run(c)
        assert out[0, :4].isnan().all() and lse[0, :4].isnan().all() and out[1, 4:].isnan().all() and out[2, 4:].isnan().all()
        _check(c, out, lse, rows=[3])
        assert not out[0, 4:].isnan().any() and not out[1, :4].isnan().any() and not lse[1].isnan().any()
    c["q"][3] = 0  # e4m3: a row of zeros has no largest value
    out, lse = _run(c)
    _check(c, out, lse, rows=[3])
    big = _case([50], 4, 1, 64, 16, BF, E4M3, seed=7)
    big["q"] *= 1e30  # past fp16 by far
    out, _ = _run(big, scale=1e-31)
    _check(big, out, _run(big, scale=1e-31)[1], scale=1e-31)
    big["q"][0, 2, 5] = 3e38  # the largest power of two there is
    _check(big, *_run(big, scale=1e-41), scale=1e-41)
    big["q"][0, 2, 5] = 1e30
    big["q"][0, 1] *= 1e-36
    _check(big, *_run(big, scale=1e-31), scale=1e-31)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_views_in_place_and_padded(dtype, cache):
    """q and out as parts of other tensors, out in place of q, nothing written beside it, tables wider than they need be."""
    c = _case([70, 0, 900], 8, 2, 128, 16, dtype, cache, seed=8)
    out, lse = _run(c)
    wide = torch.full((3, 11, 136), 3.0, dtype=dtype, device="cuda")
    _run(c, out=wide[:, 2:10, :128])
    assert torch.equal(wide[:, 2:10, :128], out) and (wide[:, :2] == 3).all() and (wide[:, 10:] == 3).all() and (wide[..., 128:] == 3).all()
    table = torch.full((3, 4000), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, :c["table"].shape[1]] = c["table"]
    far, lse2 = _run(dict(c, table=table[:, :3000]))
    torch.testing.assert_close(far.float(), out.float(), atol=2 * STEP[dtype], rtol=4 * STEP[dtype])
    _check(dict(c, table=table), far, lse2)
    q = c["q"].contiguous()
    c["q"] = q
    assert _run(c, out=q)[0].data_ptr() == q.data_ptr() and torch.equal(q, out)


def test_in_place_of_transposed_heads():
    """out with the heads outside the rows."""
    c = _case([70, 0, 900], 8, 2, 64, 16, BF, BF, seed=11)
    out, lse = _run(c)
    turned = torch.full((8, 3, 64), 3.0, dtype=BF, device="cuda").transpose(0, 1)
    _run(c, out=turned)
    assert torch.equal(turned, out)


def test_strides_of_single_rows_heads_and_pages():
    """What the strides of a dimension of one say does not count: of one row, one head, one KV head, one page, pages of one position."""
    odd = lambda t, dims: t.as_strided(t.shape, [3 if i in dims else s for i, s in enumerate(t.stride())])  # noqa: E731
    c = _case([300], 1, 1, 64, 16, BF, BF, seed=14)
    out, lse = _run(c)
    d = dict(c, q=odd(c["q"].contiguous(), (0, 1)), k=odd(c["k"], (2,)))
    got, lse2 = _run(d)
    assert torch.equal(got, out) and torch.equal(lse, lse2)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    one = dict(q=c["q"], k=odd(c["k"][:1], (0, 2)), v=c["v"][:1].nan_to_num(), table=table, lengths=torch.tensor([1], dtype=torch.int32, device="cuda"))
    one["k"] = one["k"].nan_to_num()
    _check(one, *_run(one))
    c = _case([40, 7], 4, 2, 128, 1, HF, E4M3, seed=15)
    d = dict(c, k=odd(c["k"], (1,)))
    out, lse = _run(c)
    assert torch.equal(_run(d)[0], out)
    _check(c, out, lse)


def test_another_order_of_the_same_rows():
    """Rows in another order, or alone, give what they gave but for where they are cut."""
    lengths = [900, 1, 0, 333, 5000, 64]
    c = _case(lengths, 16, 2, 128, 32, BF, E4M3, seed=12)
    out, lse = _run(c)
    order = torch.tensor([4, 2, 0, 5, 1, 3], device="cuda")
    moved = dict(c, q=c["q"][order], table=c["table"][order], lengths=c["lengths"][order])
    _check(moved, *_run(moved))
    for b in range(6):
        alone = dict(c, q=c["q"][b:b + 1], table=c["table"][b:b + 1], lengths=c["lengths"][b:b + 1])
        _check(alone, *_run(alone))


def test_early():
    """With early set, keys and values of the last positions come from the kernel in front, at every place of a tile."""
    heads, kv_heads, dim, page = 8, 2, 128, 16
    for dtype in (BF, HF):
        c = _case([1, 15, 16, 17, 400, 1000], heads, kv_heads, dim, page, dtype, dtype, seed=13)
        B = 6
        last = c["lengths"] - 1
        slots = c["table"].gather(1, (last // page).long()[:, None])[:, 0].long() * page + last % page
        for rep in range(3):
            qkv = torch.randn(B, (heads + 2 * kv_heads) * dim, device="cuda").to(dtype)
            torch.cuda._sleep(200000)
            P.paged_append(qkv, c["k"], c["v"], slots, last, heads, 1e4, early=rep > 0)
            c["q"] = qkv[:, :heads * dim].unflatten(1, (heads, dim))
            _check(c, *_run(c, early=True))


def test_no_rows():
    c = _case([5], 4, 1, 64, 16, BF, BF)
    out = P.paged_attention(c["q"][:0], c["k"], c["v"], c["table"][:0], c["lengths"][:0])
    assert out.shape == (0, 4, 64)


def test_streams_and_graphs():
    """Two captured calls on two streams at a time, with other lengths at every replay, and the same results every time."""
    cs = [_case([3000, 40, 700], 8, 2, 128, 16, BF, BF, seed=s) for s in (9, 10)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cs]
    for c in cs:
        _run(c)  # (a first launch is not a captured one)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(c))
        graphs.append(g)
    for lengths in ([3000, 40, 700], [1, 0, 256], [2999, 17, 512]):
        for c in cs:
            c["lengths"].copy_(torch.tensor(lengths))
        torch.cuda.synchronize()
        first = None
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            now = [t.clone() for o in outs for t in o]
            assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
            first = now
        for c, o in zip(cs, outs):
            _check(c, *o)
