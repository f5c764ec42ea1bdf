"""The operators of a paged KV cache, as cases that a timing harness can call.

A server keeps the keys and values of all its sequences in one pool of pages and a table that says which pages a sequence
has.  Three calls of `penny_b200.ops` carry that:

  page_tables      tokens come and leave: pages are taken from and returned to the pool on the GPU, every new token
                   gets its position and its slot (page * page_size + offset)
  paged_append     rotary positions of the new tokens' q and k, their k and v into the pages at their slots
  paged_attention  one new token per sequence over its pages

Head layouts are those of this repository's decode configuration on one rank and on eight (32 query and 8 KV heads, 4 and
1), of its small test model (8 and 2) and a few between; batch and context those of its decode benchmark and around.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
THETA = 500000.0
MOST = 64 * 16000 * 8 * 128   # values of K (and of V) that the largest attention case reads
SPARE = 5                     # pages of a pool that no sequence has


def listed():
    return [
        # one user, a short chat, the heads of one of eight ranks: all latency
        dict(name="attend 1 x 200, 4 of 1 heads", op="attend", batch=1, longest=200, kind="even", heads=4, kv_heads=1, dim=128, page=16,
             cache="bf16", by_head=False, window=0),
        # the decode benchmark's batch and context
        dict(name="attend 64 x 2048", op="attend", batch=64, longest=2048, kind="even", heads=32, kv_heads=8, dim=128, page=16,
             cache="bf16", by_head=False, window=0),
        # continuous batching padded to a captured batch: rows of mixed lengths, some without a sequence, a sliding window,
        # pages that are no power of two
        dict(name="attend 130 x 4096 padded, window 1000", op="attend", batch=130, longest=4096, kind="padded", heads=20, kv_heads=20,
             dim=64, page=24, cache="fp16", by_head=True, window=1000),
        # a busy server with an 8-bit cache
        dict(name="attend 96 x 8192 mixed, e4m3", op="attend", batch=96, longest=8192, kind="mixed", heads=32, kv_heads=8, dim=128, page=32,
             cache="e4m3", by_head=False, window=0),
        # two long documents: few rows, so each is read by many SMs
        dict(name="attend 2 x 100001", op="attend", batch=2, longest=100001, kind="even", heads=32, kv_heads=8, dim=128, page=64,
             cache="bf16", by_head=True, window=0),
        # a full pool
        dict(name="attend 64 x 16000", op="attend", batch=64, longest=16000, kind="even", heads=32, kv_heads=8, dim=128, page=16,
             cache="bf16", by_head=False, window=0),
        # a decode step's new tokens, eight of them padding
        dict(name="append 64 decode", op="append", tokens=64, requests=64, padding=8, heads=32, kv_heads=8, dim=128, page=16, types="bf16",
             cache="bf16", far=2048),
        # prompts of odd lengths into an 8-bit cache, far positions
        dict(name="append 2047, e4m3", op="append", tokens=2047, requests=3, padding=0, heads=20, kv_heads=20, dim=64, page=24, types="fp16",
             cache="e4m3", far=100000),
        # a prefill batch
        dict(name="append 16384", op="append", tokens=16384, requests=4, padding=0, heads=32, kv_heads=8, dim=128, page=16, types="bf16",
             cache="bf16", far=8),
        # the step of the decode benchmark: every sequence one token further
        dict(name="tables 64 decode", op="tables", rows=64, prompts=0, longest=2048, chunk=1, page=16),
        # a step of a busy server: most rows decode, a few take a chunk of their prompt
        dict(name="tables 1000, 7 prompts", op="tables", rows=1000, prompts=7, longest=4096, chunk=2048, page=16),
        # admission of many prompts at once
        dict(name="tables 4000, 500 prompts", op="tables", rows=4000, prompts=500, longest=2048, chunk=500, page=8),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return lo if hi <= lo else max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "tables"])
    page = rng.choice([1, 5, 16, 24, 32, 64, 128])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (4, 1, 128), (8, 2, 128), (20, 20, 64), (35, 7, 64), (15, 5, 128), (28, 2, 128), (32, 2, 64),
                                       (8, 1, 256)])
    if op == "attend":
        batch = _spread(rng, 1, 256)
        return dict(op=op, batch=batch, longest=_spread(rng, 1, min(100000, MOST // (batch * kv_heads * dim))),
                    kind=rng.choice(["even", "mixed", "padded"]), heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    cache=rng.choice(["bf16", "fp16", "e4m3"]), by_head=rng.random() < 0.5, window=rng.choice([0, 0, 0, _spread(rng, 1, 5000)]))
    if op == "append":
        types = rng.choice(["bf16", "fp16"])
        tokens = _spread(rng, 1, 16384 * 48 * 128 // ((heads + 2 * kv_heads) * dim))
        return dict(op=op, tokens=tokens, requests=_spread(rng, 1, tokens), padding=rng.choice([0, 0, _spread(rng, 1, 100)]), heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, types=types, cache=rng.choice([types, "e4m3"]), far=_spread(rng, 1, 130000))
    rows = _spread(rng, 1, 4000)
    prompts = rng.randint(0, min(rows, 500))
    return dict(op=op, rows=rows, prompts=prompts, longest=_spread(rng, 1, 8192), page=max(page, 8),
                chunk=_spread(rng, 1, min(16384, 125000 // prompts)) if prompts else 1)


def _lengths(case):
    """Lengths of an attention case's sequences, in an order that a seed changes."""
    if case["kind"] == "even":
        return [case["longest"]] * case["batch"]
    rng = random.Random(case["batch"] * 1000003 + case["longest"])
    got = [case["longest"]] + [_spread(rng, 1, case["longest"]) for _ in range(case["batch"] - 1)]
    if case["kind"] == "padded":
        got[case["batch"] - case["batch"] // 4:] = [0] * (case["batch"] // 4)
    return got


def _news(case):
    """(length, new tokens) of the rows of a tables case, in an order that a seed changes: prompts are at the start or within, the
    others decode; one row in 16 is empty and stays so."""
    rng = random.Random(case["rows"] * 1000003 + case["longest"] + case["chunk"])
    got = [(rng.choice([0, _spread(rng, 1, case["longest"])]), _spread(rng, 1, case["chunk"])) for _ in range(case["prompts"])]
    return got + [(0, 0) if i % 16 == 15 else (_spread(rng, 1, case["longest"]), 1) for i in range(case["rows"] - case["prompts"])]


def _pages(n, page):
    return -(-n // page)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s, dtype=torch.bfloat16: torch.randn(*s, device="cuda", generator=g, dtype=dtype)  # noqa: E731
    mix = random.Random(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    op, page = case["op"], case["page"]

    def owned(lengths, width, pages):
        """A table of `width` pages a row with as many in use as the lengths need, from a shuffled pool; the rest of the pool."""
        held = (ints(lengths) + page - 1) // page
        use = torch.arange(width, device="cuda")[None] < held[:, None]
        pool = torch.randperm(pages, device="cuda", generator=g).int()
        table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
        total = sum(_pages(n, page) for n in lengths)
        table[use] = pool[:total]
        return table, pool[total:]

    def pool_of(pages, kv_heads, dim, kind, by_head=False):
        shape = (pages, kv_heads, page, dim) if by_head else (pages, page, kv_heads, dim)
        if kind == "e4m3":  # (values of size one, stored as multiples of the head's scale)
            data = (normal(*shape) * 100).clamp_(-448, 448).to(TYPES[kind])
        else:
            data = normal(*shape, dtype=TYPES[kind])
        return data.transpose(1, 2) if by_head else data

    if op == "tables":
        rows = _news(case)
        mix.shuffle(rows)
        lengths, new = [r[0] for r in rows], [r[1] for r in rows]
        width = _pages(case["longest"] + case["chunk"], page) + 1
        tokens = -(-sum(new) // 64) * 64  # (a captured step's fixed number)
        need = sum(_pages(a + b, page) for a, b in rows) + SPARE
        table, rest = owned(lengths, width, need)
        free = torch.full((need,), -1, dtype=torch.int32, device="cuda")
        free[:rest.numel()] = rest
        return dict(op=op, page=page, tokens=tokens, table=table, lengths=ints(lengths), free=free, count=ints([rest.numel()]), new=ints(new),
                    back=-ints(new))
    heads, kv_heads, dim, cache = case["heads"], case["kv_heads"], case["dim"], case["cache"]
    scales = [0.008 + 0.004 * torch.rand(kv_heads, device="cuda", generator=g) if cache == "e4m3" else None for _ in range(2)]
    if op == "attend":
        lengths = _lengths(case)
        mix.shuffle(lengths)
        pages = sum(_pages(n, page) for n in lengths) + SPARE
        table, _ = owned(lengths, _pages(case["longest"], page) + 1, pages)
        dtype = torch.float16 if cache == "fp16" else torch.bfloat16
        qkv = normal(case["batch"], (heads + 2 * kv_heads) * dim, dtype=dtype) * 2  # the step's projection, rotated by now
        return dict(op=op, q=qkv[:, :heads * dim].unflatten(1, (heads, dim)), k=pool_of(pages, kv_heads, dim, cache, case["by_head"]),
                    v=pool_of(pages, kv_heads, dim, cache, case["by_head"]), table=table, lengths=ints(lengths), longest=case["longest"],
                    window=case["window"], k_scale=scales[0], v_scale=scales[1],
                    lse=torch.empty(case["batch"], heads, dtype=torch.float32, device="cuda"))
    tokens, requests = case["tokens"], case["requests"]
    each = _pages(tokens, requests)
    at = torch.arange(tokens, device="cuda")
    pages = (tokens if each == 1 else _pages(tokens, page)) + SPARE
    pool = torch.randperm(pages, device="cuda", generator=g)
    start = torch.randint(0, case["far"], (requests,), device="cuda", generator=g)
    offset = torch.randint(0, page, (tokens,), device="cuda", generator=g)
    slots = pool[at] * page + offset if each == 1 else pool[at // page] * page + at % page
    positions = (start[at // each] + at % each).int()
    pad = case["padding"]
    dtype = TYPES[case["types"]]
    return dict(op=op, heads=heads, tokens=tokens, qkv=normal(tokens + pad, (heads + 2 * kv_heads) * dim, dtype=dtype),
                out=torch.zeros(tokens + pad, (heads + kv_heads) * dim, dtype=dtype, device="cuda"),
                k=pool_of(pages, kv_heads, dim, cache), v=pool_of(pages, kv_heads, dim, cache),
                slots=torch.cat([slots, slots.new_full((pad,), -1)]), positions=torch.cat([positions, positions.new_zeros(pad)]),
                k_scale=scales[0], v_scale=scales[1])


def _tables(table, lengths, free, count, new, page, tokens):
    """page_tables in plain operations.  Scatters add the difference to what is there, so that what is masked out adds zero."""
    width, pool = table.shape[1], free.numel()
    old, want = lengths.long(), new.long()
    held = (old + page - 1) // page
    come, leave = want.clamp(min=0), (-want).clamp(min=0)
    offsets = torch.cat([come.new_zeros(1), come.cumsum(0)])
    # pages of the tokens that leave: rows and pages in descending order onto the stack
    shorter = (old - leave).clamp(min=0)
    gone = held - (shorter + page - 1) // page
    gone_to = gone.cumsum(0)
    pushed = gone_to[-1]
    e = torch.arange(pool, device=table.device)
    first = pushed - 1 - e  # this one's number among the released pages, rows and pages ascending
    row = torch.searchsorted(gone_to, first.clamp(min=0), right=True).clamp(max=old.numel() - 1)
    at = held[row] - gone[row] + first - (gone_to[row] - gone[row])
    released = torch.where(first >= 0, table[row, at.clamp(0, width - 1)], 0)
    to = (count + e).clamp(max=pool - 1)
    free.index_add_(0, to, torch.where(first >= 0, released - free[to], 0).int())
    # pages of the tokens that come: from the top of the stack, rows and pages ascending
    fits = (old + come <= width * page) & (offsets[1:] <= tokens)
    need = torch.where(fits, (old + come + page - 1) // page - held, 0)
    taken_to = need.cumsum(0)
    granted = (want <= 0) | (fits & ((need == 0) | (taken_to <= count + pushed)))
    need = torch.where(granted, need, 0)
    j = torch.arange(tokens, device=table.device)
    row = torch.searchsorted(offsets, j, right=True).sub(1).clamp(max=old.numel() - 1)
    real = (j < offsets[-1]) & granted[row]
    pos = torch.where(real, old[row] + j - offsets[row], 0)
    nth = pos // page - held[row]  # of the row's new pages; negative: a page that it had
    popped = free[(count + pushed - 1 - (taken_to[row] - need[row] + nth)).clamp(0, pool - 1)]
    mine = table[row, (pos // page).clamp(max=width - 1)]
    fresh = real & (nth >= 0)
    begins = fresh & ((pos % page == 0))
    table.view(-1).index_add_(0, row * width + (pos // page).clamp(max=width - 1), torch.where(begins, popped - mine, 0).int())
    slots = torch.where(real, torch.where(fresh, popped, mine).long() * page + pos % page, -1)
    count.add_((pushed - need.sum()).int())
    lengths.copy_(torch.where(want > 0, torch.where(granted, old + come, old), shorter))
    return slots, pos.int(), offsets.int(), granted


def _append(s):
    qkv, k, v, heads, n = s["qkv"], s["k"], s["v"], s["heads"], s["tokens"]
    kv_heads, dim = k.shape[2:]
    half = dim // 2
    x = qkv[:n].float().view(n, heads + 2 * kv_heads, 2, half)
    freq = THETA ** (-torch.arange(half, device=qkv.device, dtype=torch.float64) / half)
    angle = s["positions"][:n].double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[:, :heads + kv_heads].unbind(2)
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    s["out"][:n] = turned.flatten(1).to(qkv.dtype)
    slots = s["slots"][:n]
    for pool, new, scale in ((k, turned[:, heads:], s["k_scale"]), (v, x[:, heads + kv_heads:].flatten(2), s["v_scale"])):
        if scale is not None:
            new = (new / scale[:, None]).clamp(-448, 448)
        pool.view(-1, kv_heads, dim).view(torch.uint8)[slots] = new.to(pool.dtype).contiguous().view(torch.uint8)
    return s["out"], k, v


def _rows(pool, pages, within):
    """pool[pages, within], for types that cannot be indexed too."""
    return pool.view(torch.uint8)[pages, within].view(pool.dtype) if pool.dtype == TYPES["e4m3"] else pool[pages, within]


def _attend(s):
    q, k, v, lengths = s["q"], s["k"], s["v"], s["lengths"]
    batch, heads, dim = q.shape
    page, kv_heads = k.shape[1:3]
    at = torch.arange(s["longest"], device=q.device)
    pages = s["table"][:, at // page].clamp(min=0)
    there = at[None] < lengths[:, None]
    if s["window"]:
        there = there & (at[None] >= lengths[:, None] - s["window"])
    there = there[:, None, None]
    qs = q.float().view(batch, kv_heads, heads // kv_heads, dim) / math.sqrt(dim)
    if s["k_scale"] is not None:
        qs = qs * s["k_scale"][:, None, None]
    scores = qs @ _rows(k, pages, at % page).float().permute(0, 2, 3, 1)
    scores = scores.masked_fill(~there, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == -math.inf, 0)).exp()
    total = p.sum(-1, keepdim=True)
    o = p @ _rows(v, pages, at % page).float().transpose(1, 2) / total.masked_fill(total == 0, 1)
    if s["v_scale"] is not None:
        o = o * s["v_scale"][:, None, None]
    return o.reshape(q.shape).to(q.dtype), (top + total.log()).reshape(batch, heads)


def run(s):
    if own:
        import penny_b200.ops as ops
    if s["op"] == "tables":
        f = ops.page_tables if own else _tables
        state = s["table"], s["lengths"], s["free"], s["count"]
        said = f(*state, s["new"], s["page"], s["tokens"])
        f(*state, s["back"], s["page"], 0)  # the tokens leave again: the state is as before
        return *said, *state
    if s["op"] == "append":
        if own:
            ops.paged_append(s["qkv"], s["k"], s["v"], s["slots"], s["positions"], s["heads"], THETA, out=s["out"], k_scale=s["k_scale"],
                             v_scale=s["v_scale"])
            return s["out"], s["k"], s["v"]
        return _append(s)
    if own:
        out = ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=s["window"], k_scale=s["k_scale"],
                                  v_scale=s["v_scale"], lse=s["lse"])
        return out, s["lse"]
    return _attend(s)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "tables":
        return None
    k, v = s["k"], s["v"]
    kv_heads, dim = k.shape[2:]
    if s["op"] == "append":
        heads, n = s["heads"], s["tokens"]
        z = s["qkv"].double().view(-1, heads + 2 * kv_heads, dim)[:n]
        c = torch.complex(z[..., :dim // 2], z[..., dim // 2:])[:, :heads + kv_heads]
        freq = torch.exp(torch.arange(dim // 2, device="cuda", dtype=torch.float64) * (-2 * math.log(THETA) / dim))
        c = c * torch.polar(torch.ones_like(freq), s["positions"][:n, None].double() * freq)[:, None]
        turned = torch.cat([c.real, c.imag], -1)
        out = s["out"].double()
        out[:n] = turned.flatten(1)
        got = []
        for pool, new, scale in ((k, turned[:, heads:], s["k_scale"]), (v, z[:, heads + kv_heads:], s["v_scale"])):
            pool = pool.double().flatten(0, 1)
            pool[s["slots"][:n]] = new if scale is None else (new / scale.double()[:, None]).clamp(-448, 448)
            got.append(pool.view(k.shape))
        return out, *got
    q = s["q"].double()
    batch, heads, _ = q.shape
    out, lse = torch.zeros_like(q), torch.full((batch, heads), -math.inf, dtype=torch.float64, device="cuda")
    page = k.shape[1]
    for b, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - s["window"]) if s["window"] else 0
        if n == 0:
            continue
        at = torch.arange(lo, n, device="cuda")
        rows = [_rows(pool, s["table"][b, at // page], at % page).double() for pool in (k, v)]
        rows = [r if sc is None else r * sc.double()[:, None] for r, sc in zip(rows, (s["k_scale"], s["v_scale"]))]
        keys, values = (r.repeat_interleave(heads // kv_heads, 1) for r in rows)
        logits = torch.einsum("hd,thd->ht", q[b], keys) / dim ** 0.5
        lse[b] = logits.logsumexp(-1)
        out[b] = torch.einsum("ht,thd->hd", (logits - lse[b][:, None]).exp(), values)
    return out, lse


def work(case):
    if case["op"] == "tables":
        rows = _news(case)
        tokens, fresh = sum(n for _, n in rows), sum(_pages(a + b, case["page"]) - _pages(a, case["page"]) for a, b in rows)
        # both ways: lengths and new tokens read, lengths, offsets and grants written, a page id from one place to another
        return {"bytes": 2 * (len(rows) * 17 + fresh * 8) + tokens * 12, "flops": 0}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "append":
        turned = (heads + kv_heads) * dim
        return {"bytes": case["tokens"] * (12 + 2 * (2 * turned + kv_heads * dim) + 2 * size * kv_heads * dim), "flops": case["tokens"] * turned * 3}
    seen = [min(n, case["window"] or n) for n in _lengths(case)]
    ids = sum(_pages(n, case["page"]) for n in seen)
    return {"bytes": sum(seen) * kv_heads * dim * 2 * size + case["batch"] * (heads * (dim * 4 + 4) + 4) + ids * 4,
            "flops": 4 * sum(seen) * heads * dim}
