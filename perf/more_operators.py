"""The operators of several continuations of one prompt, as cases that a timing harness can call.

A server that samples a prompt several times, or whose requests begin with the same text, keeps that text's keys and values once:
the rows of its block table have the same first pages, and every page counts the rows that have it.  The calls of `penny_b200.ops`
for that:

  page_fork, page_copy     empty rows begin as copies of others: whole pages are shared, a page that the row ends inside is copied
                           in all layers' pools; page_tables(refs=) lets rows leave again
  page_compact, page_copy  the pages in use move to the front of the pools
  page_groups              the rows that have the same first pages, from the tables
  paged_attention(groups=) one new token per row; positions that a group's rows share are read once for all of them
  token_logprobs           log probabilities of the tokens that were chosen, with entropy and top alternatives

Head layouts are those of this repository's decode configuration on one rank and on eight (32 query and 8 KV heads, 4 and
1), of its small test model (8 and 2) and a few between; the vocabulary that of the decode configuration.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
MOST = 100 * 16500 * 8 * 128  # values of K that all rows of an attention case see, shared ones counted for every row
POOLS = 640 << 20             # values of all pools of a fork or a compaction
SPARE = 5                     # pages of a pool that no row has


def listed():
    return [
        # one prompt sampled eight times, the heads of one of eight ranks
        dict(name="fork 1 x 8, 1 head", op="fork", prompts=1, each=8, length=200, layers=24, kv_heads=1, dim=128, page=16, cache="bf16"),
        # eight prompts, eight continuations each, the heads of the decode configuration on one rank
        dict(name="fork 8 x 8", op="fork", prompts=8, each=8, length=1000, layers=24, kv_heads=8, dim=128, page=16, cache="bf16"),
        # a small pool of few layers, 8 bits
        dict(name="compact 200 pages, e4m3", op="compact", pages=200, rows=8, full=0.4, layers=2, kv_heads=2, dim=128, page=32, cache="e4m3"),
        # a pool half of which is free again
        dict(name="compact 600 pages", op="compact", pages=600, rows=40, full=0.5, layers=24, kv_heads=8, dim=128, page=16, cache="bf16"),
        # the decode benchmark's batch behind one system prompt, eight rows without it
        dict(name="groups 64, 1 prompt", op="groups", rows=64, groups=1, lone=8, prefix=2048, own=200, page=16),
        # a busy server with many prompts
        dict(name="groups 4000, 500 prompts", op="groups", rows=4000, groups=500, lone=300, prefix=1500, own=300, page=16),
        # one user's four samples of a short chat, the heads of one of eight ranks: all latency
        dict(name="attend 4 x (200 + 20), 4 of 1", op="attend", rows=4, groups=1, lone=0, prefix=200, own=20, kind="even", heads=4, kv_heads=1,
             dim=128, page=16, cache="bf16", window=0),
        # the decode benchmark's batch behind a system prompt of 4000 tokens
        dict(name="attend 64 x (4000 + 300)", op="attend", rows=64, groups=1, lone=0, prefix=4000, own=300, kind="even", heads=32, kv_heads=8,
             dim=128, page=16, cache="bf16", window=0),
        # several documents with a few questions each, rows that share nothing and rows without a sequence; an 8-bit cache
        dict(name="attend 130, 9 prompts, e4m3", op="attend", rows=130, groups=9, lone=20, prefix=8192, own=700, kind="padded", heads=32, kv_heads=8,
             dim=128, page=32, cache="e4m3", window=0),
        # many questions about one long document
        dict(name="attend 100 x (16000 + 500)", op="attend", rows=100, groups=1, lone=0, prefix=16000, own=500, kind="even", heads=32, kv_heads=8,
             dim=128, page=64, cache="bf16", window=0),
        # a decode step's tokens with the alternatives that an API returns
        dict(name="logprobs 64 x 128256, top 20", op="logprobs", rows=64, vocab=128256, top=20, type="bf16", masked=False),
        # the tokens of a given text
        dict(name="logprobs 2047 x 128256", op="logprobs", rows=2047, vocab=128256, top=0, type="bf16", masked=False),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return lo if hi <= lo else max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["fork", "compact", "groups", "attend", "attend", "attend", "logprobs", "logprobs"])
    page = rng.choice([1, 5, 16, 24, 32, 64, 128])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (4, 1, 128), (8, 2, 128), (20, 20, 64), (35, 7, 64), (15, 5, 128), (28, 2, 128), (32, 2, 64),
                                       (8, 1, 256)])
    cache = rng.choice(["bf16", "fp16", "e4m3"])
    if op in ("fork", "compact"):
        page, layers = max(page, 5), _spread(rng, 1, 28)
        most = POOLS // (2 * layers * page * kv_heads * dim)  # pages
        pool = dict(op=op, layers=layers, kv_heads=kv_heads, dim=dim, page=page, cache=cache)
        if op == "compact":
            rows = _spread(rng, 1, max(1, min(100, most // 3)))
            return dict(pool, pages=_spread(rng, 2 * rows + 4, most), rows=rows, full=rng.uniform(0.1, 0.95))
        forks = _spread(rng, 1, max(1, min(12, (most - SPARE) // 4)))
        prompts = _spread(rng, 1, max(1, min(12, (most - SPARE) // (2 * forks + 1))))
        longest = (most - prompts * forks - SPARE) // prompts * page
        return dict(pool, prompts=prompts, each=forks, length=_spread(rng, 1, max(1, min(8000, longest))))
    if op == "logprobs":
        vocab = _spread(rng, 2, 160000)
        return dict(op=op, rows=_spread(rng, 1, min(8000, 2000 * 128256 // vocab)), vocab=vocab, top=min(vocab, rng.choice([0, 1, 5, 20, 32])),
                    type=rng.choice(["bf16", "fp16", "fp32"]), masked=rng.random() < 0.3)
    rows = _spread(rng, 2, 4000 if op == "groups" else 256)
    lone = rng.choice([0, _spread(rng, 1, rows)])
    groups = _spread(rng, 1, max(1, (rows - lone) // 2))
    if op == "groups":
        return dict(op=op, rows=rows, groups=groups, lone=lone, prefix=_spread(rng, 1, 8000), own=_spread(rng, 1, 2000), page=max(page, 5))
    own_most = _spread(rng, 1, min(4000, MOST // (rows * kv_heads * dim) // 2))
    return dict(op=op, rows=rows, groups=groups, lone=lone, prefix=_spread(rng, 1, min(60000, MOST // (rows * kv_heads * dim) - own_most)),
                own=own_most, kind=rng.choice(["even", "mixed", "padded"]), heads=heads, kv_heads=kv_heads, dim=dim, page=page, cache=cache,
                window=rng.choice([0, 0, 0, _spread(rng, 1, 8000)]))


def _pages(n, page):
    return -(-n // page)


def _rows(case):
    """(group or -1, whole pages that its group shares, own positions) of the rows of a groups or an attend case.  Rows are admitted as
    requests come, so those of a group do not lie side by side."""
    rng = random.Random(case["rows"] * 1000003 + case["prefix"] * 101 + case["groups"])
    even = case.get("kind", "mixed") == "even"
    of = [(case["prefix"] if even or g == 0 else _spread(rng, 1, case["prefix"])) // case["page"] for g in range(case["groups"])]
    got = []
    for i in range(case["rows"] - case["lone"]):
        got.append((i % case["groups"], of[i % case["groups"]], case["own"] if even else _spread(rng, 1, case["own"])))
    for i in range(case["lone"]):
        got.append((-1, 0, 0 if case.get("kind") == "padded" and i % 2 else _spread(rng, 1, case["own"])))
    return got


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s, dtype=torch.bfloat16: torch.randn(*s, device="cuda", generator=g, dtype=dtype)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    op = case["op"]
    if op == "logprobs":
        logits = normal(case["rows"], case["vocab"], dtype=TYPES[case["type"]]) * 3
        noise = torch.rand(case["rows"], case["vocab"], device="cuda", generator=g, dtype=torch.float32).clamp_(1e-9, 1 - 1e-7)
        if case["masked"]:  # (a grammar's mask: most tokens must not be chosen)
            logits[:, 1:].masked_fill_(noise[:, :-1] < 0.9, -math.inf)
        tokens = noise.log_().neg_().log_().neg_().add_(logits).argmax(-1)  # sampled
        return dict(op=op, logits=logits, tokens=tokens, top=case["top"])
    page = case["page"]

    def pool_of(pages, kv_heads, dim, kind):
        if kind == "e4m3":  # (values of size one, stored as multiples of the head's scale)
            return (normal(pages, page, kv_heads, dim) * 100).clamp_(-448, 448).to(TYPES[kind])
        return normal(pages, page, kv_heads, dim, dtype=TYPES[kind])

    if op == "fork":
        n, forks, length = case["prompts"], case["prompts"] * case["each"], case["length"]
        held, width = _pages(length, page), _pages(length, page) + 2
        pages = n * held + forks + SPARE
        pool = torch.randperm(pages, device="cuda", generator=g).int()
        table = torch.full((n + forks, width), -1, dtype=torch.int32, device="cuda")
        table[:n, :held] = pool[:n * held].view(n, held)
        lengths = ints([length] * n + [0] * forks)
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:pages - n * held] = pool[n * held:]
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[pool[:n * held].long()] = 1
        return dict(op=op, page=page, state=[table, lengths, free, ints([pages - n * held]), refs], source=ints([i // case["each"] for i in range(forks)]),
                    target=ints(list(range(n, n + forks))), back=ints([0] * n + [-length] * forks),
                    pools=[pool_of(pages, case["kv_heads"], case["dim"], case["cache"]) for _ in range(2 * case["layers"])])
    if op == "compact":
        rng, pages, rows = random.Random(case["pages"] * 1000003 + case["rows"]), case["pages"], case["rows"]
        used = min(max(rows + 1, int(pages * case["full"])), pages - 1)
        cuts = sorted(rng.sample(range(1, used), rows - 1)) if rows > 1 else []
        held = [b - a for a, b in zip([0] + cuts, cuts + [used])]
        random.Random(seed).shuffle(held)
        lengths = [n * page - rng.randrange(page) for n in held]
        pool = torch.randperm(pages, device="cuda", generator=g).int()
        table = torch.full((rows + 1, max(held) + 1), -1, dtype=torch.int32, device="cuda")
        at = 0
        for r, n in enumerate(held):
            table[r, :n] = pool[at:at + n]
            at += n
        table[rows, :held[0]] = table[0, :held[0]]  # a fork that ends with a page
        lengths.append(held[0] * page)
        lengths[0] = held[0] * page
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:pages - used] = pool[used:]
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[pool[:used].long()] = 1
        refs[table[0, :held[0]].long()] = 2
        state = [table, ints(lengths), free, ints([pages - used]), refs]
        return dict(op=op, page=page, state=state, before=[t.clone() for t in state],
                    pools=[pool_of(pages, case["kv_heads"], case["dim"], case["cache"]) for _ in range(2 * case["layers"])])
    rows = _rows(case)
    random.Random(seed).shuffle(rows)
    shared = {}
    for group, pre, _ in rows:
        shared[group] = pre if group >= 0 else 0
    total = sum(shared.values()) + sum(_pages(n, page) for _, _, n in rows) + SPARE
    pool = torch.randperm(total, device="cuda", generator=g).tolist()
    of = {group: [pool.pop() for _ in range(pre)] for group, pre in sorted(shared.items())}
    width = max(len(of[group]) + _pages(n, page) for group, _, n in rows) + 1
    table = [of[group] + [pool.pop() for _ in range(_pages(n, page))] for group, _, n in rows]
    table = ints([ids + [-1] * (width - len(ids)) for ids in table])
    lengths = ints([len(of[group]) * page + n for group, _, n in rows])
    if op == "groups":
        return dict(op=op, page=page, table=table, lengths=lengths)
    heads, kv_heads, dim, cache = case["heads"], case["kv_heads"], case["dim"], case["cache"]
    scales = [0.008 + 0.004 * torch.rand(kv_heads, device="cuda", generator=g) if cache == "e4m3" else None for _ in range(2)]
    qkv = normal(len(rows), (heads + 2 * kv_heads) * dim, dtype=torch.float16 if cache == "fp16" else torch.bfloat16) * 2  # the step's projection
    return dict(op=op, q=qkv[:, :heads * dim].unflatten(1, (heads, dim)), k=pool_of(total, kv_heads, dim, cache), v=pool_of(total, kv_heads, dim, cache),
                table=table, lengths=lengths, longest=max(len(of[group]) * page + n for group, _, n in rows), window=case["window"],
                groups=_groups(table, lengths, page),  # (made once a step, for all layers)
                k_scale=scales[0], v_scale=scales[1], lse=torch.empty(len(rows), heads, dtype=torch.float32, device="cuda"))


def _into(size, at, values, there, fill):
    """A list of `size` with values[i] at at[i] where `there`."""
    got = torch.full((size + 1,), fill, dtype=values.dtype, device=values.device)
    return got.scatter_(0, torch.where(there, at, size), values)[:size]


def _fork(table, lengths, free, count, refs, source, target, page):
    """page_fork in plain operations."""
    pages, width = free.numel(), table.shape[1]
    s, t = source.long(), target.long()
    old = lengths[s].long()
    full, part = old // page, old % page > 0
    ok = (lengths[t] == 0) & (s != t)
    taken = (part & ok).long().cumsum(0)
    granted = ok & (~part | (taken <= count))
    fresh = part & granted
    new = free[(count - taken).clamp(0, pages - 1)]
    last = table[s, full.clamp(max=width - 1)]
    cols = torch.arange(width, device=table.device)
    use = (cols < full[:, None]) & granted[:, None]
    refs += torch.zeros_like(refs).index_add_(0, torch.where(use, table[s], 0).flatten().long(), use.flatten().int())
    refs += torch.zeros_like(refs).index_add_(0, torch.where(fresh, new, 0).long(), fresh.int())
    mine = torch.where(use, table[s], table[t])
    table[t] = torch.where((cols == full[:, None]) & fresh[:, None], new[:, None], mine)
    lengths[t] = torch.where(granted, old, lengths[t].long()).int()
    count -= fresh.sum().int()
    return _into(s.numel(), taken - 1, last, fresh, -1), _into(s.numel(), taken - 1, new, fresh, -1), granted


def _leave(table, lengths, free, count, refs, new, page):
    """page_tables(refs=) in plain operations, for rows that leave."""
    pages, (rows, width) = free.numel(), table.shape
    old = lengths.long()
    shorter = (old + new.clamp(max=0)).clamp(min=0)
    cols = torch.arange(width, device=table.device)
    gone = ((cols >= ((shorter + page - 1) // page)[:, None]) & (cols < ((old + page - 1) // page)[:, None])).flatten()
    ids = torch.where(gone, table.flatten(), pages).long()  # (behind the last page: what counts for none)
    left = torch.zeros(pages + 1, dtype=torch.int32, device=table.device).index_add_(0, ids, gone.int())[:pages]
    refs -= left
    nth = torch.arange(rows * width, device=table.device)
    last = torch.full((pages + 1,), -1, device=table.device).scatter_reduce_(0, ids, nth, "amax")
    back = torch.cat([(refs == 0) & (left > 0), refs.new_zeros(1, dtype=torch.bool)])[ids] & (last[ids] == nth)
    behind = back.flip(0).long().cumsum(0).flip(0) - 1  # pages that go back from the same place on, this one not counted
    free.copy_(torch.where(torch.arange(pages, device=table.device) < count, free, torch.where(
        torch.arange(pages, device=table.device) < count + back.sum(), _into(pages, (count + behind).clamp(0, pages), ids.int(), back, -1), free)))
    count += back.sum().int()
    lengths.copy_(shorter)


def _compact(table, lengths, free, count, refs, page):
    """page_compact in plain operations."""
    pages = free.numel()
    at = torch.arange(pages, device=table.device)
    used = refs > 0
    n = used.sum()
    goes, room = used & (at >= n), ~used & (at < n)
    most = pages // 2
    copy_from, copy_to = (_into(most, (m.long().cumsum(0) - 1).clamp(0, most), at.int(), m, -1) for m in (goes, room))
    to = torch.where(goes, copy_to[(goes.long().cumsum(0) - 1).clamp(0, most - 1)].long(), at)
    mine = torch.arange(table.shape[1], device=table.device) < ((lengths.long() + page - 1) // page)[:, None]
    table.copy_(torch.where(mine, to[table.clamp(min=0).long()], table.long()))
    refs.copy_(torch.zeros_like(refs).index_add_(0, to, torch.where(used, refs, 0)))
    free.copy_(torch.where(at < pages - n, pages - 1 - at, free.long()))
    count.copy_((pages - n).int().view(1))
    return copy_from, copy_to


def _copy(pools, copy_from, copy_to):
    real = copy_from >= 0
    a, b = copy_from[real].long(), copy_to[real].long()
    for pool in pools:
        pool.view(torch.uint8)[b] = pool.view(torch.uint8)[a]


def _groups(table, lengths, page):
    """page_groups in plain operations."""
    rows, width = table.shape
    r = torch.arange(rows, device=table.device)
    whole = (lengths.long() - 1).clamp(min=0) // page  # pages in front of the one with the last position
    first = torch.where((whole > 0) & (table[:, 0] >= 0), table[:, 0].long(), -1 - r)
    leader = torch.where(first[:, None] == first, r, rows).amin(1)
    same = (table == table[leader]) & (table >= 0) & (torch.arange(width, device=table.device) < whole[:, None])
    common = same.int().cumprod(1).sum(1)
    least = torch.full((rows,), width, device=table.device).scatter_reduce_(0, leader, common, "amin")
    members = torch.zeros(rows, dtype=torch.long, device=table.device).index_add_(0, leader, torch.ones_like(r))
    shared = torch.where(members[leader] > 1, least[leader] * page, 0)
    order = (leader * rows + r).argsort()
    ends = members.cumsum(0)
    begins = leader == r
    starts = _into(rows + 1, begins.long().cumsum(0) - 1, ends - members, begins, rows)
    return order.int(), starts.int(), shared.int()


def _gathered(pool, pages, within):
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
    scores = qs @ _gathered(k, pages, at % page).float().permute(0, 2, 3, 1)
    scores = scores.masked_fill(~there, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == -math.inf, 0)).exp()
    total = p.sum(-1, keepdim=True)
    o = p @ _gathered(v, pages, at % page).float().transpose(1, 2) / total.masked_fill(total == 0, 1)
    if s["v_scale"] is not None:
        o = o * s["v_scale"][:, None, None]
    return o.reshape(q.shape).to(q.dtype), (top + total.log()).reshape(batch, heads)


def _logprobs(logits, tokens, top):
    x = logits.float()
    most = x.amax(-1, keepdim=True)
    below = x - most
    p = below.exp()
    total = p.sum(-1, keepdim=True)
    lse = most + total.log()
    entropy = total.log() - torch.where(p > 0, p * below, 0).sum(-1, keepdim=True) / total
    # numbers in the order of the values, the lowest id first of equal ones
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 20) - torch.arange(x.shape[1], device=x.device)
    ids = key.topk(top, -1).indices
    return x.gather(1, tokens[:, None])[:, 0] - lse[:, 0], entropy[:, 0], x.gather(1, ids) - lse, ids


def run(s):
    if own:
        import penny_b200.ops as ops
    op = s["op"]
    if op == "logprobs":
        return tuple(ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])) if own else _logprobs(s["logits"], s["tokens"], s["top"])
    if op == "groups":
        return tuple((ops.page_groups if own else _groups)(s["table"], s["lengths"], s["page"]))
    if op == "fork":
        if own:
            moves = ops.page_fork(*s["state"], s["source"], s["target"], s["page"])
            ops.page_copy(s["pools"], moves.copy_from, moves.copy_to)
            table, lengths, free, count, refs = s["state"]
            ops.page_tables(table, lengths, free, count, s["back"], s["page"], 0, refs=refs)  # the continuations end: the state is as before
        else:
            moves = _fork(*s["state"], s["source"], s["target"], s["page"])
            _copy(s["pools"], *moves[:2])
            _leave(*s["state"], s["back"], s["page"])
        return *moves, *s["state"], *s["pools"]
    if op == "compact":
        torch._foreach_copy_(s["state"], s["before"])  # (so that there is something to move every time; sources keep their contents)
        if own:
            moves = ops.page_compact(*s["state"], s["page"])
            ops.page_copy(s["pools"], moves.copy_from, moves.copy_to)
        else:
            moves = _compact(*s["state"], s["page"])
            _copy(s["pools"], *moves)
        return *moves, *s["state"], *s["pools"]
    if own:
        out = ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=s["window"], k_scale=s["k_scale"],
                                  v_scale=s["v_scale"], lse=s["lse"], groups=s["groups"])
        return out, s["lse"]
    return _attend(s)


def exact(case, seed):
    op = case["op"]
    if op == "groups":
        return None
    s = prepare(case, seed)
    if op == "logprobs":
        if case["rows"] * case["vocab"] > 600 << 20:
            return None
        parts = []
        for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
            y = torch.log_softmax(x.double(), -1)
            parts.append((y.gather(1, t[:, None])[:, 0], -torch.special.xlogy(y.exp(), y.exp()).sum(-1), y.sort(-1, descending=True).values[:, :case["top"]]))
        a, b, c = (torch.cat(p) for p in zip(*parts))
        return a, b, c, None
    if op in ("fork", "compact"):
        # where every page's contents are in the end, by a walk over the lists
        table, lengths, free, count, refs = (t.tolist() for t in s["state"])
        pairs = []
        if op == "fork":
            stack = free[:count[0]]
            for i in s["source"].tolist():
                if lengths[i] % case["page"]:
                    pairs.append((table[i][lengths[i] // case["page"]], stack.pop()))
        else:
            n = sum(c > 0 for c in refs)
            pairs = list(zip([p for p in range(n, len(refs)) if refs[p]], [p for p in range(n) if not refs[p]]))
        pools = [p.double() for p in s["pools"]] if s["pools"][0].numel() * len(s["pools"]) < 1 << 28 else None
        for p in pools or []:
            for a, b in pairs:
                p[b] = p[a].clone()
        return None if pools is None else (*[None] * (8 if op == "fork" else 7), *pools)
    q, k, v = s["q"].double(), s["k"], s["v"]
    batch, heads, dim = q.shape
    out, lse = torch.zeros_like(q), torch.full((batch, heads), -math.inf, dtype=torch.float64, device="cuda")
    page, kv_heads = k.shape[1:3]
    for b, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - s["window"]) if s["window"] else 0
        if n == 0:
            continue
        at = torch.arange(lo, n, device="cuda")
        rows = [_gathered(pool, s["table"][b, at // page], at % page).double() for pool in (k, v)]
        rows = [r if sc is None else r * sc.double()[:, None] for r, sc in zip(rows, (s["k_scale"], s["v_scale"]))]
        keys, values = (r.repeat_interleave(heads // kv_heads, 1) for r in rows)
        logits = torch.einsum("hd,thd->ht", q[b], keys) / dim ** 0.5
        lse[b] = logits.logsumexp(-1)
        out[b] = torch.einsum("ht,thd->hd", (logits - lse[b][:, None]).exp(), values)
    return out, lse


def work(case):
    op = case["op"]
    size = {"e4m3": 1, "bf16": 2, "fp16": 2, "fp32": 4}[case.get("cache", case.get("type", "bf16"))]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 4 * n}
    if op in ("fork", "compact"):
        each = case["page"] * case["kv_heads"] * case["dim"] * size * 2 * case["layers"]
        if op == "fork":
            forks, held = case["prompts"] * case["each"], _pages(case["length"], case["page"])
            copies = forks if case["length"] % case["page"] else 0
            return {"bytes": copies * 2 * each + forks * (held * 8 + 16), "flops": 0}
        used = min(max(case["rows"] + 1, int(case["pages"] * case["full"])), case["pages"] - 1)
        moves = used * (case["pages"] - used) // case["pages"]  # of a pool in random order, about
        return {"bytes": moves * 2 * each + case["pages"] * 12, "flops": 0}
    rows = _rows(case)
    page = case["page"]
    if op == "groups":
        return {"bytes": sum(4 * pre + 12 for _, pre, _ in rows), "flops": 0}
    seen = [(group, pre * page, pre * page + n, max(0, pre * page + n - case["window"]) if case["window"] else 0) for group, pre, n in rows]
    least = {}
    for group, pre, end, lo in seen:
        least[group] = min(least.get(group, lo), lo)
    read = sum(end - max(pre, lo) for _, pre, end, lo in seen)
    read += sum(max(0, pre - least[group]) for group, pre in {(group, pre) for group, pre, _, _ in seen if group >= 0})
    return {"bytes": read * case["kv_heads"] * case["dim"] * 2 * size + len(rows) * (case["heads"] * (case["dim"] * 4 + 4) + 4),
            "flops": 4 * sum(end - lo for _, _, end, lo in seen) * case["heads"] * case["dim"]}
