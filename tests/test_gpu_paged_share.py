"""Rows that have pages in common: forks, rows that leave, compaction, copies and groups, against loops over lists."""
import random

import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Lists:
    """The state of a cache whose rows share pages as Python lists, moved a page at a time."""

    def __init__(self, rows, width, pages, page, rng):
        self.page, self.width, self.pages = page, width, pages
        self.table, self.lengths, self.refs = [[-1] * width for _ in range(rows)], [0] * rows, [0] * pages
        self.free = list(range(pages))
        rng.shuffle(self.free)

    def tensors(self, stride=None):
        t = _ints(self.table)
        if stride:
            wide = torch.full((len(self.table), stride), -7, dtype=torch.int32, device="cuda")
            wide[:, :self.width] = t
            t = wide[:, :self.width]
        free = torch.full((self.pages,), -5, dtype=torch.int32, device="cuda")
        free[:len(self.free)] = _ints(self.free)
        return t, _ints(self.lengths), free, _ints([len(self.free)]), _ints(self.refs)

    def held(self, n):
        return -(-n // self.page)

    def step(self, new, tokens):
        gone = [(r, i) for r in range(len(new)) if new[r] < 0 for i in range(self.held(max(0, self.lengths[r] + new[r])), self.held(self.lengths[r]))]
        for r, i in gone:
            self.refs[self.table[r][i]] -= 1
        back = set()
        for r, i in reversed(gone):
            p = self.table[r][i]
            if self.refs[p] == 0 and p not in back:
                back.add(p)
                self.free.append(p)
        for r, n in enumerate(new):
            if n < 0:
                self.lengths[r] = max(0, self.lengths[r] + n)
        slots, granted, end, asked, there = [-1] * tokens, [], 0, 0, len(self.free)
        for r, n in enumerate(new):
            first, end, L = end, end + max(0, n), self.lengths[r]
            ok = n <= 0
            if n > 0 and L + n <= self.width * self.page and end <= tokens and (L % self.page == 0 or self.refs[self.table[r][L // self.page]] <= 1):
                need = self.held(L + n) - self.held(L)
                asked += need
                ok = need == 0 or asked <= there
            granted.append(ok)
            if not ok or n <= 0:
                continue
            for i in range(self.held(L), self.held(L + n)):
                self.table[r][i] = p = self.free.pop()
                self.refs[p] = 1
            for j in range(n):
                slots[first + j] = self.table[r][(L + j) // self.page] * self.page + (L + j) % self.page
            self.lengths[r] = L + n
        return slots, granted

    def fork(self, source, target):
        before, there, asked, taken = list(self.lengths), len(self.free), 0, set()
        copies, granted = [], []
        for s, t in zip(source, target):
            rows = range(len(self.table))
            ok = s in rows and t in rows and s != t and before[t] == 0 and t not in taken
            if ok:
                taken.add(t)  # (granted a page or not)
                if before[s] % self.page:
                    asked += 1
                    ok = asked <= there
            granted.append(ok)
            if not ok:
                continue
            full = before[s] // self.page
            self.table[t][:full] = self.table[s][:full]
            for p in self.table[s][:full]:
                self.refs[p] += 1
            if before[s] % self.page:
                p = self.free.pop()
                self.refs[p] = 1
                copies.append((self.table[s][full], p))
                self.table[t][full] = p
            self.lengths[t] = before[s]
        return copies, granted

    def compact(self):
        used = [p for p in range(self.pages) if self.refs[p] > 0]
        n = len(used)
        moves = list(zip([p for p in used if p >= n], [p for p in range(n) if self.refs[p] == 0]))
        to = dict(moves)
        for r, L in enumerate(self.lengths):
            for i in range(self.held(L)):
                self.table[r][i] = to.get(self.table[r][i], self.table[r][i])
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.free = list(range(self.pages - 1, n - 1, -1))
        return moves

    def same(self, table, lengths, free, count, refs):
        assert lengths.tolist() == self.lengths and count.item() == len(self.free)
        assert free.tolist()[:len(self.free)] == self.free
        assert refs.tolist() == self.refs
        t = table.tolist()
        for r, n in enumerate(self.lengths):
            assert t[r][:self.held(n)] == self.table[r][:self.held(n)], r
        # the pages of the rows and of the stack are all there are
        counts = [0] * self.pages
        for r, n in enumerate(self.lengths):
            for p in self.table[r][:self.held(n)]:
                counts[p] += 1
        assert counts == self.refs and sorted(self.free + [p for p in range(self.pages) if counts[p]]) == list(range(self.pages))


def _pairs(moves):
    got = [(a, b) for a, b in zip(moves.copy_from.tolist(), moves.copy_to.tolist())]
    real = [p for p in got if p[0] >= 0]
    assert got[:len(real)] == real and all(p == (-1, -1) for p in got[len(real):])
    return real


@pytest.mark.parametrize("rows,width,pages,page,chunk", [
    (2, 1, 1, 1, 1), (2, 3, 2, 16, 20), (4, 5, 9, 16, 30), (40, 12, 200, 5, 30), (130, 40, 2000, 1, 9), (257, 6, 700, 24, 60), (300, 90, 9000, 16, 700),
    (1030, 4, 2500, 128, 300), (2500, 9, 9500, 7, 40), (8192, 3, 12000, 16, 40)])
def test_steps(rows, width, pages, page, chunk):
    """Rows are forked, grow and leave at random, pools run full, and the pages are moved together in between."""
    rng = random.Random(rows * 7 + page)
    want = Lists(rows, width, pages, page, rng)
    state = want.tensors(stride=width + 3 if rows % 2 else None)
    for step in range(8):
        tokens = rng.choice([0, 4 * rows, 40 * rows])
        new = []
        for r in range(rows):
            kind = rng.random()
            new.append(0 if kind < 0.2 else 1 if kind < 0.4 else rng.randint(1, chunk) if kind < 0.6 else
                       -rng.randint(1, width * page + 5) if kind < 0.8 else -want.lengths[r])
        got = P.page_tables(*state[:4], _ints(new), page, tokens, refs=state[4])
        slots, granted = want.step(new, tokens)
        assert got.granted.tolist() == granted and got.slots.tolist() == slots, step
        want.same(*state)
        empty = [r for r in range(rows) if want.lengths[r] == 0]
        rng.shuffle(empty)
        target = empty[:rng.randint(0, len(empty))] + rng.choices(range(-1, rows + 1), k=3)
        rng.shuffle(target)
        source = [rng.choice(range(-1, rows + 1)) if rng.random() < 0.1 else rng.randrange(rows) for _ in target]
        source, target = source[:8192], target[:8192]
        fork = P.page_fork(*state, _ints(source), _ints(target), page)
        copies, granted = want.fork(source, target)
        assert fork.granted.tolist() == granted and _pairs(fork) == copies, step
        want.same(*state)
        if step % 3 == 2:
            assert _pairs(P.page_compact(*state, page)) == want.compact()
            want.same(*state)
    if state[0].stride(0) > width:
        assert (torch.as_strided(state[0], (rows, 3), (width + 3, 1), width) == -7).all()  # nothing behind the rows


def test_no_forks_and_no_pages():
    rng = random.Random(0)
    want = Lists(3, 4, 1, 16, rng)
    state = want.tensors()
    none = _ints([])
    got = P.page_fork(*state, none, none, 16)
    assert got.granted.numel() == 0 and got.copy_from.numel() == 0
    P.page_copy([], none, none)
    moves = P.page_compact(*state, 16)
    assert moves.copy_from.numel() == 0
    want.compact()
    want.same(*state)


def test_one_call_releases_a_page_of_many_rows():
    """All rows of a fork leave at once: each page is on the stack once, in the place of the last row that had it."""
    want = Lists(600, 40, 3000, 8, random.Random(1))
    want.step([300] + [0] * 599, 300)
    want.fork([0] * 599, list(range(1, 600)))
    state = want.tensors()
    new = [-want.lengths[r] if r % 5 else 0 for r in range(600)]
    P.page_tables(*state[:4], _ints(new), 8, 0, refs=state[4])
    want.step(new, 0)
    want.same(*state)
    new = [-300 if r % 5 == 0 else 0 for r in range(600)]
    P.page_tables(*state[:4], _ints(new), 8, 0, refs=state[4])
    want.step(new, 0)
    want.same(*state)
    assert want.refs == [0] * 3000


def test_what_is_not_there():
    """Counts, lengths and pages that no state can have: nothing past the ends."""
    table = _ints([[0, 99, -4, 2 ** 31 - 1], [-1] * 4, [-1] * 4])
    lengths, free, count, refs = _ints([60, 0, -8]), _ints([3, 77, 1, 2]), _ints([900]), _ints([1, 1, 1, 1])
    got = P.page_fork(table, lengths, free, count, refs, _ints([0, 0, 0]), _ints([1, 2, 1]), 16)
    assert got.granted.tolist() == [True, True, False] and int(count) == 2 and lengths.tolist() == [60, 60, 60]
    assert table.tolist()[1][:3] == [0, 99, -4] and refs.tolist()[0] == 3
    pools = [torch.randn(4, 16, 2, 64, device="cuda").bfloat16() for _ in range(3)]
    before = [p.clone() for p in pools]
    P.page_copy(pools, got.copy_from, got.copy_to)  # from pages that the pool does not have: nothing is copied
    assert all(torch.equal(a, b) for a, b in zip(pools, before))
    P.page_tables(table, lengths, free, _ints([-3]), _ints([-2 ** 31, -60, 0]), 16, 0, refs=refs)
    assert lengths.tolist()[:2] == [0, 0]
    P.page_groups(table, lengths, 16)
    P.page_compact(table, _ints([2 ** 31 - 1, -5, 0]), free, count, refs, 16)


def _layouts(pages, page, heads, dim, dtype):
    def fill(t):
        return t.copy_(torch.randint(0, 255, t.shape, device="cuda", dtype=torch.uint8)) if t.dtype == torch.uint8 else t.normal_()
    raw = torch.uint8 if dtype == torch.float8_e4m3fn else dtype
    new = lambda *s: fill(torch.empty(*s, dtype=raw, device="cuda"))  # noqa: E731
    yield "dense", [new(pages, page, heads, dim) for _ in range(5)]
    yield "by head", [new(pages, heads, page, dim).transpose(1, 2) for _ in range(3)]
    yield "heads outside", [new(heads, pages, page, dim).permute(1, 2, 0, 3) for _ in range(2)]
    yield "positions outside", [new(page, pages, heads, dim).transpose(0, 1) for _ in range(2)]
    both = new(pages, page, 2 * heads, dim)
    yield "k and v in one", [both[:, :, :heads], both[:, :, heads:]]
    wide = new(pages, page, heads, dim + 16)
    yield "padded", [wide[..., :dim]]
    yield "by head, padded", [new(pages, heads, page + 1, dim + 16).transpose(1, 2)[:, 1:, :, 16:]]


@pytest.mark.parametrize("pages,page,heads,dim,dtype", [(9, 16, 8, 128, torch.bfloat16), (40, 1, 1, 64, torch.float8_e4m3fn), (7, 5, 3, 256, torch.float16),
                                                        (300, 24, 2, 16, torch.bfloat16), (5, 700, 4, 128, torch.float8_e4m3fn)])
def test_copy(pages, page, heads, dim, dtype):
    rng = random.Random(pages)
    for name, pools in _layouts(pages, page, heads, dim, dtype):
        ids = list(range(pages))
        rng.shuffle(ids)
        n = pages // 3
        pairs = list(zip(ids[:n], ids[n:2 * n]))
        pairs += [(ids[0], ids[2 * n])]                    # a page that goes to two
        pairs.insert(1, (pages, ids[-1]))                  # pages that are none: left out
        pairs.insert(2, (ids[0], pages + 5))
        pairs.insert(2, (ids[0], -1))
        pairs += [(-1, ids[-1])] * 500                     # the end of a list that has room for more
        want = [p.clone() for p in pools]
        for a, b in pairs:
            if 0 <= a < pages and 0 <= b < pages:
                for w in want:
                    w[b] = w[a].clone()
        wholes = [p._base.clone() if p._base is not None else p.clone() for p in pools]
        P.page_copy([p.view(dtype) if p.dtype == torch.uint8 and p.is_contiguous() else p for p in pools], _ints([a for a, _ in pairs]), _ints([b for _, b in pairs]))
        for got, w, whole in zip(pools, want, wholes):
            assert torch.equal(got, w), name
            if got._base is not None and len(pools) == 1:  # nothing between the rows was touched
                back = got.clone()
                got.copy_(torch.as_strided(whole, got.shape, got.stride(), got.storage_offset()))
                assert torch.equal(got._base, whole), name
                got.copy_(back)


def test_copy_of_many_pools():
    pools = [torch.randn(6, 4, 2, 64, device="cuda").bfloat16() for _ in range(300)]
    want = [p.clone() for p in pools]
    P.page_copy(pools, _ints([0, 3]), _ints([5, 1]))
    for p, w in zip(pools, want):
        w[5], w[1] = w[0].clone(), w[3].clone()
        assert torch.equal(p, w)


def _groups_of(table, lengths, page):
    rows, width = len(table), len(table[0])
    whole = [max(0, min(n, width * page) - 1) // page for n in lengths]
    leader = []
    for r in range(rows):
        same = [x for x in range(r) if leader[x] == x and whole[r] and whole[x] and table[x][0] == table[r][0] >= 0]
        leader.append(same[0] if same else r)
    order, starts, shared = [], [], [0] * rows
    for g in range(rows):
        mine = [r for r in range(rows) if leader[r] == g]
        if not mine:
            continue
        starts.append(len(order))
        order += mine
        if len(mine) > 1:
            least = width
            for r in mine:
                n = 0
                while n < min(whole[r], whole[g]) and table[r][n] == table[g][n] >= 0:
                    n += 1
                least = min(least, n)
            for r in mine:
                shared[r] = least * page
    return order, starts + [rows] * (rows + 1 - len(starts)), shared


@pytest.mark.parametrize("rows,width,page,first", [(1, 1, 1, 1), (2, 3, 4, 1), (5, 9, 16, 2), (33, 300, 16, 1), (64, 40, 24, 3), (100, 7, 1, 100), (257, 130, 5, 9),
                                                   (1000, 20, 16, 50), (1025, 5, 16, 1), (8192, 3, 16, 700), (8191, 4, 2, 1)])
def test_groups(rows, width, page, first):
    """Tables whose rows begin with one of a few texts and part somewhere; rows of every length, ids below zero, a wider table."""
    rng = random.Random(rows + width)
    texts = [[rng.randrange(10 * width) for _ in range(width)] for _ in range(first)]
    table, lengths = [], []
    for r in range(rows):
        t = list(rng.choice(texts))
        at = rng.randrange(width + 1) if rng.random() < 0.5 else width
        t[at:] = [rng.randrange(-1, 2 ** 31 - 1) for _ in range(width - at)]
        table.append(t)
        lengths.append(rng.choice([0, -3, 1, page, page + 1, width * page, width * page + 9, rng.randrange(width * page + 1)] if rng.random() < 0.3 else
                                  [width * page - rng.randrange(page)]))
    t = torch.full((rows, width + 2), 5, dtype=torch.int32, device="cuda")
    t[:, :width] = _ints(table)
    got = P.page_groups(t[:, :width], _ints(lengths), page)
    for a, b, name in zip(got, _groups_of(table, lengths, page), got._fields):
        assert a.tolist() == b, name


def test_graph_and_stream():
    """Fork, copy, step, groups and leave in one graph, on a stream of its own, that is replayed: the state goes on, the copies are made."""
    cache = P.PagedKVCache(2, 8, 100, 2, head_dim=64, page_size=8, sharing=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = _ints([43] + [0] * 7)
        cache.advance(first, 43)
        for t in cache.k + cache.v:
            t.normal_()
        source, target, one, leave = _ints([0] * 7), _ints(list(range(1, 8))), _ints([0] + [1] * 7), _ints([0] + [-44] * 7)
        snapshot = cache.snapshot()
        pools = [t.clone() for t in cache.k + cache.v]

        def round_():
            fork = cache.fork(source, target)
            step = cache.advance(one, 7)
            groups = cache.groups()
            cache.advance(leave, 0)
            return fork, step, groups
        want = [[t.clone() for t in part] for part in round_()]
        after = [t.clone() for t in cache.k + cache.v]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = round_()
        for _ in range(3):
            for t, old in zip(cache.k + cache.v, pools):
                t.copy_(old)
            graph.replay()
            for part, w in zip(got, want):
                for a, b in zip(part, w):
                    assert torch.equal(a, b)
            assert all(torch.equal(a, b) for a, b in zip(cache.k + cache.v, after))
            table, lengths, free, count, refs = snapshot
            n = int(count)  # (what is behind the rows' pages and the stack's top says nothing)
            assert torch.equal(cache.table[0, :6], table[0, :6]) and torch.equal(cache.free[:n], free[:n])
            assert torch.equal(cache.lengths, lengths) and torch.equal(cache.free_count, count) and torch.equal(cache.refs, refs)
        assert got[0].granted.all() and got[1].granted.all() and got[2].shared.tolist() == [40] * 8
        assert got[1].positions.tolist() == [43] * 7
        s.synchronize()


def test_a_row_cut_back_into_shared_pages():
    cache = P.PagedKVCache(1, 4, 64, 1, head_dim=64, page_size=8, sharing=True)
    cache.advance(_ints([20, 0, 0, 0]), 20)
    cache.k[0].normal_()
    cache.fork(_ints([0]), _ints([1]))
    cache.advance(_ints([0, -9, 0, 0]), 0)  # 11 positions: inside the second page, which row 0 has too
    step = cache.advance(_ints([1, 1, 0, 0]), 2)
    assert step.granted.tolist() == [True, False, True, True] and cache.lengths.tolist() == [21, 11, 0, 0]
    fork = cache.fork(_ints([1]), _ints([2]))
    assert fork.granted.item()
    assert cache.advance(_ints([0, 0, 1, 0]), 1).granted.all()
    assert torch.equal(cache.rows_of(0, 2, 11)[0], cache.rows_of(0, 0, 11)[0])
    cache.advance(_ints([0, -11, 0, 0]), 0)
    cache.advance(_ints([-21, 0, -12, 0]), 0)
    assert int(cache.free_count) == cache.pages and not cache.refs.any()


def test_compaction_keeps_what_rows_hold():
    rng = random.Random(5)
    cache = P.PagedKVCache(3, 30, 90, 2, head_dim=64, page_size=8, pages=200, sharing=True, dtype=torch.float8_e4m3fn)
    cache.advance(_ints([rng.randrange(40) for _ in range(20)] + [0] * 10), 2000)
    for t in cache.k + cache.v:
        t.copy_(torch.randn(t.shape, device="cuda").to(t.dtype))
    cache.fork(_ints([rng.randrange(20) for _ in range(10)]), _ints(list(range(20, 30))))
    cache.advance(torch.where(torch.arange(30, device="cuda") % 3 == 0, -cache.lengths, 0).int(), 0)
    lengths = cache.lengths.tolist()
    before = [[cache.rows_of(i, r, lengths[r]) for r in range(30)] for i in range(3)]
    cache.compact()
    used = int((cache.refs > 0).sum())
    assert not (cache.refs[used:] > 0).any() and int(cache.free_count) == 200 - used and cache.lengths.tolist() == lengths
    for i in range(3):
        for r in range(30):
            for a, b in zip(cache.rows_of(i, r, lengths[r]), before[i][r]):
                assert torch.equal(a, b)
    assert cache.advance(_ints([1] * 30), 30).granted.all()
