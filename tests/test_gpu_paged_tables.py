"""Block tables and slot maps from request lengths, against a loop over lists."""
import random

import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Lists:
    """The same state as Python lists, moved a page at a time."""

    def __init__(self, rows, width, pages, page, rng):
        self.page, self.width = page, width
        self.table, self.lengths = [[-1] * width for _ in range(rows)], [0] * rows
        self.free = list(range(pages))
        rng.shuffle(self.free)
        self.count = pages

    def tensors(self, stride=None):
        t = _ints(self.table)
        if stride:
            wide = torch.full((len(self.table), stride), -7, dtype=torch.int32, device="cuda")
            wide[:, :self.width] = t
            t = wide[:, :self.width]
        return t, _ints(self.lengths), _ints(self.free), _ints([self.count])

    def held(self, n):
        return -(-n // self.page)

    def step(self, new, tokens):
        for r in reversed(range(len(new))):
            if new[r] < 0:
                left = max(0, self.lengths[r] + new[r])
                for i in reversed(range(self.held(left), self.held(self.lengths[r]))):
                    self.free[self.count] = self.table[r][i]
                    self.count += 1
                self.lengths[r] = left
        slots, positions, offsets, granted, end, asked, there = [-1] * tokens, [0] * tokens, [0], [], 0, 0, self.count
        for r, n in enumerate(new):
            first, end = end, end + max(0, n)
            offsets.append(end)
            L = self.lengths[r]
            ok = n <= 0
            if n > 0 and L + n <= self.width * self.page and end <= tokens:
                need = self.held(L + n) - self.held(L)
                asked += need
                ok = need == 0 or asked <= there
            granted.append(ok)
            if not ok or n <= 0:
                continue
            for i in range(self.held(L), self.held(L + n)):
                self.count -= 1
                self.table[r][i] = self.free[self.count]
            for j in range(n):
                slots[first + j] = self.table[r][(L + j) // self.page] * self.page + (L + j) % self.page
                positions[first + j] = L + j
            self.lengths[r] = L + n
        return slots, positions, offsets, granted

    def same(self, table, lengths, free, count):
        assert lengths.tolist() == self.lengths and count.item() == self.count
        assert free.tolist()[:self.count] == self.free[:self.count]
        t = table.tolist()
        for r, n in enumerate(self.lengths):
            assert t[r][:self.held(n)] == self.table[r][:self.held(n)], r


@pytest.mark.parametrize("rows,width,pages,page,chunk,tokens", [
    (1, 1, 1, 1, 1, 1), (1, 4, 3, 16, 40, 40), (3, 5, 9, 16, 30, 61), (40, 12, 200, 5, 30, 500), (130, 40, 3000, 1, 9, 1001),
    (257, 6, 900, 24, 60, 3000), (300, 9, 1500, 16, 120, 9003), (1030, 4, 2500, 128, 3, 4096), (2500, 3, 5000, 7, 12, 20000), (8192, 2, 9000, 16, 5, 30001)])
def test_steps(rows, width, pages, page, chunk, tokens):
    """Tokens come and leave at random over several steps: rows and pools that run full, too many tokens, empty rows."""
    rng = random.Random(rows * 7 + page)
    want = Lists(rows, width, pages, page, rng)
    state = want.tensors(stride=width + 3 if rows % 2 else None)
    for step in range(8):
        new = []
        for r in range(rows):
            kind = rng.random()
            new.append(0 if kind < 0.1 else 1 if kind < 0.4 else rng.randint(1, chunk) if kind < 0.75 else
                       -rng.randint(1, width * page + 5) if kind < 0.95 else -want.lengths[r])
        got = P.page_tables(*state, _ints(new), page, tokens)
        said = want.step(new, tokens)
        for a, b, name in zip(got, said, got._fields):
            assert a.tolist() == b, (step, name)
        want.same(*state)
    if state[0].stride(0) > width:
        assert (torch.as_strided(state[0], (rows, 3), (width + 3, 1), width) == -7).all()  # nothing behind the rows


@pytest.mark.parametrize("rows,chunk", [(5, 200), (900, 30), (3000, 9)])
def test_back_and_forth(rows, chunk):
    """What comes and leaves again is back in its old place."""
    rng = random.Random(rows)
    want = Lists(rows, 40, rows * 30, 16, rng)
    state = want.tensors()
    P.page_tables(*state, _ints([rng.randint(0, 200) for _ in range(rows)]), 16, 200 * rows)
    before = [t.clone() for t in state]
    new = _ints([rng.randint(0, chunk) for _ in range(rows)])
    assert P.page_tables(*state, new, 16, chunk * rows).granted.all()
    assert not torch.equal(state[1], before[1])
    P.page_tables(*state, -new, 16, 0)
    assert torch.equal(state[1], before[1]) and torch.equal(state[3], before[3])
    n = int(state[3])
    assert torch.equal(state[2][:n], before[2][:n])


def test_extremes():
    """Numbers that do not fit 32 bits together, lengths and counts that no table can have: refused or cut, nothing past the ends."""
    table, lengths, free, count = torch.zeros(4, 3, dtype=torch.int32, device="cuda"), _ints([0, 5, 40, 48]), _ints(list(range(20))), _ints([20])
    top = 2 ** 31 - 1
    got = P.page_tables(table, lengths, free, count, _ints([top, top, top, 1]), 16, 64)
    assert got.granted.tolist() == [False] * 4 and lengths.tolist() == [0, 5, 40, 48] and int(count) == 20
    assert got.slots.tolist() == [-1] * 64 and got.offsets.tolist() == [0, top, top, top, top]
    P.page_tables(table, lengths, free, count, _ints([0, -2 ** 31, 0, -1]), 16, 0)
    assert lengths.tolist() == [0, 0, 40, 47]
    # a length past the table row counts as the row, one below zero as none; a count past the stack as all of it
    lengths, count = _ints([500, -9, 48, 0]), _ints([700])
    got = P.page_tables(table, lengths, free, count, _ints([1, 16, 0, 1]), 16, 17)
    assert got.granted.tolist() == [False, True, True, False] and lengths.tolist() == [48, 16, 48, 0] and int(count) == 19
    # pages that the pool does not have: no slots
    free = torch.full((20,), 20, dtype=torch.int32, device="cuda")
    got = P.page_tables(table, _ints([0] * 4), free, _ints([20]), _ints([1] * 4), 16, 4)
    assert got.slots.tolist() == [-1] * 4


def test_out_graph_and_stream():
    """The caller's own tensors, in a graph that keeps counting, on a stream of its own."""
    rng = random.Random(3)
    want = Lists(70, 20, 900, 8, rng)
    state = want.tensors()
    new = _ints([1] * 70)
    out = P.PageStep(torch.empty(80, dtype=torch.int64, device="cuda"), torch.empty(80, dtype=torch.int32, device="cuda"),
                     torch.empty(71, dtype=torch.int32, device="cuda"), torch.empty(70, dtype=torch.bool, device="cuda"))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        P.page_tables(*state, new, 8, 80, out)
        want.step([1] * 70, 80)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = P.page_tables(*state, new, 8, 80, out)
        assert got.slots.data_ptr() == out.slots.data_ptr()
        for _ in range(20):
            graph.replay()
            said = want.step([1] * 70, 80)
        s.synchronize()
    for a, b in zip(out, said):
        assert a.tolist() == b
    want.same(*state)
