"""Attention over a paged KV cache whose rows share pages, against 64 bits."""
import math
import random

import pytest
import torch

import penny_b200.ops as P
from penny_b200._ext import ops

pytestmark = pytest.mark.gpu
BF, HALF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """Rows (group, shared positions, own positions) in a random order over a shuffled pool; pages that no row has hold NaN."""

    def __init__(self, rows, heads, kv_heads, dim, page, cache=BF, q=None, seed=0, spread=2.0, layout="dense"):
        rng = random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.page, self.dim, self.kv_heads, self.heads = page, dim, kv_heads, heads
        rows = list(rows)
        rng.shuffle(rows)
        shared = {}
        for group, pre, _ in rows:
            assert shared.setdefault(group, pre) == pre and pre % page == 0
        held = lambda n: -(-n // page)  # noqa: E731
        total = sum(held(n) for group, n in shared.items() if group is not None) + sum(held(n) for _, _, n in rows) + 3
        ids = list(range(total))
        rng.shuffle(ids)
        of = {group: [ids.pop() for _ in range(held(n))] for group, n in shared.items()}
        table = [of[group] + [ids.pop() for _ in range(held(n))] for group, _, n in rows]
        # (a table for so long rows that the kernel for shared pages is what runs; what is behind the rows' pages says nothing)
        width = max(max(len(t) for t in table) + 2, (260 << 20) // (len(rows) * page * kv_heads * dim * 2 * (1 if cache == F8 else 2)))
        self.table = _ints([t + [-1] * (width - len(t)) for t in table])
        self.lengths = _ints([pre + n for _, pre, n in rows])
        dtype = q or (BF if cache == F8 else cache)
        self.q = torch.randn(len(rows), heads, dim, device="cuda", generator=g).mul_(spread).to(dtype)
        shape = {"dense": (total, page, kv_heads, dim), "by head": (total, kv_heads, page, dim)}[layout]
        make = lambda: torch.randn(*shape, device="cuda", generator=g).mul_(100 if cache == F8 else 1).clamp_(-448, 448).to(cache)  # noqa: E731
        self.k, self.v = make(), make()
        nan = torch.full((1,), math.nan, device="cuda").to(cache)
        for t in (self.k, self.v):  # what no row has
            view = t.view(torch.uint8)
            for i in ids:
                view[i] = nan.view(torch.uint8).repeat(t[i].numel()).view(view[i].shape)
        if layout == "by head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for r, (group, pre, n) in enumerate(rows):  # what is behind a row's last position
            last = pre + n
            if n % page:
                for t in (self.k, self.v):
                    t.view(torch.uint8)[table[r][last // page], last % page:] = nan.view(torch.uint8).repeat(dim)
        self.scales = [0.01 + 0.01 * torch.rand(kv_heads, device="cuda", generator=g) if cache == F8 else None for _ in range(2)]

    def want(self, window=0, scale=None):
        """(out, lse, sum of weights times |v|, largest sum of |q| |k|) in 64 bits."""
        q = self.q.double()
        scale = self.dim ** -0.5 if scale is None else scale
        B, H = q.shape[:2]
        out, absv, lse, size = torch.zeros_like(q), torch.zeros_like(q), torch.full((B, H), -math.inf, device="cuda", dtype=torch.float64), torch.zeros(B, H, device="cuda", dtype=torch.float64)
        for b, n in enumerate(self.lengths.tolist()):
            at = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
            pages = self.table[b, at // self.page].long()
            there = (pages >= 0) & (pages < self.k.shape[0])
            at, pages = at[there], pages[there]
            if at.numel() == 0:
                continue
            rows = []
            for pool, s in ((self.k, self.scales[0]), (self.v, self.scales[1])):
                x = pool.view(torch.uint8)[pages, at % self.page].view(pool.dtype).double() if pool.dtype == F8 else pool[pages, at % self.page].double()
                rows.append((x if s is None else x * s.double()[:, None]).repeat_interleave(H // self.kv_heads, 1))
            logits = torch.einsum("hd,thd->ht", q[b], rows[0]) * scale
            w = logits.softmax(-1)
            lse[b], out[b], absv[b] = logits.logsumexp(-1), torch.einsum("ht,thd->hd", w, rows[1]), torch.einsum("ht,thd->hd", w, rows[1].abs())
            size[b] = torch.einsum("hd,thd->ht", q[b].abs(), rows[0].abs()).amax(-1) * abs(scale)
        return out, lse, absv, size

    def groups(self):
        return P.page_groups(self.table, self.lengths, self.page)

    def check(self, window=0, scale=None, groups=None, **more):
        lse = torch.full(self.q.shape[:2], math.nan, device="cuda")
        out = P.paged_attention(self.q, self.k, self.v, self.table, self.lengths, lse=lse, window=window, scale=scale, k_scale=self.scales[0],
                                v_scale=self.scales[1], groups=groups or self.groups(), **more)
        assert ops.gemm_error() == 0
        want, want_lse, absv, size = self.want(window, scale)
        # A score is a sum of dim products in fp32 and three roundings; a weight follows it, has 2^-21 of its own (exponential, base)
        # and is rounded to its type (fp16 ones stand so high that 2^-31 of the largest is lost), the output once more.
        h = torch.finfo(out.dtype).eps / 2
        n = int(self.lengths.clamp(min=1).max())
        rel = 2 * (self.dim + 8) * 2.0 ** -24 * size + 2.0 ** -20 + n * 2.0 ** -31
        assert ((out.double() - want).abs() <= (2 * h + 2 * rel[..., None] + n * 2.0 ** -24) * absv + h * want.abs() * (1 + h) + 1e-30).all(), \
            ((out.double() - want).abs() / (absv + 1e-30)).max()
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        assert ((lse.double() - want_lse).abs().masked_fill(empty, 0) <= rel + (n + 8) * 2.0 ** -24 + want_lse.abs().masked_fill(empty, 0) * 2.0 ** -22).all()
        return out


LAYOUTS = [(4, 1, 128), (32, 8, 128), (8, 2, 64), (20, 20, 64), (35, 7, 64), (28, 2, 128), (8, 1, 256), (64, 1, 64), (24, 2, 256), (150, 1, 128), (300, 1, 64)]


def test_one_group():
    """The smallest: two rows over one tile of shared positions."""
    Case([(0, 128, 5)] * 2, 4, 1, 128, 16).check()


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("cache", [BF, HALF, F8])
def test_layouts(heads, kv_heads, dim, cache):
    rng = random.Random(heads)
    rows = [(0, 160, rng.randint(1, 60)) for _ in range(5)] + [(1, 528, rng.randint(1, 300)) for _ in range(3)] + [(None, 0, n) for n in (0, 1, 17, 400, 0)]
    case = Case(rows, heads, kv_heads, dim, 16, cache, seed=heads)
    case.check()
    if cache == F8:
        Case(rows, heads, kv_heads, dim, 16, cache, q=HALF, seed=heads + 1).check()


@pytest.mark.parametrize("page", [1, 5, 16, 24, 63, 128, 300])
def test_page_sizes(page):
    pre = max(1, 700 // page) * page
    rows = [(0, pre, n) for n in (1, page, page + 1, 3 * page)] + [(1, page, 130)] * 2 + [(None, 0, 77)]
    Case(rows, 8, 2, 128, page, seed=page).check()
    Case(rows, 8, 2, 64, page, HALF, seed=page, layout="by head").check()


@pytest.mark.parametrize("members,own", [(2, 1), (3, 300), (33, 40), (64, 7), (65, 130), (130, 3), (300, 20)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (4, 1, 64), (8, 1, 256)])
def test_members(members, own, heads, kv_heads, dim):
    """Groups of fewer queries than a tile, of one, two, and several pairs of them."""
    rng = random.Random(members)
    rows = [(0, 1040, rng.randint(1, own)) for _ in range(members)] + [(1, 32, 50), (1, 32, 1)]
    Case(rows, heads, kv_heads, dim, 16, seed=members).check()


@pytest.mark.parametrize("window", [1, 2, 40, 128, 129, 600, 5000])
@pytest.mark.parametrize("cache", [BF, F8])
def test_windows(window, cache):
    rows = [(0, 512, n) for n in (1, 5, 64, 500)] + [(1, 48, 90)] * 3 + [(None, 0, n) for n in (0, 3, 1000)]
    Case(rows, 8, 2, 128, 16, cache, seed=window).check(window=window)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 1e-30, 20.0])
def test_scales(scale):
    case = Case([(0, 256, n) for n in (1, 5, 200)] + [(None, 0, 30)], 8, 2, 128, 16, spread=0.5)
    case.check(scale=scale)


@pytest.mark.parametrize("cache", [BF, HALF, F8])
def test_weights_that_grow_and_shrink(cache):
    """Scores that rise along the positions by more than the base may lag, fall, or stand far above all others once."""
    for kind in range(4):
        case = Case([(0, 1536, n) for n in (1, 100, 400)] + [(None, 0, 500)], 8, 2, 128, 16, cache, seed=kind, spread=1.0)
        at = torch.arange(1536, device="cuda")
        pages = case.table[0 if case.lengths[0] > 1500 else 1, at // 16].long()
        by = [at / 1536, 1 - at / 1536, (at == 700).float(), (at % 128 == 127).float()][kind] * (40.0 if cache == F8 else 4.0)
        dirn = torch.sign(case.q[0, 0].float())
        k = case.k.float() * 0.2
        k[pages, at % 16] += by[:, None, None] * dirn
        case.k = k.to(cache)
        case.check()


def test_pages_that_are_not_there():
    case = Case([(0, 640, n) for n in (20, 90, 300)] + [(None, 0, 200)], 8, 2, 128, 16, seed=3)
    groups = case.groups()
    shared = groups.shared.tolist()
    inside = [r for r in range(4) if shared[r]]
    for r in inside:  # in what they share, alike
        case.table[r, 3] = -1
        case.table[r, 9] = 10 ** 6
        case.table[r, 16:24] = 2 ** 31 - 1
    case.table[inside[0], 40] = -7  # and in a row's own pages
    case.check(groups=groups)
    case.table.fill_(-1)
    out = case.check(groups=groups)
    assert not out.any()


def test_empty_rows_and_odd_groups():
    """Rows without positions; groups in which nothing is shared; rows that grew or were cut back since the groups were found."""
    Case([(None, 0, 0)] * 5, 8, 2, 128, 16).check()
    case = Case([(0, 320, n) for n in (7, 40, 100, 200)] + [(1, 64, 30)] * 2, 8, 2, 64, 16, seed=9)
    groups = case.groups()
    for lengths in ([0] * 6, [10] * 6, [330, 321, 400, 319, 64, 65], [1, 400, 0, 325, 90, 66]):
        keep, case.lengths = case.lengths, _ints([min(a, b) for a, b in zip(lengths, case.lengths.tolist())])
        case.check(groups=groups)
        case.lengths = keep
    n = len(groups.order)
    alone = P.PageGroups(torch.arange(n, device="cuda").int(), torch.arange(n + 1, device="cuda").int(), torch.zeros(n, device="cuda").int())
    case.check(groups=alone)


def test_groups_that_say_nothing():
    """Numbers that are no groups: nothing is read or written that is not the call's, and the call ends."""
    case = Case([(0, 320, n) for n in (7, 40, 100, 200)], 8, 2, 128, 16, seed=2)
    top = 2 ** 31 - 1
    for order, starts, shared in (([9, -1, 7, top], [0, 2, 4, 4, 4], [320] * 4), ([0, 1, 2, 3], [0, 4, 0, 4, 0], [320] * 4), ([0, 1, 2, 3], [-5, top, -top, 3, 9], [top, -top, 5, 7]),
                                  ([0, 0, 0, 0], [0, 4, 4, 4, 4], [top] * 4), ([3, 2, 1, 0], [4, 3, 2, 1, 0], [-1] * 4)):
        P.paged_attention(case.q, case.k, case.v, case.table, case.lengths, groups=(_ints(order), _ints(starts), _ints(shared)))
        assert ops.gemm_error() == 0
    case.check()


def test_infinities_and_nan():
    """What softmax gives for them, in the rows that see them and in no others."""
    case = Case([(0, 256, 3), (0, 256, 200), (1, 128, 9), (1, 128, 30)], 4, 2, 128, 16, seed=4)
    base = P.paged_attention(case.q, case.k, case.v, case.table, case.lengths, groups=case.groups())
    one = [r for r in range(4) if case.lengths[r] > 255]
    page = int(case.table[one[0], 5])
    for value in (math.nan, math.inf, -math.inf):
        keep = case.k[page, 3, 0].clone()
        case.k[page, 3, 0] = value
        got = P.paged_attention(case.q, case.k, case.v, case.table, case.lengths, groups=case.groups())
        for r in range(4):
            if r in one:
                assert got[r, :2].isnan().all() and torch.equal(got[r, 2:], base[r, 2:])
            else:
                assert torch.equal(got[r], base[r])
        case.k[page, 3, 0] = keep


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(value):
    """A shared position whose values are not finite: not in rows whose window leaves it out, nor in rows that end in front of it."""
    case = Case([(0, 256, n) for n in (1, 30, 100, 300)] + [(None, 0, 40)], 4, 2, 128, 16, seed=4)
    groups = case.groups()
    call = lambda **more: P.paged_attention(case.q, case.k, case.v, case.table, case.lengths, groups=groups, **more)  # noqa: E731
    inside = [r for r in range(5) if case.lengths[r] > 255]
    page = int(case.table[inside[0], 1])  # positions 16 to 31
    for window in (0, 250, 290, 400):
        want = call(window=window)
        keep = case.v[page, 4].clone()
        case.v[page, 4] = value
        got = call(window=window)
        for r in range(5):
            sees = r in inside and (window == 0 or int(case.lengths[r]) - window <= 20)
            assert got[r].isfinite().all() != sees and (sees or torch.equal(got[r], want[r])), (window, r)
        case.v[page, 4] = keep
    lengths = case.lengths.clone()
    case.lengths[inside[1]] = 20
    want = call()
    case.v[page, 4] = value
    got = call()
    assert torch.equal(got[inside[1]], want[inside[1]]) and not got[inside[0]].isfinite().any()
    case.lengths = lengths


def test_large_values():
    """Values near the end of bf16's range, with weights that grow along the row."""
    case = Case([(0, 256, n) for n in (1, 200)], 4, 2, 128, 16, seed=4)
    case.v.mul_(1e34)
    case.check()


def test_strides_and_out():
    """q and out inside wider rows, in place, a table with wider rows; nothing else is written."""
    case = Case([(0, 192, n) for n in (3, 50, 129)] + [(None, 0, 9)] * 2, 8, 2, 128, 24, seed=5)
    want = case.check()
    wide = torch.full((5, 12, 136), 7.0, device="cuda", dtype=BF)
    wide[:, 2:10, :128] = case.q
    table = torch.full((5, case.table.shape[1] + 3), -1, device="cuda", dtype=torch.int32)
    table[:, :-3] = case.table
    args = (case.k, case.v, table[:, :-3], case.lengths)
    out = torch.full((8, 5, 144), 3.0, device="cuda", dtype=BF)
    got = P.paged_attention(wide[:, 2:10, :128], *args, out=out.transpose(0, 1)[..., 8:136], groups=case.groups())
    assert torch.equal(got, want) and (out[..., :8] == 3).all() and (out[..., 136:] == 3).all()
    P.paged_attention(wide[:, 2:10, :128], *args, out=wide[:, 2:10, :128], groups=case.groups())
    assert torch.equal(wide[:, 2:10, :128], want) and (wide[:, :2] == 7).all() and (wide[:, 10:] == 7).all() and (wide[..., 128:] == 7).all()
    assert P.paged_attention(case.q[:0], case.k, case.v, case.table[:0], case.lengths[:0], groups=(_ints([]), _ints([0]), _ints([]))).shape == (0, 8, 128)


def test_same_bits_graph_stream_and_workspace():
    """The same bits every time: on another stream, with a workspace full of NaN, replayed with longer rows; two graphs with a workspace each."""
    case = Case([(0, 2048, n) for n in range(1, 60, 3)] + [(1, 512, 100)] * 9 + [(None, 0, 300)], 32, 8, 128, 16, seed=6)
    want = case.check()
    groups = case.groups()
    n = P.paged_attention_workspace_bytes(30, 32, 8, 128, case.table.shape[1] * 16, groups=True)
    spaces = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.empty_like(case.q) for _ in range(2)]
    call = lambda i: P.paged_attention(case.q, case.k, case.v, case.table, case.lengths, out=outs[i], groups=groups, workspace=spaces[i])  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graphs = []
        for i in range(2):
            call(i)
            assert torch.equal(outs[i], want)
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[i], stream=s):
                call(i)
        s.synchronize()
    other = torch.cuda.Stream()
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    case.lengths -= 1
    graphs[0].replay()
    case.check(groups=groups)
    assert torch.equal(outs[0], P.paged_attention(case.q, case.k, case.v, case.table, case.lengths, groups=groups))
    assert ops.gemm_error() == 0


def test_narrow_tables():
    """Rows that cannot be long are read each by itself, with the workspace that the call for groups asks for."""
    case = Case([(0, 320, n) for n in (7, 40, 100, 200)] + [(None, 0, 33)], 8, 2, 128, 16, seed=2)
    groups = case.groups()
    wide = case.check(groups=groups)
    case.table = case.table[:, :40].contiguous()
    space = torch.empty(P.paged_attention_workspace_bytes(5, 8, 2, 128, 640, groups=True), dtype=torch.uint8, device="cuda")
    narrow = case.check(groups=groups, workspace=space)
    assert torch.equal(narrow, P.paged_attention(case.q, case.k, case.v, case.table, case.lengths))
    assert (wide.float() - narrow.float()).norm() <= 4e-3 * narrow.float().norm()


def test_as_without_groups():
    """Near to the attention that reads every row by itself."""
    for cache, heads in ((BF, (32, 8, 128)), (HALF, (35, 7, 64)), (F8, (8, 1, 256))):
        case = Case([(0, 800, n) for n in range(1, 400, 41)] + [(None, 0, 64)], *heads, 16, cache, seed=8)
        a, b = (P.paged_attention(case.q, case.k, case.v, case.table, case.lengths, k_scale=case.scales[0], v_scale=case.scales[1], groups=g)
                for g in (None, case.groups()))
        assert (a.float() - b.float()).norm() <= 4e-3 * a.float().norm()


def test_long_rows():
    """Many tiles, and pieces of every CTA in one item."""
    Case([(0, 40000, n) for n in (1, 300)] + [(None, 0, 9000)], 4, 1, 128, 64, seed=7).check()
    Case([(0, 20000, n % 50 + 1) for n in range(70)], 8, 2, 64, 32, HALF, seed=7).check()
