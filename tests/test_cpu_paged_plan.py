"""Index arithmetic of the paged KV cache: pages of positions, places of bad pages and slots, the cut of rows (no GPU)."""
import random

import pytest

from penny_b200.parallel import schedule


@pytest.mark.parametrize("size", [1, 2, 3, 5, 7, 16, 24, 32, 63, 64, 65, 100, 1000, 4097, 65535, 2 ** 20 + 1, 2 ** 30 - 1])
def test_page_of_a_position(size):
    rng = random.Random(size)
    top = 2 ** 31 - 1
    for n in [0, 1, top, top - 1, top // size * size, top // size * size - 1] + [rng.randrange(top) for _ in range(200)]:
        for m in {n, max(0, n // size * size - 1), n // size * size}:
            assert schedule.page_div(size, m) == m // size
    for n in (-5, 0, 1, size - 1, size, size + 1, 5 * size, 5 * size + 1):
        if n <= top:
            assert schedule.pages_of(size, n) == max(0, -(-n // size))


def test_places_of_bad_slots():
    at = schedule.slot_place
    assert at(3 * 24 + 5, 4, 24, 1000, 10) == 3050 and at(4 * 24 - 1, 4, 24, 1000, 10) == 3230
    for slot in (-1, -2 ** 63, 4 * 24, 2 ** 63 - 1, 2 ** 32):
        assert at(slot, 4, 24, 1000, 10) == -1
    assert at(2 ** 33 + 3, 2 ** 30, 16, 16, 1) == 2 ** 33 + 3


@pytest.mark.parametrize("pages,page,page_stride,pos_stride,size", [
    (100, 16, 16 * 8 * 128, 8 * 128, 2), (100, 16, 16 * 8 * 128, 128, 2), (7, 24, 24 * 64 + 16, 64, 1), (1, 5, 12345, 64, 1), (1, 1, 3, 5, 2), (5, 1, 8, 999, 2),
    (2 ** 22, 16, 16 * 1024, 1024, 2), (2 ** 15, 16, 80 * 2 * 16 * 1024, 1024, 2), (3, 16, 0, 64, 2)])
def test_steps(pages, page, page_stride, pos_stride, size):
    unit, a, b = schedule.page_steps(pages, page, page_stride, pos_stride, size)
    rng = random.Random(pages)
    for pg in {0, pages - 1, rng.randrange(pages)}:
        for pos in (0, page - 1, 3 * page + page // 2):
            at = schedule.page_step_of(pg, pages, pos, page, a, b)
            assert at * unit == (pg * page_stride + pos % page * pos_stride) * size
    for pg in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        assert schedule.page_step_of(pg, pages, 0, page, a, b) is None


def test_no_steps():
    assert schedule.page_steps(2 ** 31 - 1, 16, 16 * 24 + 8, 24, 2) is None      # 16 bytes divide the strides: 64 GB at most
    assert schedule.page_steps(2 ** 26, 16, 16 * 24, 24, 2)[0] == 16


def _walks(lengths, max_len, teams, window, tile=16):
    """Every warp's walk, and that together they are the batch: every tile once, whole rows finished by one warp, the others by a warp
    that begins them, warps in the middle and one that ends them."""
    per, warps = 4, 4 * teams
    seen = [(max(0, min(n, max_len) - window) if window else 0, max(0, min(n, max_len))) for n in lengths]
    tiles = [-(-(b - a) // tile) for a, b in seen]
    covered, empties, open_row, counts = {}, set(), None, {}
    line = [0]
    for n in tiles:
        line.append(line[-1] + (n + 3 if n else 1))  # three units for a row's start, one for an empty row
    for w in range(warps):
        parts, starts, share = schedule.paged_walk(lengths, max_len, warps, w, window, tile)
        assert starts == [seen[r][0] + tile * i for r, a, b, *_ in parts for i in range(a, b)]
        real = [p for p in parts if p[2] > p[1] or p[5]]
        for k, (r, a, b, begins, ends, empty, behind) in enumerate(real):
            if empty:
                assert tiles[r] == 0 and r not in empties and begins and ends
                empties.add(r)
                continue
            assert covered.get(r, 0) == a and b <= tiles[r] and begins == (a == 0) and ends == (b == tiles[r]) and behind == tiles[r] - b
            covered[r] = b
            assert begins or k == 0                 # one part of an earlier row, the first
            assert ends or k == len(real) - 1       # one part of a later row, the last
            if not begins:
                assert open_row == r
            open_row = None if ends else r
            if begins and not ends:
                # teams that follow, as the joining kernel counts them from the line alone
                begin = w // per * per * share
                counts[r] = (w // per, schedule.paged_teams_behind(begin, begin + per * share, line[r], line[r + 1] - line[r]) if begin + per * share < line[-1] else 0)
            if ends and not begins:
                first, later = counts[r]
                assert first + later == w // per
            if begins:
                # the team of a row's first tile, and those that follow, as the joining kernel counts them for each row
                each = per * share
                team = (line[r] + 3) // each
                assert team == w // per
                later = schedule.paged_teams_behind(team * each, (team + 1) * each, line[r], line[r + 1] - line[r])
                assert (later == 0) == (line[r + 1] <= (team + 1) * each) and team + later == (line[r + 1] - 1) // each
    assert open_row is None
    for team in range(teams):  # and a team that begins no row across its end is not taken for one
        begin, end = team * per * share, (team + 1) * per * share
        if end < line[-1]:
            r = max(i for i, x in enumerate(line[:-1]) if x <= end)
            if schedule.paged_teams_behind(begin, end, line[r], line[r + 1] - line[r]):
                assert counts[r][0] == team and counts[r][1] > 0
    assert all(covered.get(r, 0) == tiles[r] for r in range(len(lengths)))
    assert empties == {r for r in range(len(lengths)) if tiles[r] == 0}


@pytest.mark.parametrize("teams", [1, 2, 37])
@pytest.mark.parametrize("window", [0, 1, 100])
def test_every_tile_once(teams, window):
    rng = random.Random(teams)
    top = 2 ** 31 - 1
    for B in (1, 2, 5, 40):
        for max_len in (1, 17, 300, 5000):
            inside = [rng.randrange(max_len + 1) for _ in range(B)]
            for lengths in (inside, [0] * B, [max_len] * B, [top] * B, [-1] + inside[1:], [-2 ** 31] * (B - 1) + [max_len], [max_len] + [1] * (B - 1)):
                _walks(lengths, max_len, teams, window, tile=rng.choice([16, 32, 64]))


def test_teams():
    assert schedule.paged_teams(64, 8, 131) == 37 and schedule.paged_teams(1, 1, 19) == 1 and schedule.paged_teams(1, 1, 20) == 2
    assert schedule.paged_teams(1, 8, 131) == 8 and schedule.paged_teams(5, 3, 1) == 1
    for items in list(range(1, 400)) + [1000, 4096]:
        teams = schedule.paged_teams(1000, items, 1000)
        ctas = teams * items
        assert teams >= 1 and ctas <= max(items, 8 * 296)
        rounds = -(-ctas // 296)
        assert ctas >= 0.85 * rounds * 296 or items > 8 * 296  # the GPU is filled
