"""How attention over shared pages is dealt out: every tile to one CTA, and found again by the join (no GPU)."""
import random

import pytest

from penny_b200.parallel import schedule


@pytest.mark.parametrize("ctas", [1, 2, 7, 148])
def test_every_tile_once(ctas):
    rng = random.Random(ctas)
    for trial in range(60):
        items = [(rng.choice([1, 2, 3, 5, 40, rng.randint(1, 1000)]), rng.random() < 0.5) for _ in range(rng.choice([1, 2, 30, 300]))]
        line = [0]
        for n, pair in items:
            line.append(line[-1] + schedule.shared_units(n, pair))
        share = schedule.shared_share(line[-1], ctas)
        assert share * ctas >= line[-1]
        rests = {}
        for begin, (tiles, pair) in zip(line, items):
            first, last = schedule.shared_cta_of(begin, 0, pair, share), schedule.shared_cta_of(begin, tiles - 1, pair, share)
            assert 0 <= first <= last < ctas
            at = 0
            for cta in range(first, last + 1):
                a, b = schedule.shared_piece(begin, tiles, pair, share, cta)
                assert a == at and b > a
                at = b
                if a > 0:  # a piece that does not begin its item: one to a CTA, its first
                    rests[cta] = rests.get(cta, 0) + 1
                    assert begin < cta * share
            assert at == tiles
            for cta in {max(0, first - 1), min(ctas - 1, last + 1)} - set(range(first, last + 1)):
                a, b = schedule.shared_piece(begin, tiles, pair, share, cta)
                assert a == b
        assert all(n == 1 for n in rests.values())


def test_ends():
    assert schedule.shared_units(0, True) == schedule.shared_units(0, False) == 0 and schedule.shared_share(1, 148) == schedule.shared_share(2, 148)
    for pair in (False, True):
        top = (1 << 30) // 3 - 1
        share = schedule.shared_share(schedule.shared_units(top, pair), 148)
        assert schedule.shared_piece(0, top, pair, share, 147)[1] == top and schedule.shared_cta_of(0, top - 1, pair, share) == 147
    # what all rows can need is no more than the bound that a launch goes by
    assert schedule.shared_most_units(8192, 8, 4, 2 ** 31 - 1, 128, 256) > 2 ** 30
    rng = random.Random(1)
    for _ in range(200):
        rows, heads, group, most, tile = rng.randint(1, 50), rng.randint(1, 9), rng.choice([1, 4, 7, 64, 200]), rng.choice([128, 256]), rng.choice([64, 128])
        length, units, left = rng.randint(1, 3000), 0, rows
        while left:
            n = rng.randint(1, left)
            left -= n
            shared = rng.randint(0, length) if n > 1 else 0
            units += heads * -(-n * group // most) * schedule.shared_units(-(-shared // tile), most > 128 and n * group > 128)
            units += sum(heads * -(-group // most) * schedule.shared_units(-(-rng.randint(0, length - shared) // tile), most > 128 and group > 128) for _ in range(n))
        assert units <= schedule.shared_most_units(rows, heads, group, length, tile, most)
