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


def test_places_of_bad_pages_and_slots():
    place = schedule.page_place
    assert place(3, 4, 50, 16, 1000, 10) == 3 * 1000 + 2 * 10
    for page in (-1, 4, 5, -2 ** 31, 2 ** 31 - 1):
        assert place(page, 4, 50, 16, 1000, 10) == -1
    # offsets past 32 bits
    assert place(2 ** 21, 2 ** 21 + 1, 7, 16, 16 * 8 * 128 * 2, 8 * 128 * 2) == 2 ** 21 * 2 ** 15 + 7 * 2 ** 11
    at = schedule.slot_place
    assert at(3 * 24 + 5, 4, 24, 1000, 10) == 3050 and at(4 * 24 - 1, 4, 24, 1000, 10) == 3230
    for slot in (-1, -2 ** 63, 4 * 24, 2 ** 63 - 1, 2 ** 32):
        assert at(slot, 4, 24, 1000, 10) == -1
    assert at(2 ** 33 + 3, 2 ** 30, 16, 16, 1) == 2 ** 33 + 3


@pytest.mark.parametrize("max_len", [1, 255, 256, 511, 512, 1024, 4352, 100000, 2 ** 31 - 2 ** 16])
@pytest.mark.parametrize("items", [1, 2, 8, 20])
def test_every_piece_has_a_cta(max_len, items):
    rng = random.Random(max_len + items)
    for B in (1, 2, 3, 7, 37, 64, 130, 300, 1000):
        for window in (0, 1, 300, 5000):
            inside = [rng.randrange(max_len + 1) for _ in range(B)]
            edges = [max_len, 0, -1, -2 ** 31, 2 ** 31 - 1, max_len + 1]
            for lengths in [inside] + [[min(e, 2 ** 31 - 1)] * B for e in edges] + [[min(rng.choice(edges), 2 ** 31 - 1)] + inside[1:]]:
                seen, pieces, extra = schedule.paged_cut(lengths, items, max_len, window)
                for (first, end), n in zip(seen, lengths):
                    assert end == max(0, min(n, max_len)) and first == (max(0, end - window) if window else 0)
                assert all(1 <= p <= 128 for p in pieces)
                assert sum(pieces) * items <= B * items + extra  # every piece of every row has a CTA
                assert extra <= 296


def test_the_cut():
    assert schedule.paged_cut([200], 1, 4096)[1:] == ([1], 15)
    assert schedule.paged_cut([2048], 1, 4096)[1] == [8]
    assert schedule.paged_cut([100001] * 2, 8, 100032)[1] == [18, 18]
    assert schedule.paged_cut([2048] * 64, 8, 2560)[1] == [1] * 64       # the rows fill the GPU by themselves
    assert schedule.paged_cut([60000] + [100] * 63, 8, 65536)[1] == [33] + [1] * 63
    assert schedule.paged_cut([255] * 3, 8, 256)[2] == 0                  # no row can be cut: no second kernel
