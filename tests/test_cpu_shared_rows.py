"""Which positions a row of a group takes from what the group shares, and which it reads by itself: all that it sees, once (no GPU)."""
import pytest

from penny_b200.parallel import schedule


@pytest.mark.parametrize("max_len", [5, 12, 1000])
def test_every_position_once(max_len):
    for length in range(-1, 15):
        for shared in range(15):
            for window in range(16):
                end = min(max(length, 0), max_len)
                sees = list(range(max(0, end - window) if window else 0, end))
                group, own = schedule.shared_row(length, shared, max_len, window)
                assert list(range(*group)) + list(range(*own)) == sees, (length, shared, window)
    for n in (16, 2048, 4096):  # cut back to what is shared, of which the window leaves out nothing
        assert schedule.shared_row(n, n, 8192, n) == ((0, n), (n, n))
        assert schedule.shared_row(n + 1, n, 8192, n)[1] == (1, n + 1) and schedule.shared_row(n, n, 8192, n - 1)[1] == (1, n)
    assert schedule.shared_row(2 ** 31 - 1, 2 ** 31 - 1, max_len, 0) == ((0, 0), (0, max_len))


def test_tables_that_the_line_cannot_hold():
    for rows, heads, group, positions, dim in ((1024, 32, 1, 1 << 20, 128), (64, 8, 4, 8192, 128), (8192, 8, 4, 2 ** 31 - 65536, 64), (8192, 1, 200, 400, 256), (300, 2, 7, 1 << 17, 64)):
        tile, most = (128, 256) if dim <= 128 else (64, 128)
        assert schedule.shared_fits(rows, heads, group, positions, dim) == (schedule.shared_most_units(rows, heads, group, positions, tile, most) <= 1 << 30)
    assert not schedule.shared_fits(1024, 32, 1, 1 << 20, 128) and schedule.shared_fits(1024, 32, 1, 1 << 19, 128)
    assert not schedule.shared_fits(1, 65536, 1, 16, 64)  # (heads are a dimension of a grid)


def test_what_is_read_each_row_by_itself():
    """Sizes at which the kernel for shared pages was timed on both sides: us with / without."""
    for rows, positions, kv_heads, dim, size, pays in ((64, 8292, 1, 128, 2, False),   # 50.5 / 30.2
                                                       (16, 8292, 8, 128, 1, False), (64, 2112, 8, 128, 1, False), (64, 2548, 8, 128, 1, False),  # 64.7 / 47.5
                                                       (16, 8292, 8, 128, 2, True), (64, 2112, 8, 128, 2, True), (64, 8292, 8, 128, 2, True),  # 48.1 / 164.9
                                                       (64, 8292, 8, 128, 1, True), (16, 8292, 20, 64, 2, True), (4, 220, 1, 128, 2, False)):
        assert schedule.shared_pays(rows, positions, kv_heads, dim, size) == pays, (rows, positions)
    # (the bound itself, and more bytes than 64 bits hold: heads may be one head's memory)
    assert not schedule.shared_pays(64, 2048, 8, 128, 2) and schedule.shared_pays(64, 2049, 8, 128, 2)
    assert schedule.shared_pays(8192, 2 ** 31 - 65536, 2 ** 19, 256, 2) and schedule.shared_pays(8192, 2 ** 30, 2 ** 13, 256, 2)
