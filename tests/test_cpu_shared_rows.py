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
