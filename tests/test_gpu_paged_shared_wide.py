"""The tests of attention over shared pages with tables so wide that the kernel for shared pages is what runs, whatever their rows hold."""
import functools

import pytest
import torch

import test_gpu_paged_shared as shared
import test_gpu_shared_decoder as decoder
from penny_b200.parallel import schedule
from test_gpu_paged_shared import *  # noqa: F401, F403  (its tests, which make `Case`s)

pytestmark = pytest.mark.gpu


class Wide(shared.Case):
    def __init__(self, *args, **more):
        super().__init__(*args, **more)
        size = self.k.element_size()
        rows, width = self.table.shape
        width = max(width, (560 << 20) // (rows * self.page * self.kv_heads * self.dim * 2 * size) + 1)
        table = torch.full((rows, width), -1, device="cuda", dtype=torch.int32)
        table[:, :self.table.shape[1]] = self.table
        self.table = table
        assert schedule.shared_pays(rows, width * self.page, self.kv_heads, self.dim, size)
        assert schedule.shared_fits(rows, self.kv_heads, self.heads // self.kv_heads, width * self.page, self.dim)


@pytest.fixture(autouse=True)
def wide(monkeypatch):
    monkeypatch.setattr(shared, "Case", Wide)


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_decoder(use_graph, cache_dtype, monkeypatch):
    assert schedule.shared_pays(8, 160000, 2, 128, 1)
    monkeypatch.setattr(decoder, "_model", functools.partial(decoder._model, max_len=160000))
    decoder.test_forks_go_on_as_rows_of_their_own(use_graph, cache_dtype)


del Case  # noqa: F821  (not this file's)
