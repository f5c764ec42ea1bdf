"""A prompt's forward into pages says so when the step is not one prompt of a row that was empty."""
import pytest
import torch

import penny_b200.ops as P
from penny_b200.models.llama_sp import LlamaSPPrefill
from penny_b200.models.llama_tp import LlamaConfig
from penny_b200.parallel.comm import Communicator

pytestmark = pytest.mark.gpu


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_steps_that_are_no_prompt():
    cfg, T = LlamaConfig.tiny(), 256
    comm = Communicator.emulated(1, heap_bytes=64 << 20)
    try:
        m = LlamaSPPrefill(cfg, comm, tokens=T, layers=2)
        x = (torch.randn(T, cfg.hidden, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) * 0.5).bfloat16()
        cache = P.PagedKVCache(2, 4, 600, cfg.kv_heads, page_size=24)
        cache.advance(_ints(3, 0, 0, 0), 3)
        bad = [cache.advance(_ints(T, 0, 0, 0), T),            # behind three tokens that the row has
               cache.advance(_ints(0, 100, 156, 0), T),        # two prompts
               cache.advance(_ints(0, 0, 0, T - 1), T)]        # one token too few
        for step in bad:
            with pytest.raises(ValueError, match="one row that was empty"):
                m.forward(x, pages=(cache, step))
        cache.advance(-cache.lengths, 0)
        assert m.forward(x, pages=(cache, cache.advance(_ints(0, 0, T, 0), T))).equal(m.forward(x, pages=(cache, cache.advance(_ints(T, 0, 0, 0), T))))
    finally:
        comm.close()
