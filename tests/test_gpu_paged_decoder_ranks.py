"""The paged decoder on two ranks, with a communicator that adds on the host's order: two threads, one GPU, no kernel waits for another."""
import threading

import pytest
import torch

import penny_b200.ops as P
from penny_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
WORLD = 2


class _Meeting:
    """Where the ranks' tensors meet."""

    def __init__(self):
        self.barrier, self.there = threading.Barrier(WORLD, timeout=60), [None] * WORLD


class _Comm:
    def __init__(self, meeting, rank):
        self.m, self.rank = meeting, rank

    def _all(self, x):
        self.m.there[self.rank] = x
        self.m.barrier.wait()
        got = [t.clone() for t in self.m.there]  # (before anyone writes its own)
        self.m.barrier.wait()
        return got

    def all_reduce(self, x, out):
        out.copy_(sum(t.float() for t in self._all(x)))

    def all_gather(self, x, out):
        out.copy_(torch.cat(self._all(x)))


def _ranks(f):
    """f(rank) on a thread for each rank."""
    said = [None] * WORLD

    def run(r):
        try:
            said[r] = (True, f(r))
        except BaseException as e:  # noqa: B036
            said[r] = (False, e)
    threads = [threading.Thread(target=run, args=(r,)) for r in range(WORLD)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for ok, what in said:
        if not ok:
            raise what
    return [what for _, what in said]


@pytest.mark.parametrize("linears,dtype,page", [("auto", torch.bfloat16, 16), ("cublas", torch.bfloat16, 24), ("auto", E4M3, 16)])
def test_two_ranks(linears, dtype, page):
    """Logits and tokens of two steps against fp32 on the whole model; a row without a page is the same one on both ranks."""
    cfg, B, kv = LlamaConfig.tiny(), 4, 100
    full = LlamaTPDecoder(cfg, world=1, max_batch=B, max_len=160, use_graph=False, full_init=True)
    full.fill_synthetic_kv(kv)
    meeting, hk = _Meeting(), cfg.kv_heads // WORLD
    ms = [LlamaTPDecoder(cfg, comm=_Comm(meeting, r), rank=r, world=WORLD, max_batch=B, max_len=160, backend="penny_unfused", use_graph=False, full_init=True,
                         linears=linears, page_size=page, pages=B * -(-(kv + 2) // page), cache_dtype=dtype) for r in range(WORLD)]
    for r, m in enumerate(ms):
        step = m.paged.advance(torch.full((B,), kv, dtype=torch.int32, device="cuda"), B * kv)
        assert step.granted.all()
        for li in range(cfg.layers):
            for pool, rows in ((m.paged.k[li], full.kcache[li]), (m.paged.v[li], full.vcache[li])):
                new = rows[:, r * hk:(r + 1) * hk, :kv].transpose(1, 2).reshape(B * kv, hk, -1).to(dtype)
                pool.view(torch.uint8).view(m.paged.pages * page, hk, -1)[step.slots] = new.contiguous().view(torch.uint8)
        m.tokens.copy_(full.tokens)
    V = cfg.vocab // WORLD
    for n in range(2):
        tokens, positions = ms[0].tokens.clone(), ms[0].positions.clone()
        assert torch.equal(ms[1].tokens, tokens) and (positions == kv + n).all()
        # both ranks' heads side by side, as they are stored
        caches = [[torch.stack([torch.cat([m.paged.rows_of(li, b, kv + n)[i] for m in ms]) for b in range(B)]) for li in range(cfg.layers)] for i in (0, 1)]
        want = full.reference_logits(tokens, positions, *caches)
        _ranks(lambda r: ms[r].step_device())
        for r, m in enumerate(ms):
            m.check_pages()
            assert (m.paged.lengths == kv + n + 1).all()
            err = (m.logits.float() - want[:, r * V:(r + 1) * V]).abs().max().item()
            assert err < 0.05 * want.std().item() + 0.02, (n, r, err)  # (the bound of the decoder's other tests)
        assert torch.equal(ms[0].next_tokens, ms[1].next_tokens) and torch.equal(ms[0].next_tokens, torch.cat([m.logits for m in ms], 1).float().argmax(-1))
    left = page * ms[0].paged.pages // B - (kv + 2)
    for _ in range(left):
        _ranks(lambda r: ms[r].step_device())
    for m in ms:
        m.check_pages()
    _ranks(lambda r: ms[r].step_device())
    rows = []
    for m in ms:
        with pytest.raises(P.OutOfPages) as said:
            m.check_pages()
        rows.append(said.value.rows)
    assert rows == [list(range(B))] * WORLD
