"""A decoder whose rows are forked, on two ranks: two threads, one GPU, no kernel waits for another."""
import pytest
import torch

import penny_b200.ops as P
from penny_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder
from test_gpu_paged_decoder_ranks import WORLD, _Comm, _Meeting, _ranks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_len", [160, 300000])  # (each row by itself; the kernel for shared pages)
def test_two_ranks(max_len):
    """Forks, steps and log probabilities of both ranks against fp32 on the whole model; a fork without a page is the same one on both."""
    cfg, B, page, lengths = LlamaConfig.tiny(), 6, 16, [100, 37, 0, 0, 0, 0]
    full = LlamaTPDecoder(cfg, world=1, max_batch=B, max_len=160, use_graph=False, full_init=True)
    full.fill_synthetic_kv(100)
    meeting, hk = _Meeting(), cfg.kv_heads // WORLD
    ms = [LlamaTPDecoder(cfg, comm=_Comm(meeting, r), rank=r, world=WORLD, max_batch=B, max_len=max_len, backend="penny_unfused", use_graph=False, full_init=True,
                         page_size=page, pages=14, sharing=True) for r in range(WORLD)]
    for r, m in enumerate(ms):
        step = m.paged.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"), sum(lengths))
        assert step.granted.all()
        for li in range(cfg.layers):
            for pool, rows in ((m.paged.k[li], full.kcache[li]), (m.paged.v[li], full.vcache[li])):
                new = torch.cat([rows[b, r * hk:(r + 1) * hk, :n].transpose(0, 1) for b, n in enumerate(lengths)])
                pool.view(m.paged.pages * page, hk, -1)[step.slots] = new
        m.tokens.copy_(full.tokens)
    # 10 of 14 pages are taken, three forks need one each (the rest of 100 or 37 positions), the last has none
    for m in ms:
        m.fork([0, 1, 0], [2, 4, 5])
        with pytest.raises(P.OutOfPages) as said:
            m.fork([0, 1], [3, 0])
        assert said.value.rows == [0] and m.paged.lengths.tolist() == [100, 37, 100, 100, 37, 100] and int(m.paged.free_count) == 0
        assert m.paged.groups().shared.tolist() == [96, 32, 96, 96, 32, 96]
    tokens = torch.tensor([3, 500, 2000, 77, 1, 1024], device="cuda")
    for n in range(3):
        positions = ms[0].positions.clone()
        assert torch.equal(ms[1].positions, positions)
        caches = [[[torch.cat([m.paged.rows_of(li, b, int(p))[i] for m in ms]) for b, p in enumerate(positions)] for li in range(cfg.layers)] for i in (0, 1)]
        pad = [[torch.stack([torch.nn.functional.pad(c, (0, 0, 0, 160 - c.shape[1])) for c in layer]) for layer in kind] for kind in caches]
        want = full.reference_logits(tokens, positions, *pad)
        for m in ms:
            m.tokens.copy_(tokens)
        _ranks(lambda r: ms[r].step_device())
        logits = torch.cat([m.logits for m in ms], 1).float()
        assert (logits - want).abs().max() < 0.05 * want.std() + 0.02, n  # (the bound of the decoder's other tests)
        for m in ms:
            m.check_pages()
        tokens = (tokens * 7 + 11) % cfg.vocab
        for chosen in (None, tokens):
            got = _ranks(lambda r: ms[r].logprobs(5, chosen))
            assert all(torch.equal(a, b) for a, b in zip(*got))
            exact = torch.log_softmax(logits.double(), -1)
            taken = logits.argmax(-1) if chosen is None else chosen
            assert (got[0].logprobs.double() - exact.gather(1, taken[:, None])[:, 0]).abs().max() < 1e-5
            assert torch.equal(got[0].top_ids, logits.sort(dim=-1, descending=True, stable=True).indices[:, :5])
