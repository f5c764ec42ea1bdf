"""The paged KV cache where it is used: tables, appends and attention one after the other, the decoder's step, a prefill that leaves
its keys and values in pages."""
import math

import pytest
import torch

import penny_b200.ops as P
from penny_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page,dtype", [(16, torch.bfloat16), (5, torch.float16), (24, E4M3)])
def test_sequences_come_grow_and_leave(page, dtype):
    """A few sequences through several steps, prompts and single tokens mixed, one that leaves and one that takes its place; every row's
    attention against fp64 on tokens that are kept beside the cache."""
    heads, kv_heads, dim, rows = 8, 2, 64, 4
    kind = torch.bfloat16 if dtype == E4M3 else dtype
    cache = P.PagedKVCache(2, rows, 200, kv_heads, dim, page_size=page, pages=60 * 16 // page, dtype=dtype)
    if dtype == E4M3:
        cache.k_scale = cache.v_scale = [torch.full((kv_heads,), 1 / 64, device="cuda")] * 2
    kept = [[] for _ in range(rows)]  # per row: tokens' projections as stored
    g = torch.Generator(device="cuda").manual_seed(page)
    for new in ([17, 0, 40, 3], [1, 33, 1, 1], [1, 1, -41, 1], [1, 1, 90, 0], [1] * 4, [-2, 1, 1, 60]):
        total = sum(max(0, n) for n in new)
        step = cache.advance(_ints(new), total + 3)
        assert step.granted.all()
        qkv = torch.randn(total + 3, (heads + 2 * kv_heads) * dim, device="cuda", generator=g).to(kind)
        raw = qkv.clone()
        for layer in (0, 1):
            qkv.copy_(raw)
            cache.append(layer, qkv, step, heads, 1e4)
        at = 0
        for r, n in enumerate(new):
            if n < 0:
                del kept[r][n:]
            for _ in range(max(0, n)):
                kept[r].append(qkv[at].view(-1, dim)[heads:].double())
                at += 1
        assert cache.lengths.tolist() == [len(k) for k in kept]
        q = torch.randn(rows, heads, dim, device="cuda", generator=g).to(kind)
        for layer in (0, 1):
            out = cache.attend(layer, q)
            for r in range(rows):
                if not kept[r]:
                    assert (out[r] == 0).all()
                    continue
                kv = torch.stack(kept[r])
                want_k, want_v = kv[:, :kv_heads].transpose(0, 1), kv[:, kv_heads:].transpose(0, 1)
                k, v = (t.double() for t in cache.rows_of(layer, r, len(kept[r])))
                if dtype == E4M3:  # half a step of each value, 448 / 64 at most
                    assert ((k - want_k.clamp(-7, 7)).abs() <= 2.0 ** -4 * want_k.abs() * (1 + 2.0 ** -3) + 2.0 ** -16).all()
                else:
                    assert torch.equal(k, want_k) and torch.equal(v, want_v)
                k, v = (t.repeat_interleave(heads // kv_heads, 0) for t in (k, v))
                p = (torch.einsum("hd,htd->ht", q[r].double(), k) / math.sqrt(dim)).softmax(-1)
                o, size = torch.einsum("ht,htd->hd", p, v), torch.einsum("ht,htd->hd", p, v.abs())
                # (a weight and the output rounded to bf16 at the worst, and fp32's part in the scores)
                assert ((out[r].double() - o).abs() <= (2.0 ** -8 + 2.0 ** -12) * size + 2.0 ** -8 * o.abs()).all()


def _decoders(**kw):
    cfg = LlamaConfig.tiny()
    plain = LlamaTPDecoder(cfg, world=1, max_len=200, full_init=True, **{k: v for k, v in kw.items() if k in ("max_batch", "linears", "use_graph")})
    return plain, LlamaTPDecoder(cfg, world=1, max_len=200, full_init=True, **kw)


@pytest.mark.parametrize("linears,batch,page", [("auto", 5, 16), ("auto", 70, 24), ("cublas", 6, 1), ("penny", 3, 64)])
def test_decoder_step(linears, batch, page):
    """Logits of a step over pages and over contiguous caches, and both against fp32, for several steps across pages' ends."""
    plain, paged = _decoders(max_batch=batch, linears=linears, page_size=page)
    for m in (plain, paged):
        m.fill_synthetic_kv(150)
        m.capture()
    assert torch.equal(paged.paged.lengths, paged.positions)
    for step in range(4):
        tokens, positions = paged.tokens.clone(), paged.positions.clone()
        assert torch.equal(tokens, plain.tokens) or step > 0
        plain.tokens.copy_(tokens)
        plain.step_device()
        paged.step_device()
        paged.check_pages()
        assert torch.equal(paged.paged.lengths, positions + 1) and torch.equal(paged.positions, positions + 1)
        for b in (0, batch - 1):  # the same keys and values, but for the new tokens' rotation and rounding
            k, v = paged.paged.rows_of(1, b, 150)
            assert torch.equal(k, plain.kcache[1][b, :, :150]) and torch.equal(v, plain.vcache[1][b, :, :150])
        caches = [[torch.stack([paged.paged.rows_of(li, b, 151 + step)[i] for b in range(batch)]) for li in range(2)] for i in (0, 1)]
        want = paged.reference_logits(tokens, positions, *caches)
        for m in (plain, paged):
            assert (m.logits.float() - want).abs().max().item() < 0.05 * want.std().item() + 0.02, (step, m is paged)


def test_decoder_with_an_8_bit_cache():
    _, m = _decoders(max_batch=4, page_size=16, cache_dtype=E4M3)
    m.fill_synthetic_kv(100)
    m.capture()
    tokens, positions = m.tokens.clone(), m.positions.clone()
    m.step_device()
    caches = [[torch.stack([m.paged.rows_of(li, b, 101)[i] for b in range(4)]) for li in range(2)] for i in (0, 1)]
    want = m.reference_logits(tokens, positions, *caches)
    assert (m.logits.float() - want).abs().max().item() < 0.05 * want.std().item() + 0.02
    out = m.step(m.next_tokens.cpu())
    assert out.shape == (4,) and m.paged.lengths.tolist() == [102] * 4


def test_decoder_out_of_pages():
    """A pool that runs empty, and rows at their longest, are said; what the other rows have is theirs."""
    cfg = LlamaConfig.tiny()
    m = LlamaTPDecoder(cfg, world=1, max_batch=3, max_len=64, full_init=True, page_size=16, pages=7)
    m.fill_synthetic_kv(32)  # six pages of seven
    m.capture()
    assert m.paged.lengths.tolist() == [32] * 3 and int(m.paged.free_count) == 1
    with pytest.raises(RuntimeError, match="no page"):
        m.step(torch.tensor([1, 2, 3]))
    assert m.paged.lengths.tolist() == [33, 32, 32]
    m.fill_synthetic_kv(20)
    m.decode(12)
    with pytest.raises(RuntimeError, match="no page"):
        m.decode(1)
    long = LlamaTPDecoder(cfg, world=1, max_batch=2, max_len=48, full_init=True, page_size=16)
    long.fill_synthetic_kv(47)
    long.capture()
    long.decode(1)
    with pytest.raises(RuntimeError, match="no page"):
        long.step(torch.tensor([1, 2]))
    with pytest.raises(RuntimeError, match="do not hold"):
        LlamaTPDecoder(cfg, world=1, max_batch=3, max_len=64, full_init=True, page_size=16, pages=2).fill_synthetic_kv(32)
    with pytest.raises(ValueError):
        LlamaTPDecoder(cfg, world=1, max_batch=3, max_len=64, pages=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_prefill_into_pages(dtype):
    """A prompt's forward with pages gives the same rows as without, and the last token's attention over the pages is the one over the
    prompt's own keys and values."""
    from penny_b200.models.llama_sp import LlamaSPPrefill
    from penny_b200.parallel.comm import Communicator
    cfg, T = LlamaConfig.tiny(), 256
    comm = Communicator.emulated(1, heap_bytes=64 << 20)
    m = LlamaSPPrefill(cfg, comm, tokens=T, layers=2)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(T, cfg.hidden, device="cuda", generator=g) * 0.5).bfloat16()
    want = m.forward(x).clone()
    cache = P.PagedKVCache(2, 3, 400, cfg.kv_heads, page_size=24, dtype=dtype)
    cache.advance(_ints([30, 0, 0]), 30)
    step = cache.advance(_ints([0, T, 0]), T)
    got = m.forward(x, pages=(cache, step))
    # (angles of up to 256 rad: fast sines off by 2 ** -14 or so against exact ones, within bf16's rounding of q and k)
    ref = LlamaSPPrefill.reference_forward(cfg, x, 2)
    scale = ref.std().item()
    assert (got.float() - want.float()).abs().max().item() < 0.05 * scale and (got.float() - ref).abs().max().item() < 0.1 * scale
    D, G = 128, cfg.heads // cfg.kv_heads
    last = m.qkv.view(T, -1, D)
    k, v = (t.double() for t in cache.rows_of(1, 1, T))
    if dtype == torch.bfloat16:
        assert torch.equal(k.transpose(0, 1), last[:, cfg.heads:cfg.heads + cfg.kv_heads].double()) and torch.equal(v.transpose(0, 1), last[:, -cfg.kv_heads:].double())
    q = last[-1:, :cfg.heads].expand(3, -1, -1)
    out = cache.attend(1, q)
    s = torch.einsum("hgd,htd->hgt", last[-1, :cfg.heads].double().view(-1, G, D), k) / math.sqrt(D)
    p = s.softmax(-1)
    o, size = torch.einsum("hgt,htd->hgd", p, v), torch.einsum("hgt,htd->hgd", p, v.abs())
    assert ((out[1].double().view_as(o) - o).abs() <= (2.0 ** -8 + 2.0 ** -12) * size + 2.0 ** -8 * o.abs()).all()
    assert (out[2] == 0).all()
    with pytest.raises(RuntimeError, match="no pages"):
        m.forward(x, pages=(cache, cache.advance(_ints([0, T, 0]), T)))  # past the row's longest
    with pytest.raises(ValueError, match="a step of"):
        m.forward(x, pages=(cache, cache.advance(_ints([0, 0, 5]), 5)))
    assert m.forward(x).equal(want)
    comm.close()
