"""The paged decoder's rows: refused for want of a page, released, begun anew, empty at the start."""
import pytest
import torch

import penny_b200.ops as P
from penny_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _model(**kw):
    return LlamaTPDecoder(LlamaConfig.tiny(), world=1, full_init=True, **(dict(max_batch=3, max_len=64, page_size=16) | kw))


def _expected(m, tokens, positions):
    """fp32 logits of the step that has just been taken with `tokens` at `positions`, over what the cache holds."""
    B, L = len(positions), max(positions) + 1
    caches = []
    for i in (0, 1):
        caches.append([])
        for li in range(m.cfg.layers):
            rows = torch.zeros(B, m.Hkv, L, m.cfg.head_dim, device="cuda")
            for b, n in enumerate(positions):
                rows[b, :, :n] = m.paged.rows_of(li, b, n)[i]
            caches[-1].append(rows)
    return m.reference_logits(torch.tensor(tokens, device="cuda"), torch.tensor(positions, device="cuda"), *caches)


def _near(m, tokens, positions, rows):
    want = _expected(m, tokens, positions)
    err = (m.logits.float() - want).abs().amax(-1)
    assert (err[rows] < 0.05 * want.std() + 0.02).all(), err.tolist()  # (the bound of the decoder's other tests)


@pytest.mark.parametrize("graph", [True, False])
def test_a_refused_row_goes_on_when_there_are_pages(graph):
    """Two of three rows find no page: the third's token is handed over, the refused ones have not moved; one leaves, the other takes its
    token again, a new sequence begins in the free row."""
    m = _model(pages=7, use_graph=graph)
    m.fill_synthetic_kv(32)  # six pages of seven
    m.capture()
    with pytest.raises(P.OutOfPages, match="no page") as said:
        m.step(torch.tensor([11, 12, 13]))
    assert said.value.rows == [1, 2] and m.paged.lengths.tolist() == [33, 32, 32] and m.positions.tolist() == [33, 32, 32]
    _near(m, [11, 12, 13], [32, 32, 32], [0])
    first = int(said.value.next_tokens[0])
    assert first == int(m.logits[0].argmax())
    with pytest.raises(P.OutOfPages):  # still none: the same two, and the first row goes on
        m.step(torch.tensor([first, 12, 13]))
    second = int(m.logits[0].argmax())
    assert m.paged.lengths.tolist() == [34, 32, 32]
    m.release([2])
    assert m.paged.lengths.tolist() == [34, 32, 0] and m.positions.tolist() == [34, 32, 0] and int(m.paged.free_count) == 2
    out = m.step(torch.tensor([second, 12, 5])).tolist()
    assert m.paged.lengths.tolist() == [35, 33, 1] and int(m.paged.free_count) == 0
    _near(m, [second, 12, 5], [34, 32, 0], [0, 1, 2])
    assert out == m.logits.argmax(-1).tolist()
    before = m.paged.lengths.tolist()
    tokens = m.step(torch.tensor(out)).tolist()
    _near(m, out, before, [0, 1, 2])
    assert m.positions.tolist() == [n + 1 for n in before] and tokens == m.logits.argmax(-1).tolist()


def test_decode_hands_over_what_it_has():
    """decode() past the pool's end: every row's tokens up to the refused one, as far as its length says; check_pages says it once."""
    a, b = (_model(pages=n) for n in (7, 12))
    for m in (a, b):
        m.fill_synthetic_kv(30)
        m.capture()
    want = b.decode(6)
    with pytest.raises(P.OutOfPages) as said:
        a.decode(6)
    got, lengths = said.value.next_tokens, a.paged.lengths.tolist()
    assert got.shape == (6, 3) and lengths == [36, 32, 32] and said.value.rows == [1, 2]
    assert torch.equal(got[:2], want[:2])  # (both have had the same pages so far)
    a.check_pages()
    a.release([1, 2])
    assert a.paged.lengths.tolist() == [36, 0, 0]
    a.step_device()
    a.check_pages()


def test_release():
    m = _model(use_graph=False)
    m.fill_synthetic_kv(20)
    m.release([])
    assert m.paged.lengths.tolist() == [20] * 3
    m.release([0, 2, 2])
    assert m.paged.lengths.tolist() == [0, 20, 0] and int(m.paged.free_count) == m.paged.pages - 2
    for bad in ([3], [-1]):
        with pytest.raises(IndexError):
            m.release(bad)
    with pytest.raises(ValueError):
        LlamaTPDecoder(LlamaConfig.tiny(), world=1, max_batch=3, max_len=64, full_init=True).release([0])


@pytest.mark.parametrize("graph", [True, False])
def test_scales_of_an_8_bit_cache(graph):
    """Scales that are not one, a tensor for all layers or one for each: logits over what the cache holds, before and after a step."""
    cfg = LlamaConfig.tiny()
    g = torch.Generator(device="cuda").manual_seed(4)
    k = 0.01 + 0.02 * torch.rand(cfg.kv_heads, device="cuda", generator=g)
    v = [0.01 + 0.02 * torch.rand(cfg.kv_heads, device="cuda", generator=g) for _ in range(cfg.layers)]
    m = _model(cache_dtype=E4M3, cache_scales=(k, v), use_graph=graph)
    m.fill_synthetic_kv(40)
    assert m.paged.k_scale[1] is k and m.paged.v_scale[1] is v[1]
    for li in (0, 1):
        for t in m.paged.rows_of(li, 0, 40):  # normal values, 2 ** -4 of each at most from them: and not 50 times too small
            assert 0.9 < t.std() < 1.1 and t.abs().max() < 6
    m.capture()
    out = m.step(torch.tensor([3, 4, 5])).tolist()
    _near(m, [3, 4, 5], [40, 40, 40], [0, 1, 2])
    m.step(torch.tensor(out))
    _near(m, out, [41, 41, 41], [0, 1, 2])


def test_caches_that_the_decoder_cannot_have():
    one = torch.ones(LlamaConfig.tiny().kv_heads, device="cuda")
    for over in (dict(cache_dtype=torch.float16), dict(cache_dtype=torch.float32), dict(cache_scales=(one, one)), dict(cache_dtype=E4M3, cache_scales=(one, one[1:])),
                 dict(cache_dtype=E4M3, cache_scales=(one.double(), one)), dict(page_size=0, cache_scales=(one, one))):
        with pytest.raises(ValueError):
            _model(**over)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_empty_rows_at_the_start(dtype):
    """A cache that is filled with nothing: the first tokens are at position 0."""
    m = _model(cache_dtype=dtype, use_graph=False)
    m.fill_synthetic_kv(0)
    assert m.paged.lengths.tolist() == [0] * 3 and int(m.paged.free_count) == m.paged.pages
    m.step(torch.tensor([3, 4, 5]))
    # one position: the last layer's attention is its value, as it is stored (which in 8 bits is up to 2 ** -4 from the fp32 model's)
    value = torch.stack([m.paged.rows_of(m.cfg.layers - 1, b, 1)[1][:, 0] for b in range(3)])
    assert torch.equal(m.attn.view(3, m.Hkv, -1, m.cfg.head_dim).float(), value.float()[:, :, None].expand(-1, -1, m.Hq // m.Hkv, -1))
    if dtype == torch.bfloat16:
        _near(m, [3, 4, 5], [0] * 3, [0, 1, 2])
        m.step(torch.tensor([7, 8, 9]))
        _near(m, [7, 8, 9], [1] * 3, [0, 1, 2])
