"""Log probabilities of given tokens, entropy and top alternatives, against 64 bits."""
import math

import pytest
import torch

import penny_b200.ops as P

pytestmark = pytest.mark.gpu
INF = math.inf


def _want(x, tokens, top):
    """From the definition, in 64 bits; ties to the lowest id."""
    x = x.double()
    y = torch.log_softmax(x, -1)
    p = y.exp()
    entropy = -torch.where(p > 0, p * y, 0).sum(-1)
    ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    return y.gather(1, tokens[:, None])[:, 0], entropy, y.gather(1, ids), ids


def _check(x, tokens, top):
    got = P.token_logprobs(x, tokens, top)
    want = _want(x, tokens, top)
    assert got.top_ids.dtype == torch.int64 and torch.equal(got.top_ids, want[3])
    # x - m is rounded once (2^-24 of it), as is the result; log Z has the rounding of Z, of which a term exp2(y) is off by 2^-22 and by
    # what y is off: two roundings of at most 128 (smaller terms do not count), and the sums are trees of at most 2^6 steps a thread
    # and 13 more.  The entropy's terms are exp(y) y.
    part = 2.0 ** -22 + 128 * math.log(2) * 2 * 2.0 ** -24 + 80 * 2.0 ** -24
    for a, b in ((got.logprobs, want[0]), (got.top_logprobs, want[2])):
        assert torch.equal(a == -INF, b == -INF)
        b = b.masked_fill(b == -INF, 0)
        a = a.double().masked_fill(a == -INF, 0)
        assert ((a - b).abs() <= 3 * 2.0 ** -24 * (b.abs() + 20) + part).all(), (a - b).abs().max()
    assert ((got.entropy.double() - want[1]).abs() <= part * (1 + 128) + 2.0 ** -23 * 20).all()
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 0), (3, 5, 5), (2, 31, 20), (7, 33, 32), (5, 100, 1), (300, 1000, 7), (1, 4097, 32), (40, 16391, 20),
                                            (1, 128256, 20), (9, 128256, 0), (64, 128256, 20), (400, 32000, 5)])
def test_values(dtype, rows, vocab, top):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + vocab)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 4).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    _check(x, tokens, top)


@pytest.mark.parametrize("offset,stride", [(1, 5003), (3, 5000), (7, 5001), (0, 5008)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignments(dtype, offset, stride):
    big = (torch.randn(6 * stride + 16, device="cuda") * 4).to(dtype)
    for vocab in (4999, 17, 8, 3):
        x = big[offset:offset + 6 * stride].view(6, stride)[:, :vocab]
        _check(x, torch.tensor([0, vocab - 1, vocab // 2, 1, 2, 0], device="cuda"), 3)
    x = big[offset:offset + 4999].expand(5, 4999)  # one row of logits for all
    got = _check(x, torch.tensor([0, 4, 4998, 70, 4000], device="cuda"), 4)
    assert (got.top_ids == got.top_ids[0]).all()


@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "two values", "steps", "last", "signed zeros"])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (300, 20001)])
def test_orders(kind, rows, vocab):
    """Orders that make the lists run full, and ties."""
    i = torch.arange(vocab, device="cuda")
    x = {"ascending": i / vocab * 60 - 30, "descending": 30 - i / vocab * 60, "equal": i * 0 + 1.5, "two values": (i % 2) * 1.0, "steps": (i // 1000) * 0.25,
         "last": (i >= vocab - 40) * 3.0, "signed zeros": torch.where(i % 3 == 0, -0.0, 0.0)}[kind].float()
    for dtype in (torch.float32, torch.bfloat16):
        got = _check(x.to(dtype).expand(rows, vocab).contiguous(), (torch.arange(rows, device="cuda") * 977) % vocab, 32)
        assert torch.equal(got.top_ids, got.top_ids[:1].expand(rows, 32))


def test_masked_and_far_logits():
    """Tokens that cannot come, rows with only one, rows of nothing, infinities, NaN, tokens that the vocabulary does not have."""
    vocab = 3001
    x = torch.randn(9, vocab, device="cuda") * 3
    x[0, torch.rand(vocab, device="cuda") < 0.9] = -INF
    x[1] = -INF
    x[1, 2000] = 5.0
    x[2] = x[2] * 1e30
    x[3] = x[3] + 65000.0
    for dtype in (torch.float32, torch.bfloat16):
        y = x[:4].to(dtype)
        tokens = y.argmax(-1)
        tokens[0] = (y[0] == -INF).nonzero()[0, 0]
        got = _check(y, tokens, 20)
        assert got.logprobs[0] == -INF and got.logprobs[1] == 0 and got.entropy[1] == 0 and got.top_logprobs[1].tolist() == [0] + [-INF] * 19
        y = x.to(dtype)
        y[4] = -INF
        y[5, 17] = float("nan")
        y[6, 29] = INF
        y[7, :] = float("nan")
        tokens = torch.tensor([5, 5, 5, 5, 7, 3, 3, 3, -1], device="cuda")
        got = P.token_logprobs(y, tokens, 20)
        assert got.logprobs[4] == -INF and got.entropy[4] == 0 and got.top_logprobs[4].tolist() == [-INF] * 20 and got.top_ids[4].tolist() == list(range(20))
        for r in (5, 6, 7):
            assert got.logprobs[r].isnan() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all(), r
        assert got.logprobs[8].isnan() and not got.entropy[8].isnan() and not got.top_logprobs[8].isnan().any()
        for bad in (vocab, 2 ** 40, -2 ** 62):
            assert P.token_logprobs(y[:1], torch.tensor([bad], device="cuda")).logprobs.isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masks_of_the_lowest_value(dtype):
    """Tokens that are masked by the type's lowest number and not by minus infinity; rows of nothing else, and of its opposite."""
    for vocab in (5000, 128256):
        x = (torch.randn(6, vocab, device="cuda") * 3).to(dtype)
        lowest, highest = torch.finfo(dtype).min, torch.finfo(dtype).max
        x[0, torch.rand(vocab, device="cuda") < 0.9] = lowest
        x[1, 1:] = lowest
        x[2] = lowest
        x[3, 7] = highest
        x[4] = highest
        x[5, ::2] = lowest
        x[5, 1::4] = highest
        got = P.token_logprobs(x, torch.tensor([0, 0, 9, 7, 8, 1], device="cuda"), 5)
        want = _want(x, torch.tensor([0, 0, 9, 7, 8, 1], device="cuda"), 5)
        assert torch.equal(got.top_ids, want[3])
        flat = math.log(vocab)
        assert abs(got.entropy[2] - flat) < 1e-4 and abs(got.entropy[4] - flat) < 1e-4 and abs(got.logprobs[2] + flat) < 1e-4 and abs(got.logprobs[4] + flat) < 1e-4
        assert got.logprobs[1] == 0 and got.logprobs[3] == 0 and got.entropy[1] == 0 and got.entropy[3] == 0
        for a, b in zip(got[:3], want[:3]):
            far = b.abs() > 1e4  # (numbers of the type's size: as fp32 has them)
            assert ((a.double() - b).abs()[~far] < 1e-4).all() and (((a.double() - b) / b).abs()[far] < 2.0 ** -20).all() and not a.isnan().any()


def test_no_rows_graph_and_stream():
    assert [t.shape for t in P.token_logprobs(torch.zeros(0, 50, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), 3)] == [(0,), (0,), (0, 3), (0, 3)]
    x, tokens = torch.randn(5, 128256, device="cuda"), torch.arange(5, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        P.token_logprobs(x, tokens, 20)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = P.token_logprobs(x, tokens, 20)
        for _ in range(3):
            x.normal_()
            graph.replay()
            want = P.token_logprobs(x, tokens, 20)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        s.synchronize()
