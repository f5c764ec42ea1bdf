"""Outputs of the paged operators that share memory with what a call reads: refused, without a GPU; what only lies between is not."""
import random

import pytest
import torch

import penny_b200.ops as P

BF = torch.bfloat16
ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def _attend(q, out):
    k = torch.zeros(6, 16, 2, 64, dtype=BF)
    P.paged_attention(q, k, k.clone(), ints(q.shape[0], 4), ints(q.shape[0]), out=out)


def _views(n, *offsets_sizes_strides):
    flat = torch.zeros(n, dtype=BF)
    return [flat.as_strided(size, stride, offset) for offset, size, stride in offsets_sizes_strides]


SIZE = (3, 4, 64)


@pytest.mark.parametrize("a,b", [
    ((0, SIZE, (256, 64, 1)), (64, SIZE, (256, 64, 1))), ((256, SIZE, (256, 64, 1)), (0, SIZE, (256, 64, 1))),     # a head, a row further
    ((0, SIZE, (256, 64, 1)), (8, SIZE, (256, 64, 1))), ((0, SIZE, (512, 64, 1)), (192, SIZE, (512, 64, 1))),      # a few values; the last head
    ((0, SIZE, (512, 128, 1)), (568, SIZE, (512, 128, 1))), ((0, SIZE, (256, 64, 1)), (0, SIZE, (64, 192, 1))),     # between heads but for 8; other order
    ((0, SIZE, (256, 64, 1)), (704, SIZE, (512, 64, 1))), ((0, SIZE, (0, 64, 1)), (128, SIZE, (256, 64, 1))),       # other strides; q of one row for all
    ((0, (1, 4, 64), (8, 64, 1)), (192, (1, 4, 64), (999, 64, 1))), ((0, (4, 4, 64), (256, 64, 1)), (0, (4, 4, 64), (64, 256, 1))),  # rows for heads
])
def test_attention_out_across_q(a, b):
    q, out = _views(4096, a, b)
    with pytest.raises(RuntimeError, match="out is q, or apart from it"):
        _attend(q, out)


@pytest.mark.parametrize("a,b", [
    ((0, SIZE, (256, 64, 1)), (0, SIZE, (256, 64, 1))), ((0, SIZE, (512, 64, 1)), (256, SIZE, (512, 64, 1))),       # in place; beside in the rows
    ((256, SIZE, (512, 64, 1)), (0, SIZE, (512, 64, 1))), ((0, SIZE, (512, 128, 1)), (64, SIZE, (512, 128, 1))),    # the other side; between heads
    ((0, SIZE, (512, 128, 1)), (576, SIZE, (512, 128, 1))), ((0, SIZE, (256, 64, 1)), (768, SIZE, (512, 64, 1))),   # a row further; behind
    ((0, SIZE, (1024, 64, 1)), (256, SIZE, (256, 64, 1))), ((0, (1, 4, 64), (8, 64, 1)), (0, (1, 4, 64), (999, 64, 1))),  # within a row; one row
])
def test_attention_out_beside_q(a, b):
    q, out = _views(4096, a, b)
    with pytest.raises(RuntimeError, match="CUDA"):  # (past every check of the host but the last)
        _attend(q, out)


def test_attention_out_and_q_at_random():
    """Layouts within and across each other, against the sets of elements."""
    rng, n, met = random.Random(3), 0, 0
    flat, index = torch.zeros(8000, dtype=BF), torch.arange(8000)
    for _ in range(3000):
        B, H, D = rng.randint(1, 4), rng.choice([2, 4]), 64
        lay = lambda: rng.choice([(H * D, D), (2 * H * D, D), (H * 2 * D, 2 * D), (D, B * D), (D, 2 * B * D), (H * D + 8, D),  # noqa: E731
                                  (rng.randrange(8, 600, 8), rng.randrange(8, 300, 8))])
        first = lay()
        views = [((B, H, D), (*s, 1), rng.randrange(0, 1600, 8)) for s in (first, first if rng.random() < 0.6 else lay())]
        q, out = (flat.as_strided(*v) for v in views)
        at_q, at_out = (index.as_strided(*v) for v in views)
        if at_out.unique().numel() < at_out.numel():
            continue
        across = bool(torch.isin(at_q, at_out).any()) and not torch.equal(at_q, at_out)
        with pytest.raises(RuntimeError) as said:
            _attend(q, out)
        if "its rows apart" in str(said.value):
            continue
        assert ("apart from it" in str(said.value)) == across, views
        n, met = n + 1, met + across
    assert n > 1000 and 200 < met < n - 200


def _append(qkv, out, k=None, v=None):
    k = torch.zeros(6, 16, 2, 64, dtype=BF) if k is None else k
    P.paged_append(qkv, k, torch.zeros_like(k) if v is None else v, torch.zeros(qkv.shape[0], dtype=torch.int64), ints(qkv.shape[0]), 4, 1e4, out=out)


def test_append_out_across_qkv():
    for offset, stride in ((64, 512), (512, 512), (128, 1024), (640, 512)):
        qkv, out = _views(8192, (0, (3, 512), (stride, 1)), (offset, (3, 384), (stride, 1)))
        with pytest.raises(RuntimeError, match="out is the start of qkv's rows, or apart"):
            _append(qkv, out)
    for a, b in (((0, (3, 512), (1024, 1)), (512, (3, 384), (1024, 1))), ((0, (3, 512), (512, 1)), (0, (3, 384), (512, 1))), ((0, (1, 512), (8, 1)), (512, (1, 384), (8, 1)))):
        with pytest.raises(RuntimeError, match="CUDA"):
            _append(*_views(8192, a, b))


def test_append_k_across_v():
    pool = torch.zeros(6, 16, 2, 2, 64, dtype=BF)
    qkv = torch.zeros(3, 512, dtype=BF)
    for k, v in ((pool[:, :, 0], pool[:, :, 0]), (pool[:5, :, 0], pool[1:, :, 0]), (pool[:, :8, 0], pool[:, 4:12, 0])):
        with pytest.raises(RuntimeError, match="k apart from v"):
            _append(qkv, None, k, v)
    flat = torch.zeros(6, 16, 2, 64, dtype=BF)
    for k, v in ((pool[:, :, 0], pool[:, :, 1]), (pool[:, :8, 0], pool[:, 8:, 0]), (flat[:3], flat[3:]), (pool[..., 0, :], pool[..., 1, :]), (pool[:, :, 0, :, :32], pool[:, :, 0, :, 32:])):
        with pytest.raises(RuntimeError, match="CUDA"):
            _append(qkv[:, :8 * k.shape[3]], None, k, v)


def test_tables_of_their_own():
    def call(**over):
        a = dict(table=ints(3, 4), lengths=ints(3), free=ints(10), free_count=ints(1), new=ints(3), page_size=16, tokens=8, out=None) | over
        P.page_tables(**a)
    flat = ints(64)
    slots = torch.zeros(16, dtype=torch.int64)
    step = lambda **o: tuple((dict(slots=slots[:8], positions=ints(8), offsets=ints(4), granted=torch.zeros(3, dtype=torch.bool)) | o).values())  # noqa: E731
    for over in (dict(lengths=flat[:3], new=flat[2:5]), dict(free=flat[:10], new=flat[9:12]), dict(free_count=flat[1:2], new=flat[:3]), dict(table=flat[:12].view(3, 4), new=flat[8:11]),
                 dict(lengths=flat[:3], free=flat[1:11]), dict(new=flat[:3], out=step(positions=flat[:8])), dict(lengths=flat[:3], out=step(offsets=flat[2:6])),
                 dict(out=step(positions=slots.view(torch.int32)[8:16])), dict(out=step(granted=slots.view(torch.bool)[:3]))):
        with pytest.raises(RuntimeError, match="of their own"):
            call(**over)
    for over in (dict(lengths=flat[:3], new=flat[3:6], free=flat[6:16], free_count=flat[16:17], table=flat[20:32].view(3, 4), out=step(positions=flat[32:40], offsets=flat[40:44])),
                 dict(tokens=0, out=step(slots=slots[:0], positions=flat[:0])), dict(table=flat[:24].view(3, 8)[:, :4], lengths=flat[24:27])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(**over)
