"""The serving operators at the ends of their ranges: head sizes of every multiple of 16 bytes, large and
odd pages, pages inside heads, offsets past 32 bits, batches and calls of more sequences than a planning
block has threads, and logits of more than 2^31 elements. Bounds are those of
tests/test_attention_exact.py and tests/test_logprob_many_rows.py."""

from __future__ import annotations

import numpy as np
import pytest

from ptxgen import attention, logprob
from ptxgen.cache import CacheError, PagedCache
from test_attention import TYPES, Batch
from test_attention_exact import _hold, _moments


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


def _ints(x):
    import torch

    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# one token, a few, many (400 rows a sequence and more)
SHAPES = [([300, 1, 0, 77], [1, 1, 1, 1]), ([300, 17, 5], [3, 2, 6]), ([700, 450], [230, 210])]


def _tiles(news, group):
    """Whether f32 may go by the kernel that adds in order, and 16 bits by rounded weights."""
    return sum(news) * group > 48 * len(news)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news", SHAPES)
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 56, 72, 104, 120, 136, 200, 248])
@pytest.mark.parametrize("dtype", TYPES)
def test_head_sizes(ws, dtype, dim, lens, news) -> None:
    dim = dim // 2 if dtype == "float32" and dim < 128 else dim  # 4, 12, 20, ... of f32
    b = Batch(lens, news, 2, 2, dim, 16, dtype)
    _hold(b, b.run(ws), _moments(b), _tiles(news, 2), fma=dim > 128 or _tiles(news, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news", SHAPES)
@pytest.mark.parametrize("page", [2, 9, 40, 48, 256, 384, 1000])
@pytest.mark.parametrize("dtype", TYPES)
def test_pages(ws, dtype, page, lens, news) -> None:
    b = Batch(lens, news, 1, 3, 64, page, dtype)
    got = b.run(ws, window=250, sinks=11)
    _hold(b, got, _moments(b, 250, 11), _tiles(news, 3), fma=_tiles(news, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news", SHAPES)
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("dtype", TYPES)
def test_pages_inside_heads(ws, dtype, page, lens, news) -> None:
    """Each head's pages one after another, and rows of q and out with gaps."""
    import torch

    b = Batch(lens, news, 3, 2, 64, page, dtype, fused=True)
    k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (b.k, b.v))
    assert k.stride(1) > k.stride(0)
    out = torch.full((b.q.shape[0], 9, 72), 5.0, device="cuda", dtype=b.dtype)
    got = attention.prompt(b.q, b.starts, k, v, b.table, b.lens_t, workspace=ws, out=out[:, 1:7, :64])
    assert torch.equal(got, b.run(ws))
    assert (out[:, 0] == 5).all() and (out[:, 7:] == 5).all() and (out[:, :, 64:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news", SHAPES)
@pytest.mark.parametrize("dim,dtype,page", [(128, "bfloat16", 16), (128, "float16", 12),
                                            (128, "float32", 16), (256, "bfloat16", 16)])
def test_offsets_past_32_bits(ws, dim, dtype, page, lens, news) -> None:
    """A layer's keys of more than 4 GB, the sequences in its last pages: as from a small cache."""
    import torch

    b = Batch(lens, news, 2, 2, dim, page, dtype, junk=0.0)
    n = b.k.shape[0]
    each = b.k[0].numel() * b.k.element_size()
    total = (9 << 29) // each + n
    k, v = (torch.zeros((total, *t.shape[1:]), dtype=t.dtype, device="cuda") for t in (b.k, b.v))
    k[total - n:] = b.k
    v[total - n:] = b.v
    held = (torch.arange(b.table.shape[1], device="cuda")[None] * page) < b.lens_t[:, None]
    table = torch.where(held, b.table + (total - n), b.table)
    got = attention.prompt(b.q, b.starts, k, v, table, b.lens_t, workspace=ws)
    assert torch.equal(got, b.run(ws))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_more_sequences_than_threads(ws, dtype) -> None:
    rng = np.random.default_rng(0)
    lens = [int(x) for x in rng.integers(0, 60, 1500)]
    lens[700] = 2000
    news = [int(x) for x in rng.integers(0, 3, 1500)]
    b = Batch(lens, [1] * 1500, 1, 2, 64, 16, dtype)
    _hold(b, b.run(ws, decode=True), _moments(b), tiles=False)
    b = Batch(lens, news, 1, 2, 64, 16, dtype)
    _hold(b, b.run(ws), _moments(b), tiles=False)


@pytest.mark.gpu
def test_calls_of_more_slots_than_a_block_has_threads(cuda) -> None:
    """2500 slots at once: extended, forked, freed, with and without enough pages."""
    import torch

    n, page = 2500, 4
    rng = np.random.default_rng(1)
    counts = rng.integers(0, 12, n)
    need = -(-counts // page)
    order = rng.permutation(n)
    c = PagedCache.allocate(1, 9000, 1, page, 8, 2 * n, 8, dtype=torch.float32)
    starts = np.concatenate([[0], np.cumsum(counts)])
    total = int(starts[-1])
    new = torch.randn((total, 1, 8), device=cuda)
    c.extend(_ints(order), _ints(starts))
    c.write(0, _ints(order), _ints(starts), new, -new)
    c.check()
    table = np.full((2 * n, 8), -1)
    at = 0
    for slot, m in zip(order, need):
        table[slot, :m] = range(at, at + m)
        at += m
    assert np.array_equal(c.table.cpu().numpy(), table)
    assert c.lens[_ints(order).long()].tolist() == counts.tolist()
    assert int(c.refs.sum()) == at and int(c.refs.max()) == 1
    for i in (0, 1023, 1024, 1025, 2047, 2048, n - 1):
        for j in range(counts[i]):
            p = table[order[i], j // page]
            assert torch.equal(c.k[0, p, :, j % page], new[starts[i] + j])
            assert torch.equal(c.v[0, p, :, j % page], -new[starts[i] + j])
    # children of all, the last first
    children = n + np.arange(n)[::-1]
    c.fork(_ints(order), _ints(children))
    c.check()
    opens = counts % page != 0
    got, lens = c.table.cpu().numpy(), c.lens.cpu().numpy()
    fresh = at
    for slot, child, m, m_open in zip(order, children, counts, opens):
        full = m // page
        assert lens[child] == m and np.array_equal(got[child, :full], table[slot, :full])
        if m_open:
            assert got[child, full] == fresh
            fresh += 1
    assert int(c.refs.sum()) == 2 * at
    # more than there are: nothing changes, one too many among them included
    before = [t.clone() for t in (c.refs, c.table, c.lens)]
    c.extend(_ints(order), _ints(np.arange(n + 1) * 20))
    c.extend(_ints([*order[:-1], order[5]]), _ints(np.arange(n + 1)))
    c.fork(_ints(children), _ints(children))
    with pytest.raises(CacheError):
        c.check()
    assert all(torch.equal(a, b) for a, b in zip((c.refs, c.table, c.lens), before))
    c.free(_ints(order))
    assert int(c.refs.sum()) == at and not c.lens[:n].any()
    c.free(_ints(children))
    c.check()
    assert not c.refs.any() and (c.table == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 8])
def test_logits_past_2_31_elements(cuda, top) -> None:
    """The last rows of 2.4e9 logits, and of their gradient, as those of a few rows."""
    import torch

    rows, vocab, last = 24000, 100003, 1200
    x = torch.empty((rows, vocab), dtype=torch.bfloat16, device=cuda)
    x[:-last] = 1
    x[-last:].normal_()
    t = torch.randint(0, vocab, (rows,), device=cuda)
    ones = torch.ones(rows, device=cuda)
    r, s = logprob.logprobs(x, t, top=top), logprob.logprobs(x[-last:], t[-last:], top=top)
    for a, b in ((r.logp, s.logp), (r.entropy, s.entropy), (r.top_logp, s.top_logp)):
        torch.testing.assert_close(a[-last:], b, rtol=1e-6, atol=8e-5)
    assert torch.equal(r.top_ids[-last:], s.top_ids)
    if top:
        assert (r.top_ids[0] == torch.arange(top, device=cuda)).all()
        return
    g = logprob.logprobs_grad(x, t, r, ones, ones)
    h = logprob.logprobs_grad(x[-last:], t[-last:], s, ones[-last:], ones[-last:])
    # p's error twice, and one unit of bf16 where that crosses a rounding
    assert bool(((g[-last:].float() - h.float()).abs() <= 2.0 ** -7 * h.float().abs() + 1e-9).all())
