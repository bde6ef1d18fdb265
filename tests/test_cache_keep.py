"""Keeping some of a slot's last tokens: against lists on the host. Bytes and whole numbers, so all
must be equal, in what stays and in what is not touched."""

from __future__ import annotations

import random

import pytest

from ptxgen import cache as cache_module
from ptxgen.cache import CacheError, PagedCache


def _ints(x, dtype="int32"):
    import torch

    return torch.tensor(x, dtype=getattr(torch, dtype), device="cuda")


def _bits(places):
    m = sum(1 << p for p in places)
    return m - (1 << 64) if m >> 63 else m


class Filled:
    """A cache whose rows say which token of which slot they are."""

    def __init__(self, lens, layers=2, heads=2, page=4, dim=16, dtype="float32", spare=8):
        import torch

        self.page, self.layers = page, layers
        width = max(1, -(-max(lens) // page)) + 2
        pages = sum(-(-n // page) for n in lens) + spare
        t = getattr(torch, dtype)
        self.cache = PagedCache.allocate(layers, pages, heads, page, dim, len(lens) + 2, width, dtype=t)
        for x in (self.cache.k, self.cache.v):
            x.zero_()
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        slots = _ints(list(range(len(lens))))
        self.cache.extend(slots, _ints(starts))
        total = starts[-1]
        self.tokens = {s: list(range(a, b)) for s, (a, b) in enumerate(zip(starts, starts[1:]))}
        g = torch.Generator(device="cuda").manual_seed(1)
        of = t if dtype != "int8" else torch.float32
        self.rows = [[torch.randn((total, heads, dim), device="cuda", generator=g).to(of)
                      for _ in range(2)] for _ in range(layers)]
        if total:
            for i, (k, v) in enumerate(self.rows):
                self.cache.write(i, slots, _ints(starts), k, v)
            got = [self.cache.read(i, slots, _ints(starts), total, dtype=of) for i in range(layers)]
            self.rows = got
        self.of = of
        self.cache.check()

    def hold(self) -> None:
        """Every slot holds its tokens, in pages of its own that the counts know."""
        import torch

        c = self.cache
        lens, table, refs = c.lens.tolist(), c.table.tolist(), c.refs.tolist()
        counts = [0] * len(refs)
        for s, row in enumerate(table):
            tokens = self.tokens.get(s, [])
            assert lens[s] == len(tokens), s
            used = -(-len(tokens) // self.page)
            assert all(p >= 0 for p in row[:used]) and all(p == -1 for p in row[used:]), (s, row)
            for p in row[:used]:
                counts[p] += 1
            if tokens:
                for i in range(self.layers):
                    got = c.read(i, _ints([s]), _ints([0, len(tokens)]), len(tokens), dtype=self.of)
                    for a, b in zip(got, self.rows[i]):
                        assert torch.equal(a, b[tokens]), s
        assert refs == counts


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int8"])
@pytest.mark.parametrize("page", [1, 4, 16, 5])
@pytest.mark.parametrize("heads,dim", [(2, 16), (3, 128)])
def test_random_sets(cuda, heads, dim, page, dtype) -> None:
    rng = random.Random(page)
    lens = [64, 70, 1, 37, 90, 0, 12, 129, 64]
    f = Filled(lens, 2, heads, page, dim, dtype)
    slots = [8, 1, 2, 3, 4, 5, 7, 0]
    news = [64, 33, 1, 37, 64, 0, 63, 1]
    kept = [list(range(64)), rng.sample(range(33), 9), [0], [], rng.sample(range(64), 40), [], [62],
            [0]]
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    f.cache.keep(_ints(slots), _ints(starts), _ints([_bits(k) for k in kept], "int64"))
    for s, n, k in zip(slots, news, kept):
        base = len(f.tokens[s]) - n
        f.tokens[s] = f.tokens[s][:base] + [f.tokens[s][base + i] for i in sorted(k)]
    f.hold()
    f.cache.check()
    # the next tokens have room and places as ever
    f.cache.extend(_ints([3]), _ints([0, 6]))
    f.cache.check()
    assert int(f.cache.lens[3]) == 6


@pytest.mark.gpu
def test_bits_past_the_new_tokens_are_none(cuda) -> None:
    f = Filled([20, 9])
    f.cache.keep(_ints([0, 1]), _ints([0, 3, 3]), _ints([_bits([1, 3, 40, 63]), -1], "int64"))
    f.tokens[0] = f.tokens[0][:17] + [f.tokens[0][18]]
    f.hold()
    f.cache.check()


@pytest.mark.gpu
def test_pages_that_others_share(cuda) -> None:
    """A fork after the tokens were written shares their full pages: nothing may be moved there, but
    tokens that stay where they are may stay, and the others may go."""
    f = Filled([16, 16, 16])
    f.cache.fork(_ints([0, 1]), _ints([3, 4]))
    f.tokens[3], f.tokens[4] = list(f.tokens[0]), list(f.tokens[1])
    f.hold()
    f.cache.keep(_ints([0, 1, 2]), _ints([0, 8, 16, 24]),
                 _ints([_bits([2, 5]), _bits([0, 1]), _bits([2, 5])], "int64"))
    with pytest.raises(CacheError) as e:
        f.cache.check()
    assert e.value.bits == cache_module.BAD_PAGE
    f.tokens[1] = f.tokens[1][:10]
    f.tokens[2] = f.tokens[2][:8] + [f.tokens[2][10], f.tokens[2][13]]
    f.hold()


@pytest.mark.gpu
@pytest.mark.parametrize("slots,starts,bits", [
    ([0, 0], [0, 2, 4], cache_module.BAD_SLOT), ([9, 1], [0, 2, 4], cache_module.BAD_SLOT),
    ([-1, 1], [0, 2, 4], cache_module.BAD_SLOT), ([2, 1], [0, 2, 4], cache_module.TOO_LONG),
    ([0, 1], [0, 65, 67], cache_module.TOO_LONG), ([0, 1], [5, 2, 4], cache_module.TOO_LONG)])
def test_requests_that_cannot_be_met_leave_their_slot(cuda, slots, starts, bits) -> None:
    f = Filled([70, 30, 1])
    f.cache.keep(_ints(slots), _ints(starts), _ints([_bits([1])] * 2, "int64"))
    with pytest.raises(CacheError) as e:
        f.cache.check()
    assert e.value.bits == bits
    if slots[1] == 1 and slots[0] != 1:  # the other one is met
        f.tokens[1] = f.tokens[1][:28] + [f.tokens[1][29]]
    f.hold()


@pytest.mark.gpu
def test_a_refused_extend_has_no_tokens_to_keep(cuda) -> None:
    f = Filled([10])
    f.cache.extend(_ints([0]), _ints([0, 1000]))
    f.cache.keep(_ints([0]), _ints([0, 4]), _ints([_bits([3])], "int64"))
    with pytest.raises(CacheError) as e:
        f.cache.check()
    assert e.value.bits == cache_module.TOO_LONG | cache_module.REFUSED
    f.hold()


@pytest.mark.gpu
def test_bad_pages_in_a_table(cuda) -> None:
    f = Filled([16, 16])
    f.cache.table[0, 3] = 1 << 20
    before = f.cache.table.clone(), f.cache.refs.clone(), f.cache.lens.clone()
    f.cache.keep(_ints([0]), _ints([0, 4]), _ints([_bits([3])], "int64"))
    with pytest.raises(CacheError) as e:
        f.cache.check()
    assert e.value.bits == cache_module.BAD_PAGE
    import torch

    assert all(torch.equal(a, b) for a, b in zip(before, (f.cache.table, f.cache.refs, f.cache.lens)))


@pytest.mark.gpu
def test_captured(cuda) -> None:
    import torch

    f = Filled([40, 21])
    slots, starts, kept = _ints([0, 1]), _ints([0, 9, 13]), _ints([_bits([4, 6]), _bits([0, 3])], "int64")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f.cache.keep(slots, starts, kept)
    f.hold()  # nothing has run yet
    for _ in range(2):
        graph.replay()
        for s, n, k in ((0, 9, [4, 6]), (1, 4, [0, 3])):
            base = len(f.tokens[s]) - n
            f.tokens[s] = f.tokens[s][:base] + [f.tokens[s][base + i] for i in k]
        f.hold()
    f.cache.check()


@pytest.mark.gpu
def test_refused_sets(cuda) -> None:
    f = Filled([4])
    for kept in (_ints([1]), _ints([1, 1], "int64"), _ints([1], "int64").cpu(),
                 _ints([[1]], "int64")):
        with pytest.raises(ValueError, match="kept"):
            f.cache.keep(_ints([0]), _ints([0, 2]), kept)
