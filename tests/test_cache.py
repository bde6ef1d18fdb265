"""The paged key-value cache: every page operation against a plain model of it (Python lists and
whole arrays), with its refusals. The operations move bytes and whole numbers, so everything must
be equal, keys and values bit for bit."""

from __future__ import annotations

import numpy as np
import pytest

from ptxgen import cache as cache_module
from ptxgen.build import build_library
from ptxgen.cache import CacheError, PagedCache
from ptxgen.runtime import Cache, LaunchError, Rows, library

PG_ERR_ARGUMENT = -2


class Model:
    """What the operations mean, on the host."""

    def __init__(self, layers, pages, heads, page, dim, slots, width):
        self.k = np.zeros((layers, pages, heads, page, dim), np.float32)
        self.v = np.zeros_like(self.k)
        self.refs = [0] * pages
        self.table = [[-1] * width for _ in range(slots)]
        self.lens = [0] * slots
        self.page, self.width = page, width

    def _take(self, n):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if len(free) < n:
            raise CacheError(cache_module.NO_PAGES)
        return free[:n]

    def extend(self, slots, counts):
        need = [-(-(self.lens[s] + c) // self.page) - -(-self.lens[s] // self.page)
                for s, c in zip(slots, counts)]
        fresh = self._take(sum(need))
        for s, c, n in zip(slots, counts, need):
            at = -(-self.lens[s] // self.page)
            for j in range(n):
                p = fresh.pop(0)
                self.table[s][at + j] = p
                self.refs[p] = 1
            self.lens[s] += c

    def write(self, layer, slots, counts, k, v):
        t = 0
        for s, c in zip(slots, counts):
            for pos in range(self.lens[s] - c, self.lens[s]):
                p = self.table[s][pos // self.page]
                self.k[layer, p, :, pos % self.page] = k[t]
                self.v[layer, p, :, pos % self.page] = v[t]
                t += 1

    def free(self, slots):
        for s in slots:
            for j in range(-(-self.lens[s] // self.page)):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lens[s] = 0

    def fork(self, parents, children):
        opens = [c for p, c in zip(parents, children) if self.lens[p] % self.page]
        fresh = self._take(len(opens))
        for p, c in zip(parents, children):
            full, part = divmod(self.lens[p], self.page)
            for j in range(full):
                self.table[c][j] = self.table[p][j]
                self.refs[self.table[p][j]] += 1
            if part:
                new, old = fresh.pop(0), self.table[p][full]
                self.table[c][full] = new
                self.refs[new] = 1
                self.k[:, new, :, :part] = self.k[:, old, :, :part]
                self.v[:, new, :, :part] = self.v[:, old, :, :part]
            self.lens[c] = self.lens[p]

    def copy_pages(self, a, b):
        self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if not self.refs[p]]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p]]
        for h, m in zip(holes, movers):
            self.k[:, h], self.v[:, h] = self.k[:, m], self.v[:, m]
            self.refs[h], self.refs[m] = self.refs[m], 0
            self.table = [[h if e == m else e for e in row] for row in self.table]


def _equal(cache, model) -> None:
    import torch

    torch.cuda.synchronize()
    assert cache.refs.tolist() == model.refs
    assert cache.table.tolist() == model.table
    assert cache.lens.tolist() == model.lens
    for got, want in ((cache.k, model.k), (cache.v, model.v)):
        assert np.array_equal(got.float().cpu().numpy(), want)


def _starts(counts, cuda):
    import torch

    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=cuda)


def _ints(x, cuda):
    import torch

    return torch.tensor(list(x), dtype=torch.int32, device=cuda)


# layers, pages, heads, page, dim, dtype
SHAPES = [(1, 40, 1, 16, 64, "bfloat16"), (3, 57, 3, 8, 24, "float16"),
          (2, 200, 2, 5, 20, "float32"), (2, 5000, 1, 1, 8, "float32"),
          (1, 90, 5, 64, 128, "bfloat16")]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("seed", [0, 1])
def test_random_operations_match_the_model(cuda, shape, seed) -> None:
    import torch

    layers, pages, heads, page, dim, dtype = shape
    rng = np.random.default_rng(seed)
    slots, width = 23, max(3, pages // 8)
    c = PagedCache.allocate(layers, pages, heads, page, dim, slots, width,
                            dtype=getattr(torch, dtype))
    c.k.zero_()
    c.v.zero_()
    m = Model(layers, pages, heads, page, dim, slots, width)
    done = 0
    for _ in range(60):
        what = rng.choice(["extend", "extend", "fork", "free", "compact", "copy"])
        live = [s for s in range(slots) if m.lens[s]]
        empty = [s for s in range(slots) if not m.lens[s]]
        if what == "extend":
            some = rng.permutation(slots)[:rng.integers(0, 6)].tolist()
            counts = [int(rng.integers(0, min(width * page - m.lens[s], 3 * page) + 1))
                      for s in some]
            try:
                m.extend(some, counts)
            except CacheError:
                c.extend(_ints(some, cuda), _starts(counts, cuda))
                with pytest.raises(CacheError, match="free pages"):
                    c.check()
                _equal(c, m)
                continue
            fused = torch.randn((sum(counts), 2 * heads + 1, dim), device=cuda).to(c.k.dtype)
            k, v = fused[:, :heads], fused[:, heads:2 * heads]  # strided rows
            c.extend(_ints(some, cuda), _starts(counts, cuda))
            layer = int(rng.integers(layers))
            c.write(layer, _ints(some, cuda), _starts(counts, cuda), k, v)
            m.write(layer, some, counts, k.float().cpu().numpy(), v.float().cpu().numpy())
        elif what == "fork":
            n = int(rng.integers(0, len(empty) + 1))
            parents = [int(rng.choice(live or empty[n:] or [0])) for _ in range(n)]
            children = empty[:n]
            if set(parents) & set(children):
                continue
            try:
                m.fork(parents, children)
            except CacheError:
                c.fork(_ints(parents, cuda), _ints(children, cuda))
                with pytest.raises(CacheError, match="free pages"):
                    c.check()
                _equal(c, m)
                continue
            c.fork(_ints(parents, cuda), _ints(children, cuda))
        elif what == "free":
            some = rng.permutation(slots)[:rng.integers(0, 8)].tolist()
            m.free(some)
            c.free(_ints(some, cuda))
        elif what == "compact":
            m.compact()
            c.compact()
        else:
            ids = rng.permutation(pages)[:8]
            m.copy_pages(ids[:4], ids[4:])
            c.copy_pages(_ints(ids[:4], cuda), _ints(ids[4:], cuda))
        _equal(c, m)
        c.check()
        done += 1
    assert done > 30


@pytest.mark.gpu
def test_strided_cache_and_another_stream(cuda) -> None:
    """Keys and values interleaved in one array, a table wider than its rows, and the calls on a
    stream of their own."""
    import torch

    pool = torch.zeros((2, 30, 2, 4, 16, 32), dtype=torch.bfloat16, device=cuda)  # k, v by page
    k, v = pool[:, :, 0], pool[:, :, 1]
    wide = torch.full((6, 9), -1, dtype=torch.int32, device=cuda)
    c = PagedCache(k, v, torch.zeros(30, dtype=torch.int32, device=cuda), wide[:, :5],
                   torch.zeros(6, dtype=torch.int32, device=cuda))
    m = Model(2, 30, 4, 16, 32, 6, 5)
    side = torch.cuda.Stream()
    new = torch.randn((50, 4, 32), device=cuda).to(torch.bfloat16)
    slots, starts = _ints([4, 1], cuda), _starts([33, 17], cuda)
    children, parents = _ints([0, 5], cuda), _ints([4, 1], cuda)
    torch.cuda.synchronize()
    s = side.cuda_stream
    c.extend(slots, starts, stream=s)
    c.write(1, slots, starts, new, new, stream=s)
    c.fork(parents, children, stream=s)
    c.free(slots, stream=s)
    c.compact(stream=s)
    side.synchronize()
    h = new.float().cpu().numpy()
    m.extend([4, 1], [33, 17])
    m.write(1, [4, 1], [33, 17], h, h)
    m.fork([4, 1], [0, 5])
    m.free([4, 1])
    m.compact()
    _equal(c, m)
    assert (wide[:, 5:] == -1).all()


@pytest.mark.gpu
def test_many_pages_and_long_offsets(cuda) -> None:
    """A keys array of more than 2^31 elements: the last pages are reached by 64-bit offsets."""
    import torch

    c = PagedCache.allocate(1, 70000, 8, 32, 128, 3, 64)  # 2.3e9 elements each
    c.refs[:69990] = 1
    slots, starts = _ints([1], cuda), _starts([300], cuda)
    new = torch.randn((300, 8, 128), device=cuda).to(torch.bfloat16)
    c.extend(slots, starts)
    c.write(0, slots, starts, new, -new)
    c.fork(slots[:0], slots[:0])
    c.check()
    assert c.table[1, :10].tolist() == list(range(69990, 70000))
    got = c.k[0, 69990:].permute(0, 2, 1, 3).reshape(-1, 8, 128)[:300]
    assert torch.equal(got, new)
    assert torch.equal(c.v[0, 69990:].permute(0, 2, 1, 3).reshape(-1, 8, 128)[:300], -new)
    c.refs[:69990] = 0
    c.compact()
    assert c.table[1, :10].tolist() == list(range(10))
    assert torch.equal(c.k[0, :10].permute(0, 2, 1, 3).reshape(-1, 8, 128)[:300], new)


@pytest.mark.gpu
def test_requests_that_cannot_be_met_change_nothing(cuda) -> None:
    import torch

    c = PagedCache.allocate(1, 8, 1, 4, 16, 5, 3, dtype=torch.float32)
    c.k.zero_()
    c.v.zero_()
    m = Model(1, 8, 1, 4, 16, 5, 3)
    c.extend(_ints([0, 2], cuda), _starts([6, 4], cuda))
    m.extend([0, 2], [6, 4])
    bad, long = cache_module.BAD_SLOT, cache_module.TOO_LONG
    for call, bits in [
            (lambda: c.extend(_ints([0, 5], cuda), _starts([1, 1], cuda)), bad),
            (lambda: c.extend(_ints([-1], cuda), _starts([1], cuda)), bad),
            (lambda: c.extend(_ints([1, 1], cuda), _starts([1, 1], cuda)), bad),
            (lambda: c.extend(_ints([1, 0], cuda), _starts([1, 7], cuda)), long),
            (lambda: c.extend(_ints([1], cuda), _ints([3, 2], cuda)), long),
            (lambda: c.fork(_ints([0], cuda), _ints([2], cuda)), bad),      # in use
            (lambda: c.fork(_ints([0, 0], cuda), _ints([1, 1], cuda)), bad),
            (lambda: c.fork(_ints([0, 3], cuda), _ints([3, 1], cuda)), bad),  # parent a child
            (lambda: c.fork(_ints([7], cuda), _ints([1], cuda)), bad),
            (lambda: c.free(_ints([9], cuda)), bad),
            (lambda: c.copy_pages(_ints([0], cuda), _ints([8], cuda)), cache_module.BAD_PAGE)]:
        call()
        with pytest.raises(CacheError) as e:
            c.check()
        assert e.value.bits == bits
        _equal(c, m)
        c.check()  # cleared
    # a slot freed twice in one call lets go of its pages once
    c.free(_ints([0, 0], cuda))
    m.free([0])
    _equal(c, m)
    c.check()


@pytest.mark.gpu
def test_refusals(cuda) -> None:
    import torch

    c = PagedCache.allocate(1, 8, 2, 4, 16, 5, 3, dtype=torch.float32)
    s, st = _ints([0], cuda), _starts([1], cuda)
    x = torch.zeros((1, 2, 16), device=cuda)
    with pytest.raises(ValueError, match="slots"):
        c.extend(s.long(), st)
    with pytest.raises(ValueError, match="starts"):
        c.extend(s, st[:1])
    with pytest.raises(ValueError, match="k: want"):
        c.write(0, s, st, x.half(), x)
    with pytest.raises(ValueError, match="v: want"):
        c.write(0, s, st, x, x[:, :1])
    with pytest.raises(LaunchError, match="layer 1 of 1"):
        c.write(1, s, st, x, x)
    odd = torch.zeros((1, 2, 18), device=cuda)[:, :, 1:17]
    with pytest.raises(LaunchError, match="multiples of 16"):
        c.write(0, s, st, odd, odd)
    with pytest.raises(LaunchError, match="entries"):
        c.free(_ints(range(6), cuda))
    with pytest.raises(LaunchError, match="16 bytes"):
        PagedCache.allocate(1, 8, 2, 4, 10, 5, 3).compact()
    with pytest.raises(ValueError, match="rows of one page"):
        PagedCache(c.k.transpose(2, 3), c.v.transpose(2, 3), c.refs, c.table, c.lens)


def test_bad_arguments_are_refused_before_any_cuda_call() -> None:
    build_library()
    lib = library()
    at = 1 << 20  # never dereferenced: every case fails its argument check first

    def cache(**other):
        fields = dict(k=at, v=at, layer_stride=1 << 16, page_stride=1 << 10, head_stride=256,
                      refs=at, table=at, lens=at, status=at, scratch=at, table_stride=4,
                      scratch_words=4 + 3 * 64 + 2 * 8 + 2, layers=1, pages=64, heads=4,
                      page_size=4, row_bytes=64, slots=8, width=4)
        return Cache(**{**fields, **other})

    rows = Rows(at, 256, 64)
    assert lib.pg_cache_compact(None, 0) == PG_ERR_ARGUMENT
    for other in [dict(k=0), dict(v=0), dict(refs=0), dict(status=0), dict(scratch=0),
                  dict(k=at + 8), dict(page_stride=1000), dict(row_bytes=8), dict(row_bytes=24),
                  dict(pages=0), dict(layers=-1), dict(heads=0), dict(table_stride=3),
                  dict(scratch_words=100), dict(refs=at + 2), dict(width=1 << 30)]:
        assert lib.pg_cache_compact(cache(**other), 0) == PG_ERR_ARGUMENT, other
    assert lib.pg_cache_extend(cache(), 0, at, 1, 0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_extend(cache(), at, at + 1, 1, 0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_extend(cache(), at, at, 9, 0) == PG_ERR_ARGUMENT
    assert b"9 entries" in lib.pg_last_error()
    assert lib.pg_cache_free(cache(), at, -1, 0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_fork(cache(), at, 0, 1, 0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_copy(cache(), at, at, 65, 0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_write(cache(), 1, at, at, 1, 1, rows, rows, 0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_write(cache(), 0, at, at, 1, 1, Rows(at + 4, 256, 64), rows,
                              0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_write(cache(), 0, at, at, 1, 1, rows, Rows(at, 250, 64),
                              0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_write(cache(), 0, at, at, 1, -1, rows, rows, 0) == PG_ERR_ARGUMENT
    # nothing to do is no error and makes no CUDA call
    assert lib.pg_cache_extend(cache(), 0, 0, 0, 0) == 0
    assert lib.pg_cache_free(cache(), 0, 0, 0) == 0
