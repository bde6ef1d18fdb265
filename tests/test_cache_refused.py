"""What is queued behind an ``extend`` that cannot be met: the rows for it have no place in the
cache, and nothing that is there may be lost to them. Bytes and whole numbers: all must be equal."""

from __future__ import annotations

import pytest

from ptxgen import cache as cache_module
from ptxgen.build import build_library
from ptxgen.cache import CacheError, PagedCache
from ptxgen.runtime import Cache, Rows, library

PG_ERR_ARGUMENT = -2


def _ints(cuda, *x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _rows(cuda, n, fill):
    import torch

    return torch.full((n, 2, 16), float(fill), device=cuda)


def _cache(pages=6, slots=5, width=4, layers=2):
    import torch

    c = PagedCache.allocate(layers, pages, 2, 4, 16, slots, width, dtype=torch.float32)
    c.k.zero_()
    c.v.zero_()
    return c


def _state(c):
    return [t.clone() for t in (c.k, c.v, c.refs, c.table, c.lens)]


def _same(c, before) -> bool:
    import torch

    return all(torch.equal(a, b) for a, b in zip(_state(c), before))


@pytest.mark.gpu
@pytest.mark.parametrize("length", [8, 7, 1])
@pytest.mark.parametrize("why", ["no pages", "too long", "twice", "out of range"])
def test_a_refused_extend_and_its_queued_writes_change_nothing(cuda, why, length) -> None:
    c = _cache()
    slots, starts = _ints(cuda, 0, 1), _ints(cuda, 0, length, length + 3)
    c.extend(slots, starts)
    for layer in range(2):
        c.write(layer, slots, starts, _rows(cuda, length + 3, 1), _rows(cuda, length + 3, 2))
    # slot 2 continues slot 0: with 8 tokens all its pages are slot 0's own
    c.fork(_ints(cuda, 0), _ints(cuda, 2))
    c.check()
    before = _state(c)
    bits = {"no pages": cache_module.NO_PAGES, "too long": cache_module.TOO_LONG}
    slots, starts = {
        "no pages": ((0, 1, 2), (0, 7, 15, 22)),
        "too long": ((0, 2), (0, 1, 40)),
        "twice": ((0, 2, 0), (0, 1, 2, 3)),
        "out of range": ((0, 2, 5), (0, 1, 2, 3))}[why]
    slots, starts = _ints(cuda, *slots), _ints(cuda, *starts)
    n = int(starts[-1])
    c.extend(slots, starts)
    for layer in range(2):
        c.write(layer, slots, starts, _rows(cuda, n, 7), _rows(cuda, n, 8))
    assert _same(c, before)
    with pytest.raises(CacheError, match="not written") as e:
        c.check()
    assert e.value.bits & ~cache_module.REFUSED == bits.get(why, cache_module.BAD_SLOT)
    # the word is cleared, the slots' marks stay: a write that comes later has no place either
    c.write(0, _ints(cuda, 2), _ints(cuda, 0, 1), _rows(cuda, 1, 9), _rows(cuda, 1, 9))
    assert _same(c, before)
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == cache_module.REFUSED


@pytest.mark.gpu
def test_the_other_slots_of_a_step_are_written(cuda) -> None:
    c = _cache()
    c.extend(_ints(cuda, 0, 1), _ints(cuda, 0, 4, 8))
    c.write(0, _ints(cuda, 0, 1), _ints(cuda, 0, 4, 8), _rows(cuda, 8, 1), _rows(cuda, 8, 1))
    c.extend(_ints(cuda, 0), _ints(cuda, 0, 1))       # met
    c.extend(_ints(cuda, 1), _ints(cuda, 0, 12))      # 3 pages are left, slot 0 took one of 4
    c.extend(_ints(cuda, 1), _ints(cuda, 0, 1))       # none is left
    both, starts = _ints(cuda, 0, 1), _ints(cuda, 0, 1, 2)
    assert c.lens.tolist()[:2] == [5, 16]
    c.write(0, both, starts, _rows(cuda, 2, 3), _rows(cuda, 2, 4))
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == cache_module.TOO_LONG | cache_module.REFUSED
    assert (c.k[0, int(c.table[0, 1]), :, 0] == 3).all()
    assert (c.k[0, int(c.table[1, 0])] == 1).all() and not c.k[0, int(c.table[1, 3])].any()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["extend", "extend by none", "free", "fork"])
def test_what_clears_a_refusal(cuda, how) -> None:
    c = _cache()
    c.extend(_ints(cuda, 0), _ints(cuda, 0, 6))
    c.write(0, _ints(cuda, 0), _ints(cuda, 0, 6), _rows(cuda, 6, 1), _rows(cuda, 6, 1))
    slot = 1 if how == "fork" else 0
    c.extend(_ints(cuda, slot), _ints(cuda, 0, 40))
    with pytest.raises(CacheError):
        c.check()
    if how == "free":
        c.free(_ints(cuda, 0))
        c.lens[0] = 4  # a length and a page that the caller sets
        c.table[0, 0] = 0
    elif how == "fork":
        c.fork(_ints(cuda, 0), _ints(cuda, 1))
    else:
        c.extend(_ints(cuda, 0), _ints(cuda, 0, 1 if how == "extend" else 0))
    c.write(0, _ints(cuda, slot), _ints(cuda, 0, 1), _rows(cuda, 1, 5), _rows(cuda, 1, 6))
    c.check()
    last = int(c.lens[slot]) - 1
    at = int(c.table[slot, last // 4])
    assert (c.k[0, at, :, last % 4] == 5).all() and (c.v[0, at, :, last % 4] == 6).all()


@pytest.mark.gpu
def test_a_freed_slot_needs_no_other_call(cuda) -> None:
    c = _cache()
    c.extend(_ints(cuda, 0), _ints(cuda, 0, 40))
    c.free(_ints(cuda, 0))
    assert not c._refused.any()
    with pytest.raises(CacheError, match="more tokens"):
        c.check()


def test_marks_are_asked_for_before_any_cuda_call() -> None:
    build_library()
    lib = library()
    at = 1 << 20  # never dereferenced: every case fails its argument check first

    def cache(refused):
        return Cache(k=at, v=at, layer_stride=1 << 16, page_stride=1 << 10, head_stride=256,
                     refs=at, table=at, lens=at, status=at, scratch=at, refused=refused,
                     table_stride=4, scratch_words=4 + 3 * 64 + 2 * 8 + 2, layers=1, pages=64,
                     heads=4, page_size=4, row_bytes=64, slots=8, width=4)

    rows = Rows(at, 256, 64)
    for refused in (0, at + 2):
        c = cache(refused)
        assert lib.pg_cache_extend(c, at, at, 1, 0) == PG_ERR_ARGUMENT
        assert lib.pg_cache_free(c, at, 1, 0) == PG_ERR_ARGUMENT
        assert lib.pg_cache_fork(c, at, at, 1, 0) == PG_ERR_ARGUMENT
        assert lib.pg_cache_write(c, 0, at, at, 1, 1, rows, rows, 0) == PG_ERR_ARGUMENT
        assert b"marks" in lib.pg_last_error()
