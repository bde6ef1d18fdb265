"""A fork whose parent's table names a page that does not exist changes nothing, whichever of the
row's pages it is. Bytes and whole numbers: all must be equal."""

from __future__ import annotations

import pytest

from ptxgen.cache import BAD_PAGE, BAD_SLOT, CacheError, PagedCache


def _ints(cuda, *x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device=cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [-1, 999, 1 << 30])
@pytest.mark.parametrize("length,at", [(6, 0), (6, 1), (8, 0), (8, 1), (1, 0), (900, 224),
                                       (899, 224), (900, 33)])
def test_a_page_out_of_range_changes_nothing(cuda, length, at, page) -> None:
    import torch

    c = PagedCache.allocate(2, 999, 2, 4, 16, 300, 240, dtype=torch.float32)
    for t in (c.k, c.v):
        t.copy_(torch.randn_like(t))
    slots, starts = _ints(cuda, 0, 1), _ints(cuda, 0, length, length + 5)
    c.extend(slots, starts)
    c.check()
    good = int(c.table[0, at])
    c.table[0, at] = page
    before = [t.clone() for t in (c.k, c.v, c.refs, c.table, c.lens)]
    many = list(range(2, 290))  # more requests than one block has warps; the last is the bad one
    c.fork(_ints(cuda, *[1] * 287, 0), _ints(cuda, *many))
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == BAD_PAGE
    assert all(torch.equal(a, b) for a, b in zip((c.k, c.v, c.refs, c.table, c.lens), before))
    # beside a slot that is in use both are reported
    c.fork(_ints(cuda, 0), _ints(cuda, 1))
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == BAD_PAGE | BAD_SLOT
    assert all(torch.equal(a, b) for a, b in zip((c.k, c.v, c.refs, c.table, c.lens), before))
    # what lies past the length is no page of the row
    c.table[0, at] = good
    c.table[0, -(-length // 4):] = page
    c.fork(_ints(cuda, 0, 1), _ints(cuda, 2, 3))
    c.check()
    assert c.lens[:4].tolist() == [length, 5, length, 5]
    got, want = c.table[2, :-(-length // 4)].tolist(), c.table[0, :-(-length // 4)].tolist()
    assert got[:length // 4] == want[:length // 4]
    assert int(c.refs.sum()) == 2 * (-(-length // 4) + 2)
