"""A write of fewer rows than its starts name reports the tokens that have none; rows past the starts
are left out."""

from __future__ import annotations

import pytest

from ptxgen.cache import TOO_LONG, CacheError, PagedCache


@pytest.mark.gpu
def test_tokens_without_rows_are_reported(cuda) -> None:
    import torch

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device=cuda)

    c = PagedCache.allocate(1, 40, 1, 4, 16, 3, 20, dtype=torch.float32)
    c.k.zero_()
    c.v.zero_()
    slots, starts = ints(0, 2), ints(0, 50, 57)
    x = torch.randn((60, 1, 16), device=cuda)
    c.extend(slots, starts)

    def held(slot, n):
        at = torch.arange(n, device=cuda)
        return c.k[0, c.table[slot, at // 4].long(), :, at % 4]

    c.write(0, slots, starts, x[:52], x[:52])
    with pytest.raises(CacheError, match="rows") as e:
        c.check()
    assert e.value.bits == TOO_LONG
    assert torch.equal(held(0, 50), x[:50]) and torch.equal(held(2, 2), x[50:52])
    assert not held(2, 7)[2:].any()
    c.write(0, slots, starts, x, x)
    c.check()
    assert torch.equal(held(0, 50), x[:50]) and torch.equal(held(2, 7), x[50:57])
    assert int((c.k != 0).any(-1).sum()) == 57
    c.write(0, slots, ints(-3, 50, 57), x, x)
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == TOO_LONG
