"""``check`` reports what calls on any stream met, and only once."""

from __future__ import annotations

import pytest

from ptxgen import attention
from ptxgen.cache import BAD_PAGE, TOO_LONG, CacheError, PagedCache


@pytest.mark.gpu
def test_check_waits_for_calls_on_other_streams(cuda) -> None:
    """The calls stand behind 50 ms of other work on their stream when ``check`` is called."""
    import torch

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    c = PagedCache.allocate(1, 8, 2, 16, 64, 3, 2)
    ws, side = attention.Workspace(), torch.cuda.Stream()
    c.extend(ints(0), ints(0, 5))
    c.table[0, 0] = 77
    q, slot, starts, far = (torch.zeros((1, 4, 64), device="cuda", dtype=torch.bfloat16), ints(0),
                            ints(0, 1), ints(0, 99))
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
        c.extend(slot, far, stream=side.cuda_stream)
        with pytest.raises(CacheError) as e:
            c.check()
        assert e.value.bits == TOO_LONG
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
        attention.decode(q, c.k[0], c.v[0], c.table, c.lens, slots=slot, workspace=ws,
                         stream=side.cuda_stream)
        with pytest.raises(CacheError) as e:
            ws.check()
        assert e.value.bits == BAD_PAGE
        c.check()
        ws.check()


@pytest.mark.parametrize("bits", [0, 5])
def test_the_word_is_read_and_cleared_between_waits(monkeypatch, bits) -> None:
    """The order of the steps, on a word in host memory."""
    import torch

    from ptxgen import launch

    word, seen = torch.tensor([bits], dtype=torch.int32), []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: seen.append(int(word[0])))
    assert launch.take_status(word) == bits
    assert seen == ([5, 0] if bits else [0]) and int(word[0]) == 0
