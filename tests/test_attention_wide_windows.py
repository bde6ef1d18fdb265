"""Windows that hide nothing, up to the largest number, beside queries that stand before their
sequence's start: the result is that of no window, bit for bit."""

from __future__ import annotations

import pytest

from ptxgen import attention
from test_attention import TYPES, Batch


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


# dim, page, lengths, new tokens: few and many rows, whole groups of eight keys a page and others
BATCHES = [(64, 16, [9, 30, 0], [12, 3, 2]), (128, 16, [300, 9, 130], [310, 80, 130]),
           (64, 12, [300, 9], [310, 80]), (256, 16, [9, 30], [12, 3])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [350, 1 << 20, 2 ** 31 - 400, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 5, 2 ** 31 - 1])
@pytest.mark.parametrize("dim,page,lens,news", BATCHES)
def test_windows_that_hide_nothing(ws, dim, page, lens, news, window, sinks, dtype) -> None:
    import torch

    b = Batch(lens, news, 2, 2, dim, page, dtype)
    got = b.run(ws, window=window, sinks=sinks)
    b.check(got, b.definition())
    assert torch.equal(got, b.run(ws))
    # one key short of hiding nothing, and no less
    short = max(lens) - 1
    b.check(b.run(ws, window=short), b.definition(short))
    b.check(b.run(ws, window=3, sinks=2 ** 31 - 1), b.definition())
