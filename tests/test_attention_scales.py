"""Scales that are no usual ones: 0 (the mean of the values that a query sees), negative, and so small
that all scores are 0. Tolerances are those of tests/test_attention.py."""

from __future__ import annotations

import pytest

from ptxgen import attention
from test_attention import TYPES, Batch


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


# dim, page, the sequences' lengths and new tokens: one token, a few, many, and more than there are
BATCHES = [(128, 16, [1, 0, 700, 129], [1, 1, 1, 1]), (64, 5, [90, 333, 3], [4, 3, 5]),
           (128, 16, [700, 300, 40], [300, 150, 60]), (96, 12, [700, 90], [300, 90]),
           (256, 16, [400, 9], [130, 9])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.125, 1e-30, -1e-42])
@pytest.mark.parametrize("dim,page,lens,news", BATCHES)
def test_scales(ws, dim, page, lens, news, scale, window, sinks, dtype) -> None:
    b = Batch(lens, news, 2, 2, dim, page, dtype)
    want = b.definition(window, sinks, scale=scale)
    kw = dict(window=window, sinks=sinks, scale=scale)
    b.check(b.run(ws, **kw), want)
    if max(news) == 1:
        b.check(b.run(ws, decode=True, **kw), want)
