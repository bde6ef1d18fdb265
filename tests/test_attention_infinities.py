"""Values that a query sees and that are not finite, against the definition in 64 bits: an infinity
gives that infinity, whatever its weight and however the weight is held, both infinities or a NaN give
NaN, and all other results are bit for bit what they are without them."""

from __future__ import annotations

import pytest

from ptxgen import attention
from test_attention import TYPES, Batch

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


def _put(b, seq, place, column, value) -> None:
    """A number of one key's values, in the cache and in the copy that the definition reads."""
    b.v[int(b.table[seq, place // b.page]), :, place % b.page, column] = value
    b.values[seq][:, place, column] = value


def _put_key(b, seq, place, key) -> None:
    b.k[int(b.table[seq, place // b.page]), :, place % b.page] = key
    b.keys[seq][:, place] = key


def _compare(got, want, clean) -> None:
    import torch

    odd = ~torch.isfinite(want)
    assert odd.any()
    assert torch.equal(got[odd].double().nan_to_num(7.0, INF, -INF),
                       want[odd].nan_to_num(7.0, INF, -INF))
    assert torch.equal(got[~odd], clean[~odd])


# heads, group, dim, page, lengths, new tokens: single tokens, short, alone and over many blocks; a few
# tokens; tiles by whole groups of eight keys and by others, in one part and in several; large heads
FORMS = [(2, 4, 128, 16, [1, 700, 90], [1, 1, 1]), (1, 8, 128, 16, [20000, 3], [1, 1]),
         (1, 20, 64, 8, [400], [1]), (2, 3, 64, 5, [333, 64], [3, 4]),
         (2, 2, 128, 16, [700, 300], [300, 150]), (1, 4, 64, 12, [900, 70], [200, 40]),
         (1, 4, 128, 32, [6000], [70]), (1, 4, 96, 20, [6000], [70]), (1, 2, 256, 16, [500], [1]),
         (1, 2, 256, 16, [500], [90])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_visible_infinities(ws, form, dtype) -> None:
    heads, group, dim, page, lens, news = form
    b = Batch(lens, news, heads, group, dim, page, dtype)
    clean = b.run(ws)
    for seq, n in enumerate(lens):
        _put(b, seq, 0, 3, INF)
        _put(b, seq, n // 3, 4, -INF)
        _put(b, seq, n // 2, 5, NAN)
        for place, value in ((n // 4, INF), (n // 2, -INF)):
            if n > 1:
                _put(b, seq, place, dim - 1, value)
        # twice the same, in one block and in different ones
        for place in {n // 5, n // 5 + 1, n - 1} & set(range(n)):
            _put(b, seq, place, 6, INF)
    _compare(b.run(ws), b.definition(), clean)
    if max(news) == 1:
        _compare(b.run(ws, decode=True), b.definition(), clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS[1:])
def test_an_infinity_of_small_weight(ws, form, dtype) -> None:
    """Its weight is about e^-28: nothing in f16, but not in the formula."""
    heads, group, dim, page, lens, news = form
    b = Batch(lens, news, heads, group, dim, page, dtype)
    b.q[:] = b.q[0, 0]
    for seq, n in enumerate(lens):
        _put_key(b, seq, n // 3, -b.q[0, 0] * (28 / dim ** 0.5))
    clean = b.run(ws)
    for seq, n in enumerate(lens):
        _put(b, seq, n // 3, 2, INF)
        _put(b, seq, n // 3, 7, -INF)
    _compare(b.run(ws), b.definition(), clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", [NAN, INF, -INF])
def test_scores_that_are_not_finite(ws, form, what, dtype) -> None:
    """A row whose scores are NaN or +inf, or all -inf, is NaN, beside values of every kind."""
    import torch

    heads, group, dim, page, lens, news = form
    b = Batch(lens, news, heads, group, dim, page, dtype)
    clean = b.run(ws)
    row = news[0] - 1  # the first sequence's last token: its first head is the odd one
    b.q[row, 0] = 0
    b.q[row, 0, 1] = what if what != -INF else INF
    sign = 1.0 if what == INF else -1.0
    b.k[:, 0, :, 1] = sign * b.k[:, 0, :, 1].abs().clamp(0.5).nan_to_num(1.0)
    b.keys[0][0, :, 1] = sign * b.keys[0][0, :, 1].abs().clamp(0.5)
    _put(b, 0, lens[0] // 2, 4, INF)
    got = b.run(ws)
    assert torch.isnan(got[row, 0]).all()
    assert not torch.isnan(got[row, group:]).any()  # the other kv heads' rows, if there are any
    assert torch.isfinite(clean).all()
