"""Many keys of small weight beside one of weight 1 whose values are 0: the result is made of the small
ones alone. f16 holds nothing below 2^-25 and rounds coarsely below 2^-14, so weights go into the product
scaled. Tolerances are those of tests/test_attention_exact.py, but that the weights are equal, so their
roundings to the type, where they are rounded once, are equal too: e A instead of 3.5 e S."""

from __future__ import annotations

import math

import pytest

from ptxgen import attention
from test_attention import TYPES, Batch
from test_attention_exact import UNIT, _moments


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


# log2 of the weight, lengths, new tokens, heads, group, dim, page
FORMS = [(-25.5, [60000], [1], 1, 8, 128, 16), (-25.5, [9000, 400], [1, 1], 2, 2, 64, 5),
         (-17.3, [700], [1], 1, 20, 96, 16), (-25.5, [20000], [3], 1, 4, 64, 16),
         (-20.0, [9000], [130], 1, 4, 128, 16), (-20.0, [5000], [130], 1, 4, 64, 12),
         (-20.4, [9000], [130], 1, 4, 128, 16), (-20.4, [5000], [130], 1, 4, 64, 12),
         (-20.4, [3000, 2000], [900, 700], 2, 2, 128, 16),
         (-15.2, [3000, 2000], [900, 700], 2, 2, 128, 16), (-25.5, [3000], [1], 1, 2, 256, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weight,lens,news,heads,group,dim,page", FORMS)
def test_small_weights(ws, weight, lens, news, heads, group, dim, page, dtype) -> None:
    import torch

    b = Batch(lens, news, heads, group, dim, page, dtype)
    b.q[:] = 0
    b.q[:, :, 0] = 1
    for seq, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        pages, rows = b.table[seq, at // page].long(), at % page
        b.keys[seq][:] = 0
        b.keys[seq][:, n // 3, 0] = -weight * math.log(2) * dim ** 0.5
        b.values[seq][:, n // 3] = 0
        b.values[seq][:, :, 1] = (at != n // 3).to(b.dtype)
        b.k[pages, :, rows] = b.keys[seq].transpose(0, 1)
        b.v[pages, :, rows] = b.values[seq].transpose(0, 1)
    o, a, _ = _moments(b)
    got = b.run(ws).double()
    e = UNIT.get(dtype, 0.0)
    tiles = max(news) > 4 and dtype != "float32"
    bound = e * o.abs() + 4e-5 * a + (e * a if tiles else 0.0) + 2.0 ** -24
    assert bool(((got - o).abs() <= bound).all()), float(((got - o).abs() / bound).max())
    assert float(o[:, :, 1].min()) > 2.0 ** -18
