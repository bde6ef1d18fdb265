"""Attention held to what its arithmetic allows at each result, not to the largest value.

With p the weights, A = sum p |v|, S = (sum p^2 v^2)^(1/2) and e the unit of the type's rounding (2^-8
bf16, 2^-11 f16):

* a score is a sum of products in 32 bits, with |q|, |k| about 1 a coordinate under 1e-5 off, so a weight
  is 1e-5 of itself off and the result 2e-5 A;
* single and few tokens in 16 bits hold a weight as two numbers, 2^-16 (bf16) or 2^-22 (f16) of itself
  off, and round the result once: e |o| + 4e-5 A, with 2^-24 for what f16 cannot hold;
* tiles of many rows round each weight once, independently, so with a variance of at most e^2 / 3 of its
  square: six times that root, 6 / 3^(1/2) e S = 3.5 e S, is met by one in 10^9 results;
* single and few tokens in f32 take each factor in two parts: scores are under 1e-6 off at these sizes
  (2^-22 a product, either sign, over 128 of them), exp2 2^-22, the weighted values 2^-21:
  2e-6 (A + |o|). FMA adds in order, a row of n keys with up to n^(1/2) 2^-24 of its largest sum: 4e-6.

The last test's scores are all equal, so that every weight is 1 and every sum exact: a result counts the
keys of some groups of 16, and one group left out or taken twice shows."""

from __future__ import annotations

import numpy as np
import pytest

from ptxgen import attention
from test_attention import TYPES, Batch

UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


def _moments(b, window=0, sinks=0):
    """The result in 64 bits, A and S."""
    import torch

    out = [torch.zeros(b.q.shape, dtype=torch.float64, device="cuda") for _ in range(3)]
    at = 0
    for seq, (n, new) in enumerate(zip(b.lens, b.news)):
        rows = slice(at, at + new)
        at += new
        if not n or not new:
            continue
        pos = torch.arange(n - new, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        seen = key <= pos
        if window:
            seen &= (key > pos - window) | (key < sinks)
        q = b.q[rows].double().view(new, b.heads, b.group, b.dim)
        for h in range(b.heads):
            k, v = b.keys[seq][h].double(), b.values[seq][h].double()
            s = torch.einsum("tgd,kd->tgk", q[:, h], k) * b.dim ** -0.5
            s = s.masked_fill(~seen[:, None], -torch.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)  # a query before the start sees none
            heads = slice(h * b.group, (h + 1) * b.group)
            out[0][rows, heads] = p @ v
            out[1][rows, heads] = p @ v.abs()
            out[2][rows, heads] = ((p * p) @ (v * v)).sqrt()
    return out


def _hold(b, got, moments, tiles, fma=False) -> None:
    import torch

    o, a, s = moments
    err = (got.double() - o).abs()
    dtype = str(b.dtype).split(".")[1]
    if dtype == "float32":
        bound = (4e-6 if fma else 2e-6) * (a + o.abs())
    else:
        e = UNIT[dtype]
        bound = e * o.abs() + 4e-5 * a + 2.0 ** -24 + (3.5 * e * s if tiles else 0.0)
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), float((err / bound).max())


# heads, group, dim, page
HEADS = [(2, 4, 128, 16), (1, 1, 64, 16), (2, 5, 64, 8), (1, 7, 96, 24), (1, 20, 128, 64),
         (3, 1, 128, 1), (2, 3, 32, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,most", [(1, 1), (5, 100), (1, 40000), (3, 9001), (60, 2000)])
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_single_tokens(ws, heads, group, dim, page, batch, most, dtype) -> None:
    rng = np.random.default_rng(most)
    lens = [int(x) for x in rng.integers(0, most + 1, batch)]
    lens[-1] = most
    b = Batch(lens, [1] * batch, heads, group, dim, page, dtype, seed=most)
    _hold(b, b.run(ws, decode=True), _moments(b), tiles=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4)])
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_a_few_tokens(ws, heads, group, dim, page, window, sinks, dtype) -> None:
    lens, news = [5000, 64, 1, 700], [2, 2, 2, 1]
    b = Batch(lens, news, heads, group, dim, page, dtype)
    got = b.run(ws, window=window, sinks=sinks)
    _hold(b, got, _moments(b, window, sinks), tiles=group * 7 > 4 * 48)


# pages that are no groups of eight keys come another way than those that are
PAGES = [16, 128, 1, 5, 12, 20]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 5), (1, 0)])
def test_many_tokens(ws, page, dim, window, sinks, dtype) -> None:
    """400 rows a sequence and more, over more blocks of keys than the ring holds."""
    lens, news = [1900, 700, 0, 301], [530, 650, 130, 301]
    b = Batch(lens, news, 2, 2, dim, page, dtype, fused=True)
    got = b.run(ws, window=window, sinks=sinks)
    _hold(b, got, _moments(b, window, sinks), tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 150)])
def test_many_tokens_in_several_parts(ws, page, dim, window, sinks, dtype) -> None:
    """Few tiles over long lengths, which are cut in parts and joined, the same way every time."""
    import torch

    b = Batch([9000], [130], 1, 4, dim, page, dtype)
    got = b.run(ws, window=window, sinks=sinks)
    _hold(b, got, _moments(b, window, sinks), tiles=True)
    for _ in range(3):
        assert torch.equal(b.run(ws, window=window, sinks=sinks), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf")])
def test_many_tokens_beside_junk(ws, page, dim, junk, dtype) -> None:
    """Keys that some rows of a tile see and others must not: the former get the formula's NaN or
    infinity, the others are bit for bit what they are without."""
    import torch

    lens, news, window, sinks = [900, 260], [500, 260], 150, 3
    b = Batch(lens, news, 2, 2, dim, page, dtype, junk=junk)
    clean = b.run(ws, window=window, sinks=sinks)
    _hold(b, clean, _moments(b, window, sinks), tiles=True)
    place = 620  # a key of sequence 0 that queries 620..769 see
    at, row = int(b.table[0, place // page]), place % page
    b.v[at, :, row, 3] = junk
    got = b.run(ws, window=window, sinks=sinks)
    pos = torch.arange(400, 900, device="cuda")
    sees = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    sees[:500, :, 3] = ((pos >= place) & (pos < place + window))[:, None]
    assert torch.equal(got[~sees], clean[~sees])
    assert torch.equal(got[sees].nan_to_num(7.0, 8.0, 9.0),
                       torch.full_like(got[sees], junk).nan_to_num(7.0, 8.0, 9.0))
    b.v[at, :, row, 3] = 0
    b.k[at, :, row, 5] = float("nan")
    got = b.run(ws, window=window, sinks=sinks)
    hit = sees[:, :, 3].any(-1)
    assert torch.isnan(got[hit]).all() and not torch.isnan(got[~hit]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news,group,dim", [([4000], [300], 8, 128), ([2500, 900], [500, 700], 4, 64),
                                                 ([3000], [1], 4, 256), ([900], [200], 2, 256)])
def test_f32_tiles(ws, lens, news, group, dim) -> None:
    b = Batch(lens, news, 1, group, dim, 16, "float32")
    _hold(b, b.run(ws), _moments(b), tiles=True, fma=True)


FORMS = [([40000], [1], 1, 8, 128, 16), ([9001, 0, 640, 33000], [1] * 4, 2, 4, 64, 8),
         ([700] * 40, [1] * 40, 4, 2, 128, 16), ([30000, 500, 9], [3, 1, 4], 1, 5, 64, 32),
         ([20000], [3], 1, 16, 128, 24), ([6000], [130], 1, 4, 128, 16), ([6000], [130], 1, 4, 128, 12),
         ([3000, 2000], [900, 700], 2, 2, 64, 16), ([3000, 2000], [900, 700], 2, 2, 96, 5),
         ([5000], [1], 2, 2, 256, 16), ([2000], [300], 1, 2, 256, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (2100, 40)])
@pytest.mark.parametrize("lens,news,heads,group,dim,page", FORMS)
def test_every_key_counts_once(ws, lens, news, heads, group, dim, page, window, sinks,
                               dtype) -> None:
    import torch

    b = Batch(lens, news, heads, group, dim, page, dtype)
    b.q[:] = 0
    for seq, n in enumerate(lens):
        which = torch.arange(n, device="cuda") // 16 % dim
        v = torch.nn.functional.one_hot(which, dim).to(b.dtype)
        b.values[seq] = v.expand(heads, n, dim)
        at = torch.arange(n, device="cuda")
        b.v[b.table[seq, at // page].long(), :, at % page] = v[:, None]
    o = _moments(b, window, sinks)[0]
    got = b.run(ws, window=window, sinks=sinks)
    # the one rounding of a quotient of whole numbers, and what its division leaves
    bound = (UNIT.get(dtype, 0.0) + 2.0 ** -20) * o
    assert bool(((got.double() - o).abs() <= bound).all())
