"""Attention over a cache in 8 bits, and of trees of drafted tokens, against the definitions in 64 bits.

With p the weights, A = sum p |v|, S = (sum p^2 v^2)^(1/2) and e the unit of the type's rounding (2^-8
bf16, 2^-11 f16, 2^-24 f32):

* a score is a sum of products in 32 bits, under 1e-5 off at these sizes, so a weight is 1e-5 of itself
  off and the result 2e-5 A; the queries of an 8-bit cache lose no more than 2^-22 of their largest
  on the way to f16 (f32 ones, in two parts); the keys for 16-bit ones go in with 128 added, so their sums
  pass numbers up to four times as large, and the result is 8e-5 A off there;
* a weight goes into its product as two numbers, 2^-16 of itself off (bf16) or 2^-22 (f16, and all over 8
  bits; there its product with the value's scale loses what is below 2^-39 of the largest scale, with
  |q| up to 127 and n keys of no more weight than 1 each against a sum of at least 1: 2^-32 n of it),
  and the result is rounded once: e |o| + 4e-5 A + 2^-32 n s, with 2^-24 for what f16 cannot hold;
* a bf16 result over 8 bits has its weights as one f16 number each, 2^-12 of itself off, independently:
  six times the root of that variance, 3.5 2^-12 S, more;
* tiles of many rows round each weight once, independently: six times the root of that variance more,
  3.5 e S, is met by one in 10^9 results. Over 8 bits that is in f16 for bf16 results, e = 2^-11 here, and
  keys and values are rounded to f16, too: half a step each, again at random, so the values add 1.75 e S,
  and a score has a variance of c^2, c = e / 12^(1/2) times the scale and (sum q^2 k^2)^(1/2), the weights
  that much of themselves and the result 6 c (S + |o|) with the largest c. So it is for f16 results without
  room to widen in; with it, keys and values are exact there, and a weight times its value's scale goes in
  as two f16 numbers, 2^-22 of itself off, but for what is below f16's normal numbers: 2^-25, with weights
  held at 2^7, scales at half a page's largest or less and numbers up to 127, 2^-32 2 127 s = 2^-31 max |v|
  for each of n keys.

Heads above 128 are summed in f32 in order: n^(1/2) 2^-24 of the largest sum, within 4e-5 A at 4000."""

from __future__ import annotations

import random

import numpy as np
import pytest

from ptxgen import attention
from ptxgen import cache as cache_module
from ptxgen.build import build_library
from ptxgen.cache import CacheError
from ptxgen.runtime import AttentionArgs, AttentionMore, LaunchError, library

PG_ERR_ARGUMENT = -2
TYPES = ["float32", "bfloat16", "float16"]
UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


def _ints(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Batch:
    """Random sequences over scattered pages; what no sequence has is NaN, or a scale of NaN.

    masks: a list a sequence of which new tokens each of its new tokens sees."""

    def __init__(self, lens, news, heads, group, dim, page, dtype, bits8, masks=None, seed=0,
                 spread=1.0):
        import torch

        self.lens, self.news, self.masks = lens, news, masks
        self.heads, self.group, self.dim, self.page = heads, group, dim, page
        self.dtype, self.bits8 = getattr(torch, dtype), bits8
        g = torch.Generator(device="cuda").manual_seed(seed)
        counts = [-(-n // page) for n in lens]
        pages, width = sum(counts) + 2, max(1, max(counts))
        shape = (pages, heads, page, dim)
        ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        at = 0
        unused = torch.ones((pages, page), dtype=torch.bool, device="cuda")
        for i, (n, c) in enumerate(zip(lens, counts)):
            self.table[i, :c] = ids[at:at + c]
            for j in range(c):
                unused[ids[at + j].long(), :min(page, n - j * page)] = False
            at += c
        self.scales = {}
        if bits8:
            self.k, self.v = (torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda",
                                            generator=g) for _ in range(2))
            for name in ("k_scale", "v_scale"):
                s = (torch.randn(shape[:3], device="cuda", generator=g) * spread).exp() / 60
                s.transpose(1, 2)[unused] = float("nan")
                self.scales[name] = s
        else:
            self.k, self.v = (torch.randn(shape, device="cuda", generator=g).to(self.dtype)
                              for _ in range(2))
            for x in (self.k, self.v):
                x.transpose(1, 2)[unused] = float("nan")
        fused = torch.randn((sum(news), (group + 2) * heads, dim), device="cuda", generator=g)
        self.q = fused.to(self.dtype)[:, :group * heads]
        self.starts = _ints(np.concatenate([[0], np.cumsum(news)]).astype(np.int32).tolist())
        if masks is not None:
            bits = [sum(1 << t for t in m) for seq in masks for m in seq]
            self.mask = torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits],
                                     dtype=torch.int64, device="cuda")

    def run(self, ws, **more):
        args = self.k, self.v, self.table, _ints(self.lens)
        more = {**self.scales, "workspace": ws, **more}
        if self.masks is not None:
            return attention.tree(self.q, self.starts, self.mask, *args, **more)
        if more.pop("single", False):
            return attention.decode(self.q, *args, **more)
        return attention.prompt(self.q, self.starts, *args, **more)

    def rows_of(self, name, i, h):
        x, n = getattr(self, name), self.lens[i]
        ids = self.table[i, :-(-n // self.page)].long()
        y = x[ids, h].reshape(-1, self.dim)[:n].double()
        if self.bits8:
            y = y * self.scales[name + "_scale"][ids, h].reshape(-1)[:n, None].double()
        return y

    def seen(self, i, window, sinks):
        """[new tokens, keys], by counting what a token sees in order."""
        import torch

        n, new = self.lens[i], self.news[i]
        base = n - new
        out = np.zeros((new, n), bool)
        for r in range(new):
            if self.masks is None:
                sees = np.arange(max(0, base + r + 1))
            else:
                sees = np.array([*range(max(base, 0)), *(base + t for t in sorted(self.masks[i][r])
                                                         if t < new and base + t >= 0)], dtype=int)
                if base + r < 0:
                    continue
            place = np.arange(len(sees))
            if window:
                sees = sees[(place > len(sees) - 1 - window) | (place < sinks)]
            out[r, sees] = True
        return torch.from_numpy(out).cuda()

    def hold(self, got, window=0, sinks=0, tiles=False, scale=None, but=None,
             rounded=False) -> None:
        import torch

        scale = self.dim ** -0.5 if scale is None else scale
        e, at = UNIT[str(self.dtype).split(".")[1]], 0
        for i, (n, new) in enumerate(zip(self.lens, self.news)):
            rows = slice(at, at + new)
            at += new
            if not new or i == but:
                continue
            if not n:
                assert (got[rows] == 0).all()
                continue
            seen = self.seen(i, window, sinks)
            q = self.q[rows].double().view(new, self.heads, self.group, self.dim)
            for h in range(self.heads):
                k, v = self.rows_of("k", i, h), self.rows_of("v", i, h)
                s = torch.einsum("tgd,kd->tgk", q[:, h], k) * scale
                s = s.masked_fill(~seen[:, None], -torch.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0)  # one that sees none
                o, a, m = p @ v, p @ v.abs(), ((p * p) @ (v * v)).sqrt()
                y = got[rows, h * self.group:(h + 1) * self.group].double()
                bound = e * o.abs() + 4e-5 * a + 2.0 ** -24 * (self.dtype != torch.float32)
                if self.bits8:
                    bound = bound + 2.0 ** -32 * n * float(v.abs().max()) / 127
                if self.bits8 and self.dtype != torch.float32:
                    bound = bound + 4e-5 * a
                if self.bits8 and self.dtype is torch.bfloat16:
                    bound = bound + 3.5 * 2.0 ** -12 * m
                # the tiles' products over 8 bits are in f16 for both types
                e = UNIT["float16"] if self.bits8 else e
                whole = self.bits8 and self.dtype is torch.float16 and not rounded
                if tiles and not whole:
                    bound = bound + 3.5 * e * m
                if tiles and self.bits8 and self.dtype is torch.float16:
                    bound = bound + 2.0 ** -31 * n * float(v.abs().max())
                if tiles and self.bits8 and (rounded or self.dtype is torch.bfloat16):
                    c = torch.einsum("tgd,kd->tgk", q[:, h] ** 2, k ** 2).sqrt()
                    c = c.masked_fill(~seen[:, None], 0.0).amax(-1, keepdim=True) * abs(scale)
                    bound = bound + 1.75 * e * m + 6 * c * e / 12 ** 0.5 * (m + o.abs())
                e = UNIT[str(self.dtype).split(".")[1]]
                bad = ~((y - o).abs() <= bound)
                assert not bad.any(), (i, h, float(((y - o).abs() / bound).nan_to_num(1e9).max()),
                                       bad.nonzero()[:4].tolist())


# heads, group, dim, page
HEADS = [(2, 4, 128, 16), (1, 1, 64, 16), (2, 5, 64, 8), (1, 7, 96, 24), (1, 20, 128, 64),
         (3, 1, 128, 1), (2, 3, 32, 5), (1, 2, 16, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,most", [(1, 1), (5, 100), (1, 40000), (3, 9001), (60, 2000)])
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_single_tokens_over_8_bits(ws, heads, group, dim, page, batch, most, dtype) -> None:
    rng = np.random.default_rng(most)
    lens = [int(x) for x in rng.integers(0, most + 1, batch)]
    lens[-1] = most
    b = Batch(lens, [1] * batch, heads, group, dim, page, dtype, True, seed=most)
    b.hold(b.run(ws, single=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4), (1, 0)])
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_several_tokens_over_8_bits(ws, heads, group, dim, page, window, sinks, dtype) -> None:
    b = Batch([1000, 64, 1, 700, 0, 333], [2, 64, 2, 1, 3, 150], heads, group, dim, page, dtype, True)
    b.hold(b.run(ws, window=window, sinks=sinks), window, sinks, tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("page", [16, 128, 1, 5, 12])
@pytest.mark.parametrize("dim", [16, 64, 96, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 5)])
def test_many_tokens_over_8_bits(ws, page, dim, window, sinks, dtype) -> None:
    """400 rows a sequence and more, over more blocks of keys than the ring holds."""
    b = Batch([1900, 700, 0, 301], [530, 650, 130, 301], 2, 2, dim, page, dtype, True)
    b.hold(b.run(ws, window=window, sinks=sinks), window, sinks, tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [144, 256])
def test_large_heads_over_8_bits(ws, dim, new, dtype) -> None:
    b = Batch([700, 41, 0], [new, min(new, 41), new], 2, 3, dim, 16, dtype, True)
    b.hold(b.run(ws))
    b.hold(b.run(ws, window=30, sinks=2), 30, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [0.0, 4.0])
def test_scales_of_unlike_size(ws, spread, dtype) -> None:
    """From e^-16 to e^16 of one another: the largest may have the least weight."""
    b = Batch([3000, 200], [1, 1], 2, 4, 128, 16, dtype, True, spread=spread)
    b.scales["k_scale"].clamp_(max=0.05)
    b.hold(b.run(ws, single=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_queries_of_any_size(ws, size, dtype) -> None:
    if dtype == "float16" and size > 1:
        size = 1000.0
    b = Batch([500, 30], [1, 1], 2, 4, 64, 16, dtype, True)
    b.q = (b.q * size).to(b.dtype)
    b.q[0, 1] = 0
    b.hold(b.run(ws, single=True, scale=0.125 / size), scale=0.125 / size)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 20, 70])
@pytest.mark.parametrize("dim", [64, 256])
def test_scales_that_are_not_finite(ws, dim, new, dtype) -> None:
    """They reach the rows that see them and no others."""
    import torch

    for name in ("k_scale", "v_scale"):
        b = Batch([100, 100, 100], [new] * 3, 2, 2, dim, 16, dtype, True)
        key = 100 - new // 2 - 1  # the first rows of more than one do not see it
        page = int(b.table[1, key // 16])
        b.scales[name][page, 1, key % 16] = float("nan")
        got = b.run(ws).view(3, new, 2, 2, dim)
        blind = max(0, key - (100 - new))
        assert torch.isfinite(got[[0, 2]]).all() and torch.isfinite(got[1, :, 0]).all()
        assert torch.isfinite(got[1, :blind, 1]).all() and torch.isnan(got[1, blind:, 1]).all()


@pytest.mark.gpu
def test_out_strides_slots_and_streams_over_8_bits(ws) -> None:
    import torch

    b = Batch([90, 200, 5], [1, 1, 1], 2, 3, 64, 16, "bfloat16", True)
    want = b.run(ws, single=True)
    wide = torch.full((3, 9, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    got = b.run(ws, single=True, out=wide[:, 2:8])
    assert torch.equal(got, want) and (wide[:, [0, 1, 8]] == 7.0).all()
    side, other = torch.cuda.Stream(), attention.Workspace()
    torch.cuda.synchronize()
    got = b.run(other, single=True, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)
    # slots: the same sequences in another order
    got = attention.decode(b.q[[2, 0]], b.k, b.v, b.table, _ints(b.lens), slots=_ints([2, 0]),
                           workspace=ws, **b.scales)
    assert torch.equal(got, want[[2, 0]])
    graph = torch.cuda.CUDAGraph()
    lens = _ints(b.lens)
    with torch.cuda.graph(graph):
        got = attention.decode(b.q, b.k, b.v, b.table, lens, workspace=ws, **b.scales)
    graph.replay()
    assert torch.equal(got, want)


# (lens, news, max_len): prompts whose keys are widened block by block, and in the workspace first
WAYS = [([900, 200], [70, 60], None), ([1500, 1000], [900, 700], None)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("spread", [0.0, 2.0])
@pytest.mark.parametrize("lens,news,max_len", WAYS)
def test_prompts_with_scales_of_unlike_size(ws, lens, news, max_len, spread, dtype) -> None:
    """Values far apart, also from page to page; pages of zeros; a head of nothing else."""
    b = Batch(lens, news, 2, 4, 128, 16, dtype, True, spread=spread)
    b.scales["k_scale"].clamp_(max=0.05)
    v = b.scales["v_scale"]
    for i in range(len(lens)):
        v[b.table[i, 2:60:7].long()] *= 2.0 ** -20
        v[b.table[i, 5:60:7].long()] *= 2.0 ** 6
        v[b.table[i, 0:8].long()] = 0.0  # all of the first 128 tokens
        b.v[b.table[i, 24:33].long()] = 0  # ... and of others, by numbers that are 0
        v[b.table[i].long().clamp(min=0), 1] = 0.0
    b.hold(b.run(ws, max_len=max_len), tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [1e-6, 1e4])
@pytest.mark.parametrize("lens,news,max_len", WAYS)
def test_prompts_with_queries_of_any_size(ws, lens, news, max_len, size, dtype) -> None:
    if dtype == "float16" and size > 1:
        size = 1000.0
    b = Batch(lens, news, 1, 4, 64, 16, dtype, True)
    b.q = (b.q * size).to(b.dtype)
    b.q[0, 1] = 0
    b.q[1:3] = b.q[1:3] * 2.0 ** -10  # rows have their own
    b.hold(b.run(ws, scale=-0.125 / size, max_len=max_len), scale=-0.125 / size, tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_wide_tables_and_larger_workspaces(ws, dtype) -> None:
    """A table for far more tokens than there are: nothing of the workspace goes by it."""
    import torch

    b = Batch([1500, 1000], [900, 700], 2, 4, 128, 16, dtype, True)
    want = b.run(ws, max_len=1500)
    table = torch.full((2, 1 << 16), -1, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = b.table
    b.table, narrow = table, b.table
    b.hold(b.run(ws), tiles=True, rounded=True)
    b.table = narrow
    large = attention.Workspace(size=200 << 20)
    assert torch.equal(b.run(large, max_len=1500), want)
    large.check()
    with pytest.raises(ValueError, match="bytes at least"):
        attention.Workspace(size=1 << 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_sequences_longer_than_max_len(cuda, dtype) -> None:
    w = attention.Workspace()
    b = Batch([1500, 1000], [900, 700], 2, 4, 128, 16, dtype, True)
    got = b.run(w, max_len=1000)
    with pytest.raises(CacheError) as e:
        w.check()
    assert e.value.bits == cache_module.TOO_LONG
    b.hold(got, tiles=True, but=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("news,masked", [([1, 1, 1], False), ([9, 9, 9], False), ([70, 60, 50], False),
                                         ([900, 400, 800], False), ([5, 6, 7], True), ([64, 60, 50], True)])
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("bad", ["slot", "slot below", "page", "page below", "length", "length below"])
def test_what_only_the_device_sees(cuda, bad, bits8, news, masked, dtype) -> None:
    """The second sequence is refused; the others have their results, and the next call is sound."""
    import torch

    w = attention.Workspace()
    masks = _trees(2, news) if masked else None
    b = Batch([1100, 1000, 900], news, 1, 8, 64, 16, dtype, bits8, masks)
    want = b.run(w)
    w.check()
    slots, table, lens = _ints([0, 1, 2]), b.table.clone(), _ints(b.lens)
    bit = {"slot": cache_module.BAD_SLOT, "page": cache_module.BAD_PAGE,
           "length": cache_module.TOO_LONG}[bad.split()[0]]
    if bad.startswith("slot"):
        slots[1] = -1 if "below" in bad else 3
    elif bad.startswith("page"):
        table[1, 60] = -1 if "below" in bad else b.k.shape[0]
    else:
        lens[1] = -1 if "below" in bad else table.shape[1] * 16 + 1
    more = dict(workspace=w, slots=slots, **b.scales)
    if masked:
        got = attention.tree(b.q, b.starts, b.mask, b.k, b.v, table, lens, **more)
    else:
        got = attention.prompt(b.q, b.starts, b.k, b.v, table, lens, **more)
    with pytest.raises(CacheError) as e:
        w.check()
    # a length that is cut to the table's width goes over entries that no page has been set to
    assert e.value.bits in (bit, bit | (cache_module.BAD_PAGE if bad == "length" else 0))
    b.hold(got, tiles=True, but=1)
    assert torch.equal(b.run(w), want)
    w.check()


@pytest.mark.gpu
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("news,masked", [([5, 6], True), ([64, 60], True), ([70, 60], False),
                                         ([900, 700], False)])
def test_graphs_streams_and_slots(ws, news, masked, bits8) -> None:
    """Captured once and replayed with other queries and lengths; on a second stream with a workspace
    of its own at the same time; rows that no sequence has stay."""
    import torch

    masks = _trees(3, news) if masked else None
    b = Batch([1500, 1000], news, 2, 4, 64, 16, "bfloat16", bits8, masks)
    rows = sum(news)
    q = torch.cat([b.q, b.q[:3]])
    out = torch.full_like(q, 5.0)
    lens, table = _ints(b.lens), b.table[[1, 0]].contiguous()
    mask = torch.cat([b.mask, b.mask[:3]]) if masked else None
    other, side = attention.Workspace(), torch.cuda.Stream()

    def go(w, to, stream=None):
        more = dict(workspace=w, slots=_ints([1, 0]) if stream is None else slots, out=to, stream=stream,
                    **b.scales)
        if masked:
            attention.tree(q, b.starts, mask, b.k, b.v, table, lens[[1, 0]] if stream is None else turned,
                           **more)
        else:
            attention.prompt(q, b.starts, b.k, b.v, table, lens[[1, 0]] if stream is None else turned,
                             **more)

    slots, turned = _ints([1, 0]), _ints(b.lens[::-1])
    want = b.run(ws)
    twice = torch.full_like(q, 5.0)
    torch.cuda.synchronize()
    go(other, twice, side.cuda_stream)
    go(ws, out, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out[:rows], want) and torch.equal(twice[:rows], want)
    assert (out[rows:] == 5.0).all() and (twice[rows:] == 5.0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(ws, out, torch.cuda.current_stream().cuda_stream)
    q.mul_(0.5)
    turned -= 16
    b.q, b.lens = q[:rows], [n - 16 for n in b.lens]
    out.fill_(5.0)
    graph.replay()
    want = b.run(ws)
    assert torch.equal(out[:rows], want) and (out[rows:] == 5.0).all()
    other.check()


# --- trees --------------------------------------------------------------------------------------


def _tree(rng, n):
    parents = [-1] + [rng.randint(max(-1, i - 5), i - 1) for i in range(1, n)]
    masks = []
    for i, p in enumerate(parents):
        masks.append([*(masks[p] if p >= 0 else []), i])
    return parents, masks


def _trees(seed, news):
    rng = random.Random(seed)
    return [_tree(rng, n)[1] if n else [] for n in news]


@pytest.mark.gpu
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4), (3, 2), (1, 0)])
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_trees(ws, heads, group, dim, page, window, sinks, dtype, bits8) -> None:
    lens, news = [2000, 64, 1, 7, 133, 0], [7, 3, 1, 7, 5, 0]
    b = Batch(lens, news, heads, group, dim, page, dtype, bits8, _trees(dim, news))
    b.hold(b.run(ws, window=window, sinks=sinks), window, sinks, tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 5), (40, 30), (2, 0)])
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_large_trees(ws, heads, group, dim, page, window, sinks, dtype, bits8) -> None:
    lens, news = [1300, 64, 700, 190, 60], [64, 64, 63, 62, 33]
    b = Batch(lens, news, heads, group, dim, page, dtype, bits8, _trees(dim, news))
    b.hold(b.run(ws, window=window, sinks=sinks), window, sinks, tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [3, 64])
@pytest.mark.parametrize("dim", [160, 256])
def test_trees_with_large_heads(ws, dim, new, dtype, bits8) -> None:
    news = [new, new, 1]
    b = Batch([500, new, 40], news, 1, 3, dim, 16, dtype, bits8, _trees(dim, news))
    b.hold(b.run(ws))
    b.hold(b.run(ws, window=5, sinks=3), 5, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [1, 8])
@pytest.mark.parametrize("window,sinks", [(0, 0), (4, 0), (4, 6)])
def test_masks_that_are_no_trees(ws, window, sinks, group, dtype) -> None:
    """Any set: none, not even itself; tokens behind it; bits past the sequence's tokens."""
    rng = random.Random(group)
    lens, news = [30, 30, 12, 150], [20, 30, 12, 60]
    masks = [[sorted(rng.sample(range(64), rng.choice([0, 0, 1, 5, 20, 64]))) for _ in range(n)]
             for n in news]
    b = Batch(lens, news, 2, group, 64, 16, dtype, False, masks)
    b.hold(b.run(ws, window=window, sinks=sinks), window, sinks, tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [1, 8])
def test_sequences_shorter_than_their_trees(ws, group, dtype) -> None:
    """Tokens before the start see nothing and are not seen."""
    lens, news = [10, 0, 30, 5], [20, 9, 30, 64]
    b = Batch(lens, news, 2, group, 64, 16, dtype, False, _trees(1, news))
    b.hold(b.run(ws), tiles=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news,group", [([3, 2, 1], 4), ([64, 60, 1], 8)])
def test_a_tree_of_one_branch_is_a_prompt(ws, news, group, dtype) -> None:
    import torch

    masks = [[list(range(i + 1)) for i in range(n)] for n in news]
    b = Batch([300, 64, 1], news, 2, group, 64, 16, dtype, False, masks)
    got = b.run(ws)
    b.masks = None
    want = b.run(ws)
    if sum(news) * group > 48 * 3 and dtype == "float32":
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)  # another kernel's sums
    else:
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [2, 16])
def test_values_that_are_not_finite_in_other_branches(ws, group) -> None:
    import torch

    for value in (float("nan"), float("inf")):
        for dtype in TYPES:
            # token 0 and two branches: 1, 3, 5... and 2, 4, 6...
            masks = [[[0, *range(2 - i % 2, i + 1, 2)] if i else [0] for i in range(20)]]
            b = Batch([50], [20], 1, group, 64, 16, dtype, False, masks)
            pos = 50 - 20 + 7
            b.v[int(b.table[0, pos // 16]), 0, pos % 16, 5] = value
            got = b.run(ws)
            sees = torch.tensor([7 in m for m in masks[0]], device="cuda")
            assert torch.isfinite(got[~sees]).all()
            rest = torch.ones(64, dtype=torch.bool, device="cuda")
            rest[5] = False
            assert torch.isfinite(got[sees][:, :, rest]).all()
            odd = got[sees][:, :, 5].float()
            assert (torch.isnan(odd) if value != value else odd == value).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_more_tokens_than_a_tree_has(cuda, dtype) -> None:
    """The sequence has no result; the others have theirs."""
    import torch

    w = attention.Workspace()
    news = [65, 4]
    masks = [[[0]] * 65, _trees(1, [4])[0]]
    b = Batch([100, 40], news, 1, 2, 64, 16, dtype, False, masks)
    out = torch.full((69, 2, 64), 3.0, device="cuda").to(b.dtype)
    b.run(w, out=out)
    with pytest.raises(CacheError) as e:
        w.check()
    assert e.value.bits == cache_module.TOO_LONG
    alone = Batch([100, 40], news, 1, 2, 64, 16, dtype, False, masks)
    alone.starts, alone.q, alone.mask = _ints([0, 0, 4]), b.q[65:], b.mask[65:]
    assert torch.allclose(alone.run(w), out[65:], rtol=0.02, atol=0.02)
    w.check()


@pytest.mark.gpu
def test_refused_tensors(ws) -> None:
    import torch

    b = Batch([30, 20], [3, 2], 2, 2, 64, 16, "bfloat16", True, _trees(1, [3, 2]))
    s = b.scales["k_scale"]
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_scale=s.double()), dict(v_scale=s[:1]),
                dict(k_scale=s.cpu()), dict(k_scale=None, v_scale=None)):
        with pytest.raises(ValueError):
            b.run(ws, **bad)
    plain = Batch([30, 20], [3, 2], 2, 2, 64, 16, "bfloat16", False, _trees(1, [3, 2]))
    with pytest.raises(ValueError):
        plain.run(ws, k_scale=s, v_scale=s)
    mask = b.mask
    for bad in (None, mask[:4], mask.int(), mask.cpu(), mask[None]):
        b.mask = bad
        with pytest.raises(ValueError, match="mask"):
            b.run(ws)
    b.mask = mask
    b.k, b.v = b.k[..., :24].contiguous(), b.v[..., :24].contiguous()
    b.q = b.q[..., :24].contiguous()
    with pytest.raises(LaunchError, match="multiple of 16"):
        b.run(ws)


def test_branches() -> None:
    assert attention.branches([]) == []
    assert attention.branches([-1, 0, 0, 1, -1]) == [1, 0b11, 0b101, 0b1011, 0b10000]
    chain = attention.branches([*range(-1, 63)])
    assert chain[62] == (1 << 63) - 1 and chain[63] == -1
    for bad in ([0], [-1, 1], [-1, -2], [-1] * 65):
        with pytest.raises(ValueError):
            attention.branches(bad)


def _args(**over) -> AttentionArgs:
    a = AttentionArgs(q=256, k=256, v=256, out=256, starts=4, table=4, lens=4, workspace=256,
                      workspace_bytes=64 << 20, dtype=2, batch=1, queries=1, heads=1, group=1, dim=32,
                      page_size=4, pages=1, width=1, slot_rows=1, scale=1.0)
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("args,more", [
    (dict(), dict(k_scale=4)), (dict(), dict(v_scale=4)), (dict(dim=24), dict(k_scale=4, v_scale=4)),
    (dict(), dict(k_scale=2, v_scale=4)), (dict(), dict(k_scale=4, v_scale=4, k_scale_page=2)),
    (dict(), dict(k_scale=4, v_scale=4, v_scale_head=1)), (dict(), dict(mask=12)),
    (dict(starts=0), dict(mask=8)), (dict(dtype=7), dict(k_scale=4, v_scale=4)),
    (dict(k=8), dict(k_scale=4, v_scale=4)), (dict(window=-1), dict(mask=8))], ids=str)
def test_refused_by_the_c_entry(args, more) -> None:
    build_library()
    assert library().pg_attention_ex(_args(**args), AttentionMore(**more), 0) == PG_ERR_ARGUMENT
    assert b"pg_attention_ex" in library().pg_last_error()


def test_nothing_to_do() -> None:
    build_library()
    lib = library()
    assert lib.pg_attention_ex(_args(batch=0, queries=0), AttentionMore(mask=8), 0) == 0
    assert lib.pg_attention_ex(_args(batch=0, queries=0), None, 0) == 0
    assert lib.pg_attention_ex(None, None, 0) == PG_ERR_ARGUMENT
