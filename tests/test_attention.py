"""Attention over a paged cache against its definition in 64 bits.

Tolerances. With |v| <= V over the keys a query sees and its weights summing to 1, rounding each
weight to the values' type before the product moves the result by at most e V (e = 2^-8 for bf16,
2^-11 for f16), and rounding the result by e V again; the roundings fall both ways, so bf16 is
held to half of that sum (u = 2^-9). A score is a sum of `dim` products in 32
bits: with |q|, |k| about 1 a coordinate its error is under dim^(1/2) 2^-22 or 1e-5, which moves
every weight by 1e-5 of itself, and the sums over keys add less; exp2 is good to 2^-22. So the
16-bit types are held to 2 u V + 4e-5 V and f32 to 4e-5 V."""

from __future__ import annotations

import numpy as np
import pytest

from ptxgen import attention
from ptxgen.build import build_library
from ptxgen.cache import BAD_PAGE, BAD_SLOT, TOO_LONG, CacheError
from ptxgen.runtime import AttentionArgs, LaunchError, library

PG_ERR_ARGUMENT = -2
UNIT = {"float32": 0.0, "bfloat16": 2.0 ** -9, "float16": 2.0 ** -11}


class Batch:
    """A ragged batch over a cache of scattered pages. ``junk`` fills whatever no query may see:
    the rest of a last page, pages nobody holds, and (with a window) keys all queries have left."""

    def __init__(self, lens, news, heads, group, dim, page, dtype, seed=0, junk=float("nan"),
                 fused=False):
        import torch

        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = getattr(torch, dtype)
        self.lens, self.news, self.heads, self.group, self.dim = lens, news, heads, group, dim
        self.page, self.junk = page, junk
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + 2
        self.keys, self.values = [], []
        # keys and values interleaved by page, as one array would hold them
        pool = torch.full((pages, 2, heads, page, dim), junk, device="cuda", dtype=self.dtype)
        self.k, self.v = pool[:, 0], pool[:, 1]
        ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max([1, *counts]) + 1), pages + 7, device="cuda",
                                dtype=torch.int32)  # past the length: no page at all
        at = 0
        for b, n in enumerate(lens):
            mine = ids[at:at + counts[b]]
            at += counts[b]
            self.table[b, :counts[b]] = mine
            k, v = (torch.randn((heads, n, dim), device="cuda", generator=g).to(self.dtype)
                    for _ in range(2))
            self.keys.append(k)
            self.values.append(v)
            for j in range(counts[b]):
                part = slice(j * page, min(n, (j + 1) * page))
                size = part.stop - part.start
                self.k[mine[j].long(), :, :size] = k[:, part]
                self.v[mine[j].long(), :, :size] = v[:, part]
        self.lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        starts = np.concatenate([[0], np.cumsum(news)])
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        hq = heads * group
        q = torch.randn((int(starts[-1]), hq + (2 if fused else 0), dim), device="cuda",
                        generator=g)
        self.q = q.to(self.dtype)[:, :hq]

    def definition(self, window=0, sinks=0, scale=None):
        import torch

        scale = self.dim ** -0.5 if scale is None else scale
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        at = 0
        for b, (n, new) in enumerate(zip(self.lens, self.news)):
            for i in range(new):
                pos = n - new + i
                if pos < 0:
                    continue
                seen = torch.arange(pos + 1, device="cuda")
                if window:
                    seen = seen[(seen > pos - window) | (seen < sinks)]
                k, v = self.keys[b][:, seen].double(), self.values[b][:, seen].double()
                q = self.q[at + i].double().view(self.heads, self.group, self.dim)
                s = torch.einsum("hgd,hkd->hgk", q, k) * scale
                out[at + i] = (torch.softmax(s, -1) @ v).reshape(-1, self.dim)
            at += new
        return out

    def run(self, ws, decode=False, **kw):
        if decode:
            return attention.decode(self.q, self.k, self.v, self.table, self.lens_t, workspace=ws,
                                    **kw)
        return attention.prompt(self.q, self.starts, self.k, self.v, self.table, self.lens_t,
                                workspace=ws, **kw)

    def check(self, got, want):
        import torch

        top = max([1.0, *(float(v.abs().max()) for v in self.values if v.numel())])
        u = UNIT[str(self.dtype).split(".")[1]]
        got = got.double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        err = (got - want).abs().nan_to_num(0.0)
        bound = 2 * u * top + 4e-5 * top
        assert float(err.max() if err.numel() else 0.0) <= bound, (float(err.max()), bound)


@pytest.fixture(scope="module")
def ws(cuda):
    w = attention.Workspace()
    yield w
    w.check()


TYPES = ["bfloat16", "float16", "float32"]
# heads, group, dim, page
HEADS = [(2, 4, 128, 16), (1, 1, 64, 16), (3, 5, 64, 8), (1, 16, 128, 32), (2, 7, 96, 24),
         (1, 20, 128, 64), (2, 8, 32, 16), (1, 3, 256, 16), (4, 1, 128, 1), (1, 70, 64, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_decode_ragged(ws, heads, group, dim, page, dtype) -> None:
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 200, 1000, 0, 129]
    b = Batch(lens, [1] * len(lens), heads, group, dim, page, dtype, fused=True)
    b.check(b.run(ws, decode=True), b.definition())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (100, 4), (64, 70), (5000, 3), (33, 0)])
def test_decode_window_and_sinks(ws, window, sinks, dtype) -> None:
    lens = [1, 2, 5, 31, 99, 100, 101, 170, 300, 513, 0, 4999]
    b = Batch(lens, [1] * len(lens), 2, 4, 64, 16, dtype, seed=window)
    b.check(b.run(ws, decode=True, window=window, sinks=sinks), b.definition(window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,most,heads,group", [(1, 40000, 1, 8), (3, 9001, 2, 4),
                                                    (40, 700, 4, 2), (150, 90, 8, 1)])
def test_decode_long_and_split(ws, batch, most, heads, group, dtype) -> None:
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(0, most, batch)]
    lens[-1] = most
    b = Batch(lens, [1] * batch, heads, group, 128, 16, dtype)
    got = b.run(ws, decode=True)
    b.check(got, b.definition())
    import torch

    for _ in range(3):  # the parts join in one order, whichever arrives last
        assert torch.equal(b.run(ws, decode=True), got)
    b.check(b.run(ws, decode=True, max_len=most), b.definition())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_prompt_ragged(ws, heads, group, dim, page, dtype) -> None:
    lens = [1, 40, 0, 130, 300, 300, 7, 129]
    news = [1, 40, 0, 3, 150, 0, 9, 128]  # none, all, more than there are
    b = Batch(lens, news, heads, group, dim, page, dtype, fused=True)
    b.check(b.run(ws), b.definition())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page", HEADS)
def test_prompt_few_tokens(ws, heads, group, dim, page, dtype) -> None:
    """A few drafted tokens a sequence, none of some, more than there are of others."""
    lens = [1, 40, 0, 130, 300, 301, 2, 129, 64, 1000]
    news = [1, 4, 2, 3, 0, 5, 4, 1, 2, 6]
    b = Batch(lens, news, heads, group, dim, page, dtype, fused=True)
    b.check(b.run(ws), b.definition())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (16, 0), (100, 4), (64, 70), (257, 5),
                                          (5000, 3)])
def test_prompt_few_tokens_window_and_sinks(ws, window, sinks, dtype) -> None:
    lens, news = [700, 3, 1400, 91, 5000], [5, 3, 1, 4, 7]
    b = Batch(lens, news, 2, 3, 64, 16, dtype, seed=window)
    b.check(b.run(ws, window=window, sinks=sinks), b.definition(window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (100, 4), (128, 130), (257, 5),
                                          (5000, 3)])
def test_prompt_window_and_sinks(ws, window, sinks, dtype) -> None:
    lens, news = [700, 90, 1400], [300, 90, 5]
    b = Batch(lens, news, 2, 2, 64, 16, dtype, seed=window)
    b.check(b.run(ws, window=window, sinks=sinks), b.definition(window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,news", [([20000], [3]), ([5000, 6000], [1, 17]), ([1000], [1000])])
def test_prompt_few_rows_over_long_lengths(ws, lens, news, dtype) -> None:
    import torch

    b = Batch(lens, news, 1, 4, 128, 16, dtype)
    got = b.run(ws)
    b.check(got, b.definition())
    for _ in range(3):
        assert torch.equal(b.run(ws), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf")])
def test_what_lies_in_masked_places_does_not_matter(ws, junk, dim, dtype) -> None:
    """Keys that some queries see and others must not hold junk: those that see it get the
    formula's NaN or infinity, the others are untouched."""
    import torch

    lens, news, window = [260, 140], [200, 3], 40
    b = Batch(lens, news, 2, 2, dim, 16, dtype, junk=junk)
    clean = b.run(ws, window=window, sinks=2)
    place = 150  # a key of sequence 0 that queries 150..189 see
    page, row = int(b.table[0, place // 16]), place % 16
    b.v[page, :, row, 3] = junk
    b.values[0][:, place, 3] = junk
    got = b.run(ws, window=window, sinks=2)
    want = b.definition(window, 2)
    pos = torch.arange(60, 260, device="cuda")
    hit = (pos >= place) & (pos < place + window)
    sees = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    sees[:200, :, 3] = hit[:, None]
    assert torch.equal(torch.isfinite(got), ~sees)
    assert torch.equal(got[sees].double().nan_to_num(7.0), want[sees].nan_to_num(7.0))
    assert torch.equal(got[~sees], clean[~sees])
    # a key instead of a value: only the scores of those that see it
    b.v[page, :, row, 3] = 0
    b.k[page, :, row, 5] = float("nan")
    got = b.run(ws, window=window, sinks=2)
    assert torch.equal(torch.isnan(got).any(-1).any(-1)[:200], hit)
    assert not torch.isnan(got[200:]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 5)])
def test_masked_places_of_a_few_tokens(ws, dim, page, dtype) -> None:
    """Drafted tokens of which the first must not see the last one's key and value, nor the last
    what has left its window."""
    import torch

    lens, news, window = [90, 333, 64], [4, 3, 4], 20
    b = Batch(lens, news, 2, 2, dim, page, dtype, junk=float("nan"))
    clean = b.run(ws, window=window, sinks=1)
    b.check(clean, b.definition(window, 1))
    # a key that token 0 of sequence 0 sees and its later ones have left; one that only the last
    # of sequence 1 sees; and sequence 2's whole last token
    for s, place in ((0, 67), (1, 332), (2, 63)):
        at, row = int(b.table[s, place // page]), place % page
        b.v[at, :, row, 7] = float("inf")
        b.values[s][:, place, 7] = float("inf")
    got, want = b.run(ws, window=window, sinks=1), b.definition(window, 1)
    hit = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    hit[[0, 6, 10], :, 7] = True
    assert torch.equal(torch.isfinite(want), ~hit)
    assert torch.equal(torch.isfinite(got), ~hit) and (got[hit] == float("inf")).all()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("decode", [False, True])
def test_large_scores(ws, decode, dtype) -> None:
    """Scores of some hundreds: weights that are 0 or 1, and a maximum that keeps growing."""
    import torch

    n = 900
    b = Batch([n], [1 if decode else 70], 1, 2, 64, 16, dtype)
    ramp = torch.linspace(-30, 30, n, device="cuda")[None, :, None]
    k = (ramp * torch.sign(b.q[0, 0])[None, None]).to(b.dtype)
    b.keys[0] = k
    for j in range(-(-n // 16)):
        part = k[:, 16 * j:16 * j + 16]
        b.k[int(b.table[0, j]), :, :part.shape[1]] = part
    want = b.definition(scale=0.25)
    got = b.run(ws, decode=decode, scale=0.25).double()
    # a score near 700 has an error of 700 2^-24 times a few, so weights one of 2e-3 at most
    top = float(b.values[0].abs().max())
    assert float((got - want).abs().max()) <= (2 * UNIT[dtype] + 2e-3) * top


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_slots_streams_and_outputs(ws, dtype) -> None:
    import torch

    lens = [100, 37, 64, 250]
    b = Batch(lens, [1] * 4, 2, 4, 64, 16, dtype)
    full = b.run(ws, decode=True)
    slots = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    wide = torch.full((2, 10, 64), 7.0, device="cuda", dtype=b.dtype)
    side, mine = torch.cuda.Stream(), attention.Workspace()
    torch.cuda.synchronize()
    got = attention.decode(b.q[[3, 1]], b.k, b.v, b.table, b.lens_t, slots=slots, workspace=mine,
                           out=wide[:, 1:9], stream=side.cuda_stream)
    side.synchronize()
    b.check(got, b.definition()[[3, 1]])
    assert (wide[:, 0] == 7).all() and (wide[:, 9] == 7).all()
    b.check(full, b.definition())
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    got = attention.prompt(b.q[[3, 1]], starts, b.k, b.v, b.table, b.lens_t, slots=slots,
                           workspace=mine)
    b.check(got, b.definition()[[3, 1]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("decode", [False, True])
def test_what_only_the_device_can_see(cuda, decode, dtype) -> None:
    """A page id, slot, length or starts out of range: left out, and reported."""
    import torch

    w = attention.Workspace()
    b = Batch([100, 60], [1, 1], 1, 2, 64, 16, dtype)
    table = b.table.clone()
    table[0, 2] = 12345
    args = (b.q, b.k, b.v) if decode else (b.q, b.starts, b.k, b.v)
    call = attention.decode if decode else attention.prompt
    got = call(*args, table, b.lens_t, workspace=w)
    with pytest.raises(CacheError) as e:
        w.check()
    assert e.value.bits == BAD_PAGE
    b.check(got[1:], b.definition()[1:])
    slots = torch.tensor([5, 1], dtype=torch.int32, device="cuda")
    got = call(*args, b.table, b.lens_t, slots=slots, workspace=w)
    with pytest.raises(CacheError) as e:
        w.check()
    assert e.value.bits == BAD_SLOT
    assert not got[0].any()
    b.check(got[1:], b.definition()[1:])
    lens = torch.tensor([100, 60000], dtype=torch.int32, device="cuda")
    got = call(*args, b.table, lens, workspace=w)
    with pytest.raises(CacheError) as e:
        w.check()
    assert e.value.bits & TOO_LONG
    b.check(got[:1], b.definition()[:1])
    if not decode:
        got = attention.prompt(b.q, torch.tensor([0, 1, 9], dtype=torch.int32, device="cuda"),
                               b.k, b.v, b.table, b.lens_t, workspace=w)
        with pytest.raises(CacheError) as e:
            w.check()
        assert e.value.bits == TOO_LONG
        b.check(got[:1], b.definition()[:1])
    w.check()


@pytest.mark.gpu
def test_refusals(ws) -> None:
    import torch

    b = Batch([100], [1], 2, 2, 64, 16, "bfloat16")
    q, k, v, t, n = b.q, b.k, b.v, b.table, b.lens_t
    for match, args in [("q: want", (q[0], k, v, t, n)), ("k: want", (q, k.float(), v, t, n)),
                        ("v: want", (q, k, v[:, :1], t, n)),
                        ("multiple", (q[:, :3], k, v, t, n)),
                        ("table", (q, k, v, t.long(), n)), ("lens", (q, k, v, t, n.float())),
                        ("sequences", (q.expand(2, -1, -1), k, v, t, n)),
                        ("rows of one page", (q, k.transpose(1, 2), v.transpose(1, 2), t, n))]:
        with pytest.raises(ValueError, match=match):
            attention.decode(*args, workspace=ws)
    with pytest.raises(ValueError, match="starts"):
        attention.prompt(q, b.starts.long(), k, v, t, n, workspace=ws)
    with pytest.raises(ValueError, match="out"):
        attention.decode(q, k, v, t, n, workspace=ws, out=q.float())
    with pytest.raises(LaunchError, match="window"):
        attention.decode(q, k, v, t, n, workspace=ws, window=-1)
    with pytest.raises(LaunchError, match="sinks"):
        attention.decode(q, k, v, t, n, workspace=ws, sinks=-1)
    odd = Batch([10], [1], 1, 1, 20, 16, "bfloat16")
    with pytest.raises(LaunchError, match="multiple"):
        odd.run(ws, decode=True)
    large = Batch([10], [1], 1, 1, 264, 16, "bfloat16")
    with pytest.raises(LaunchError, match="at most 256"):
        large.run(ws, decode=True)
    none = attention.decode(q[:0], k, v, t[:0], n[:0], workspace=ws)
    assert none.shape == (0, 4, 64)


def test_bad_arguments_are_refused_before_any_cuda_call() -> None:
    build_library()
    lib = library()
    at = 1 << 20  # never dereferenced: every case fails its argument check first

    def args(**other):
        fields = dict(q=at, k=at, v=at, out=at, starts=0, slots=0, table=at, lens=at, workspace=at,
                      workspace_bytes=64 << 20, q_token=256, q_head=128, out_token=256,
                      out_head=128, k_page=4096, k_head=2048, v_page=4096, v_head=2048,
                      table_stride=4, dtype=2, batch=2, queries=2, heads=2, group=1, dim=64,
                      page_size=16, pages=8, width=4, slot_rows=2, window=0, sinks=0, max_len=0,
                      scale=0.125)
        return AttentionArgs(**{**fields, **other})

    assert lib.pg_attention(None, 0) == PG_ERR_ARGUMENT
    for other in [dict(dtype=0), dict(dtype=5), dict(batch=-1), dict(heads=0), dict(group=0),
                  dict(dim=0), dict(dim=12), dict(dim=264), dict(page_size=0), dict(pages=0),
                  dict(width=0), dict(width=1 << 28), dict(slot_rows=0), dict(window=-1),
                  dict(sinks=-1), dict(max_len=-1), dict(scale=float("nan")), dict(queries=3),
                  dict(q=0), dict(out=0), dict(table=0), dict(lens=0), dict(workspace=0),
                  dict(q=at + 8), dict(out=at + 2), dict(k_page=4100), dict(v_head=2044),
                  dict(q_token=130), dict(out_head=130), dict(starts=at + 2), dict(lens=at + 1),
                  dict(workspace=at + 16), dict(workspace_bytes=1 << 20),
                  dict(heads=70000), dict(starts=at, queries=1 << 30, group=4)]:
        assert lib.pg_attention(args(**other), 0) == PG_ERR_ARGUMENT, other
    assert b"queries" in lib.pg_last_error()
    assert lib.pg_attention(args(batch=0, queries=0), 0) == 0  # nothing to do, no CUDA call
