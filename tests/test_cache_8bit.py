"""The paged cache in 8 bits: what is written, read back and moved. A row's scale is one f32 division
and its numbers are quotients rounded to whole ones, so all must be equal to the definition's, which
divides in 64 bits: the quotient of two f32 numbers is a half there only if it is one. Reading back
multiplies in f32 and rounds to the type asked for, as numpy and torch do, so that is equal too."""

from __future__ import annotations

import numpy as np
import pytest

from ptxgen import cache as cache_module
from ptxgen.build import build_library
from ptxgen.cache import CacheError, PagedCache
from ptxgen.runtime import Cache, Rows, Scales, library

PG_ERR_ARGUMENT = -2
TYPES = ["float32", "bfloat16", "float16"]


def _ints(*x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def quantised(x):
    """(q, scale) of the rows of x [..., dim], f32 numbers on the host."""
    x = x.astype(np.float32)
    finite = np.isfinite(x).all(-1)
    with np.errstate(invalid="ignore"):
        scale = np.where(finite, np.abs(x).max(-1) / np.float32(127), np.float32(np.nan)).astype(np.float32)
        some = finite & (scale > 0)
        q = np.rint(x.astype(np.float64) / np.where(some, scale, 1).astype(np.float64)[..., None])
    return np.where(some[..., None], np.clip(q, -127, 127), 0).astype(np.int8), scale


def _rows(rng, tokens, heads, dim, kind):
    x = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    x *= np.exp(rng.standard_normal((tokens, heads, 1))).astype(np.float32)
    if kind == "halves":  # numbers that stand exactly between two, and their neighbours
        x = rng.integers(-254, 255, x.shape).astype(np.float32) / 2
        x[..., 0] = 127.0
        x *= (2.0 ** rng.integers(-9, 6, (tokens, heads, 1))).astype(np.float32)
        x = np.where(rng.random(x.shape) < 0.2, np.nextafter(x, np.float32(0)), x)
    elif kind == "odd rows":
        flat = x.reshape(-1, dim)
        flat[::7] = 0.0
        flat[1::7, 0] = np.nan
        flat[2::7, -1] = np.inf
        flat[3::7, dim // 2] = -np.inf
        flat[4::7] = -flat[4::7, :1]
        flat[5::7, 1:] = 0.0
    elif kind == "tiny":
        x *= np.float32(1e-38)
        x.reshape(-1, dim)[::3] *= np.float32(1e-5)
    elif kind == "huge":
        x = np.clip(x, -3, 3) * np.float32(1e38)
    return x


# layers, pages, heads, page, dim
SHAPES = [(1, 40, 1, 16, 64), (2, 57, 3, 8, 128), (1, 200, 2, 5, 16), (1, 60, 5, 24, 96),
          (1, 90, 1, 64, 512), (2, 400, 2, 1, 48), (1, 30, 2, 16, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["normal", "halves", "odd rows", "tiny", "huge"])
@pytest.mark.parametrize("layers,pages,heads,page,dim", SHAPES)
def test_written_and_read_back(cuda, layers, pages, heads, page, dim, kind, dtype) -> None:
    import torch

    if dtype == "float16" and kind in ("tiny", "huge"):
        kind = "halves"
    rng = np.random.default_rng(dim)
    slots, counts = [2, 0, 3], [29, 1, 17]
    cache = PagedCache.allocate(layers, pages, heads, page, dim, 5, 60, dtype=torch.int8)
    cache.k.fill_(99)
    cache.v.fill_(-99)
    cache.k_scale.fill_(7.0)
    cache.v_scale.fill_(9.0)
    t = getattr(torch, dtype)
    fused = torch.from_numpy(_rows(rng, 50, 2 * heads, dim, kind)).to(t).cuda()
    k, v = fused[:, :heads], fused[:, heads:]  # three rows that no slot has
    starts = _ints(0, 29, 30, 47)
    cache.extend(_ints(*slots), starts)
    layer = layers - 1
    cache.write(layer, _ints(*slots), starts, k, v)
    wide = torch.full((50, 2 * heads + 1, dim), 5.0, device="cuda").to(t)
    out = cache.read(layer, _ints(*slots), starts, 50, dtype=t,
                     out=(wide[:, 1:heads + 1], wide[:, heads + 1:]))
    table = cache.table.tolist()
    used = np.zeros((pages, page), bool)
    for rows, got, q_in, s_in, plain in ((k, out[0], cache.k, cache.k_scale, 99),
                                         (v, out[1], cache.v, cache.v_scale, -99)):
        q, scale = quantised(rows.float().cpu().numpy())
        held, scales = q_in.cpu().numpy(), s_in.cpu().numpy()
        at = 0
        for s, n in zip(slots, counts):
            for pos in range(n):
                p, r = table[s][pos // page], pos % page
                used[p, r] = True
                assert np.array_equal(held[layer, p, :, r], q[at]), (s, pos)
                assert np.array_equal(scales[layer, p, :, r], scale[at], equal_nan=True), (s, pos)
                at += 1
        # nothing else is touched
        assert (held[layer].transpose(0, 2, 1, 3)[~used] == plain).all()
        assert layers == 1 or (held[0] == plain).all()
        want = (torch.from_numpy(q.astype(np.float32)) * torch.from_numpy(scale)[..., None]).to(t)
        assert torch.equal(got[:47].cpu().nan_to_num(1234.0), want[:47].nan_to_num(1234.0))
        assert (got[47:] == 5.0).all()
    assert (wide[:, 0] == 5.0).all()
    new = cache.read(layer, _ints(*slots), starts, 47)
    assert new[0].dtype is torch.bfloat16 and new[0].shape == (47, heads, dim)
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_of_other_caches_are_read_back_as_they_are(cuda, dtype) -> None:
    import torch

    t = getattr(torch, dtype)
    cache = PagedCache.allocate(2, 30, 3, 8, 40, 4, 10, dtype=t)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((31, 3, 40), device="cuda", generator=g).to(t) for _ in range(2))
    slots, starts = _ints(1, 3), _ints(0, 20, 31)
    cache.extend(slots, starts)
    cache.write(1, slots, starts, k, v)
    got = cache.read(1, slots, starts, 31)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    # the last few tokens of one of them
    got = cache.read(1, _ints(1), _ints(0, 7), 7)
    assert torch.equal(got[0], k[13:20]) and torch.equal(got[1], v[13:20])
    with pytest.raises(ValueError, match="dtype"):
        cache.read(1, slots, starts, 31, dtype=torch.float16)
    cache.check()


@pytest.mark.gpu
def test_page_operations_take_the_scales_along(cuda) -> None:
    import torch

    cache = PagedCache.allocate(3, 64, 2, 8, 32, 10, 8, dtype=torch.int8)
    g = torch.Generator(device="cuda").manual_seed(2)
    slots, starts = _ints(0, 1, 2, 3), _ints(0, 21, 24, 40, 64)
    cache.extend(slots, starts)
    rows = [[torch.randn((64, 2, 32), device="cuda", generator=g) * 2 ** i for i in range(2)]
            for _ in range(3)]

    def same(of, at) -> None:
        for layer in range(3):
            n = [21, 3, 16, 24][at]
            lo = [0, 21, 24, 40][at]
            got = cache.read(layer, _ints(of), _ints(0, n), n, dtype=torch.float32)
            for a, b in zip(got, rows[layer]):
                q, s = quantised(b[lo:lo + n].cpu().numpy())
                assert np.array_equal(a.cpu().numpy(), q.astype(np.float32) * s[..., None])

    for layer in range(3):
        cache.write(layer, slots, starts, *rows[layer])
    cache.fork(_ints(0, 1, 3), _ints(5, 6, 7))
    for of, at in ((5, 0), (6, 1), (7, 3)):
        same(of, at)
    cache.free(_ints(0, 2))
    cache.compact()
    for of, at in ((5, 0), (6, 1), (7, 3), (1, 1), (3, 3)):
        same(of, at)
    # a whole page elsewhere, and the table after it
    page, free = int(cache.table[3, 0]), int((cache.refs == 0).nonzero()[0])
    cache.copy_pages(_ints(page), _ints(free))
    cache.table[3, 0] = free
    same(3, 3)
    cache.check()


@pytest.mark.gpu
def test_strided_scales_on_another_stream_and_captured(cuda) -> None:
    """A layer's scales may lie apart, as a part of a larger allocation."""
    import torch

    k, v = (torch.zeros((2, 20, 2, 8, 16), dtype=torch.int8, device="cuda") for _ in range(2))
    wide = torch.full((2, 2, 20, 5, 8), 3.0, device="cuda")
    refs = torch.zeros(20, dtype=torch.int32, device="cuda")
    table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    cache = PagedCache(k, v, refs, table, lens, wide[0, :, :, 1:3], wide[1, :, :, 1:3])
    g = torch.Generator(device="cuda").manual_seed(3)
    x, y = (torch.randn((9, 2, 16), device="cuda", generator=g) for _ in range(2))
    slots, starts = _ints(2), _ints(0, 9)
    cache.extend(slots, starts)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    cache.write(1, slots, starts, x, y, stream=side.cuda_stream)
    got = cache.read(1, slots, starts, 9, dtype=torch.float32, stream=side.cuda_stream)
    side.synchronize()

    def same() -> None:
        for a, b in zip(got, (x, y)):
            q, s = quantised(b.cpu().numpy())
            assert np.array_equal(a.cpu().numpy(), q.astype(np.float32) * s[..., None])

    same()
    assert (wide[:, :, :, [0, 3, 4]] == 3.0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(1, slots, starts, x, y)
        got = cache.read(1, slots, starts, 9, dtype=torch.float32)
    x.normal_(generator=g)
    graph.replay()
    same()
    cache.check()


@pytest.mark.gpu
def test_what_only_the_device_sees(cuda) -> None:
    import torch

    cache = PagedCache.allocate(1, 4, 1, 4, 16, 3, 4, dtype=torch.int8)
    rows = torch.ones((8, 1, 16), device="cuda")
    cache.extend(_ints(0), _ints(0, 8))
    cache.write(0, _ints(0), _ints(0, 8), rows, rows)
    cache.check()
    before = cache.k.clone(), cache.k_scale.clone()
    out = torch.full((8, 1, 16), 5.0, device="cuda"), torch.full((8, 1, 16), 5.0, device="cuda")
    for slots, starts, bits in ((_ints(7), _ints(0, 8), cache_module.BAD_SLOT),
                                (_ints(1), _ints(0, 8), cache_module.BAD_PAGE),
                                (_ints(0), _ints(0, 9), cache_module.TOO_LONG | cache_module.BAD_PAGE)):
        cache.read(0, slots, starts, 8, dtype=torch.float32, out=out)
        with pytest.raises(CacheError) as e:
            cache.check()
        assert e.value.bits == bits
    assert (out[0][1:] == 5.0).logical_or(out[0][1:] == 1.0).all()
    for slots, bits in ((_ints(7), cache_module.BAD_SLOT), (_ints(1), cache_module.BAD_PAGE)):
        cache.write(0, slots, _ints(0, 8), 2 * rows, rows)
        with pytest.raises(CacheError) as e:
            cache.check()
        assert e.value.bits == bits
    cache.extend(_ints(0), _ints(0, 100))  # refused, and the write behind it leaves its rows out
    cache.write(0, _ints(0), _ints(0, 8), 2 * rows, rows)
    with pytest.raises(CacheError) as e:
        cache.check()
    assert e.value.bits == cache_module.TOO_LONG | cache_module.REFUSED
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.k_scale, before[1])


@pytest.mark.gpu
def test_refused_tensors(cuda) -> None:
    import torch

    k = torch.zeros((1, 4, 2, 8, 32), dtype=torch.int8, device="cuda")
    refs = torch.zeros(4, dtype=torch.int32, device="cuda")
    table, lens = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), _ints(0)
    s = torch.zeros((1, 4, 2, 8), device="cuda")
    PagedCache(k, k.clone(), refs, table, lens, s, s.clone())
    for bad in ((None, None), (s, None), (None, s), (s, s.double()), (s[:, :3], s), (s, s.cpu()),
                (s, s.transpose(0, 1).contiguous().transpose(0, 1).expand(1, 4, 2, 8)[..., :8].half()),
                (torch.zeros((1, 4, 2, 16), device="cuda")[..., ::2], s)):
        with pytest.raises(ValueError, match="scale"):
            PagedCache(k, k.clone(), refs, table, lens, *bad)
    f = torch.zeros((1, 4, 2, 8, 32), device="cuda")
    with pytest.raises(ValueError, match="int8"):
        PagedCache(f, f.clone(), refs, table, lens, s, s.clone())
    cache = PagedCache(k, k.clone(), refs, table, lens, s, s.clone())
    rows = torch.zeros((3, 2, 32), device="cuda")
    for a, b in ((rows, rows.half()), (rows.double(), rows.double()), (rows.to(torch.int8),) * 2,
                 (rows[..., :16], rows), (rows, rows[:2])):
        with pytest.raises(ValueError):
            cache.write(0, _ints(0), _ints(0, 3), a, b)
    for more in (dict(dtype=torch.int8), dict(out=(rows, rows)), dict(tokens=4, out=(rows, rows))):
        with pytest.raises(ValueError):
            cache.read(0, _ints(0), _ints(0, 3), **{"tokens": 3, **more})


def _c(**over):
    c = Cache(k=16, v=16, layer_stride=64, page_stride=64, head_stride=64, refs=4, table=4, lens=4,
              status=4, scratch=4, refused=4, table_stride=2, scratch_words=1000, layers=1, pages=4, heads=1,
              page_size=4, row_bytes=16, slots=2, width=2)
    for n, v in over.items():
        setattr(c, n, v)
    return c


@pytest.mark.parametrize("entry", ["write", "read", "copy", "fork", "compact", "keep"])
@pytest.mark.parametrize("scales", [None, dict(k=0), dict(v=0), dict(k=2), dict(layer_stride=2),
                                    dict(page_stride=6), dict(head_stride=1), "large"], ids=str)
def test_refused_by_the_c_entries(entry, scales) -> None:
    build_library()
    lib, rows = library(), Rows(16, 16, 16)
    if scales is None and entry in ("read", "keep"):
        return  # such a cache may have none
    c = _c(row_bytes=528) if scales == "large" else _c()
    s = None if scales is None else Scales(k=4, v=4, layer_stride=4, page_stride=4, head_stride=4)
    for n, v in (scales if isinstance(scales, dict) else {}).items():
        setattr(s, n, v)
    rc = {"write": lambda: lib.pg_cache8_write(c, s, 0, 4, 4, 1, 1, 3, rows, rows, 0),
          "read": lambda: lib.pg_cache_read(c, s, 0, 4, 4, 1, 1, 3, rows, rows, 0),
          "copy": lambda: lib.pg_cache8_copy(c, s, 4, 4, 1, 0),
          "fork": lambda: lib.pg_cache8_fork(c, s, 4, 4, 1, 0),
          "compact": lambda: lib.pg_cache8_compact(c, s, 0),
          "keep": lambda: lib.pg_cache_keep(c, s, 4, 4, 8, 1, 0)}[entry]()
    assert rc == PG_ERR_ARGUMENT


@pytest.mark.parametrize("args", [
    dict(dtype=0), dict(dtype=9), dict(layer=1), dict(layer=-1), dict(tokens=-1), dict(n=-1),
    dict(n=3), dict(slots=0), dict(starts=2), dict(rows=Rows(0, 16, 16)), dict(rows=Rows(16, 8, 16)),
    dict(rows=Rows(16, 16, 8)), dict(cache=_c(k=0)), dict(cache=_c(row_bytes=24)),
    dict(cache=_c(refused=0)), dict(cache=None)], ids=lambda a: "-".join(a))
def test_refused_rows(args) -> None:
    build_library()
    lib = library()
    of = dict(cache=_c(), layer=0, slots=4, starts=4, n=1, tokens=1, dtype=3, rows=Rows(16, 16, 16))
    of |= args
    s = Scales(k=4, v=4, layer_stride=4, page_stride=4, head_stride=4)
    for fn in (lib.pg_cache8_write, lib.pg_cache_read):
        assert fn(of["cache"], s, of["layer"], of["slots"], of["starts"], of["n"], of["tokens"],
                  of["dtype"], of["rows"], of["rows"], 0) == PG_ERR_ARGUMENT


def test_nothing_to_do() -> None:
    build_library()
    lib, c, rows = library(), _c(), Rows(16, 16, 16)
    s = Scales(k=4, v=4, layer_stride=4, page_stride=4, head_stride=4)
    assert lib.pg_cache8_write(c, s, 0, 0, 0, 0, 5, 3, rows, rows, 0) == 0
    assert lib.pg_cache8_write(c, s, 0, 4, 4, 1, 0, 3, rows, rows, 0) == 0
    assert lib.pg_cache_read(c, s, 0, 4, 4, 1, 0, 3, rows, rows, 0) == 0
    assert lib.pg_cache_read(c, None, 0, 4, 4, 1, 0, 0, rows, rows, 0) == 0
    assert lib.pg_cache8_copy(c, s, 0, 0, 0, 0) == lib.pg_cache8_fork(c, s, 0, 0, 0, 0) == 0
    assert lib.pg_cache_keep(c, s, 0, 0, 0, 0, 0) == 0
    assert lib.pg_cache_keep(c, None, 4, 4, 0, 1, 0) == PG_ERR_ARGUMENT
    assert lib.pg_cache_keep(c, None, 4, 4, 12, 1, 0) == PG_ERR_ARGUMENT
