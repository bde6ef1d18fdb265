"""Drawn tokens and their log probabilities against the definition in 64 bits.

Tolerances. A token has none: weights and sums are 64-bit on both sides, and a token changes only where a
target falls within the sums' rounding (about 1e-14 of them) of a border, or stands exactly on one, where
the sums are of whole numbers and exact. A log probability is the log of two such sums' quotient, rounded
once: 2^-24 of itself, and 1e-12 where it is next to 0."""

from __future__ import annotations

import numpy as np
import pytest

from ptxgen import sampling
from ptxgen.build import build_library
from ptxgen.runtime import LaunchError, SampleArgs, library

PG_ERR_ARGUMENT = -2
LOWEST = float(np.finfo(np.float32).min)


def _draw(x, u, t, k, p, least):
    """(token, logp, how many are kept) of one row, by the definition."""
    x = x.astype(np.float64)
    m = x.max() if x.size else np.nan
    if not (np.isfinite(m) and t >= 0 and p == p and least <= 1 and u == u):
        return -1, np.nan, 0
    if t == 0:
        return int(x.argmax()), 0.0, 1
    with np.errstate(over="ignore"):
        w = np.where(x > -np.inf, np.exp(np.maximum(x - m, LOWEST * 2) / t), 0.0)
    order = np.lexsort((np.arange(x.size), -x))
    s = w[order]
    n = x.size
    if 0 < k < n:
        n = k
    if p < 1:
        upto = s[:n].cumsum()
        n = int((upto - s[:n] < p * upto[-1]).sum())
    if least > 0:
        n = min(n, int((s >= least).sum()))
    n = max(n, 1)
    keep = np.zeros(x.size, dtype=bool)
    keep[order[:n]] = True
    w = np.where(keep, w, 0.0)
    c = w.cumsum()
    past = (c > max(u, 0.0) * c[-1]).nonzero()[0]
    at = int(past[0]) if past.size else int((w > 0).nonzero()[0][-1])
    return at, float(np.log(w[at] / c[-1])), n


def _check(x, u, dtype, stride=None, offset=0, **settings):
    import torch

    rows, vocab = x.shape
    wide = torch.full((rows, stride or vocab), float("nan"), device="cuda").to(dtype)
    logits = wide[:, offset:offset + vocab]
    logits.copy_(torch.from_numpy(x))
    exactly = logits.float().cpu().numpy()
    given = {n: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v
             for n, v in settings.items()}
    r = sampling.sample(logits, torch.from_numpy(u).cuda(), **given)
    got, logp = r.tokens.cpu().numpy(), r.logp.cpu().numpy()
    none = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    rows_of = {n: np.broadcast_to(np.asarray(settings.get(n, d), np.int32 if n == "top_k" else
                                             np.float32), (rows,)) for n, d in none.items()}
    for i in range(rows):
        at, lp, n = _draw(exactly[i], float(u[i]), *(float(rows_of[m][i]) if m != "top_k" else
                                                     int(rows_of[m][i]) for m in none))
        what = (i, n, {m: rows_of[m][i] for m in none}, u[i])
        assert got[i] == at, (what, got[i], at)
        np.testing.assert_allclose(logp[i], lp, rtol=2.0 ** -23.9, atol=1e-12, err_msg=str(what))


def _some(rng, rows):
    """Settings of all kinds, a row each."""
    return dict(temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.5, 20.0], rows).astype(np.float32),
                top_k=rng.choice([0, 0, 1, 2, 13, 600, 5000], rows).astype(np.int32),
                top_p=rng.choice([1.0, 1.0, 0.05, 0.5, 0.9, 0.999], rows).astype(np.float32),
                min_p=rng.choice([0.0, 0.0, 0.001, 0.1, 1.0], rows).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 500, 4097, 8193, 32001, 50257])
def test_all_limits_together(cuda, vocab, dtype) -> None:
    import torch

    rng = np.random.default_rng(vocab)
    rows = 40 if vocab < 10000 else 24
    x = (rng.standard_normal((rows, vocab)) * rng.choice([0.1, 1, 3], (rows, 1))).astype(np.float32)
    _check(x, rng.random(rows, dtype=np.float32), getattr(torch, dtype), vocab + 11, 3,
           **_some(rng, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,vocab", [("float32", 128256), ("bfloat16", 128256),
                                         ("float32", 200001), ("float16", 400003)])
def test_vocabularies_cut_in_parts(cuda, dtype, vocab) -> None:
    """The last two have parts that do not stay in shared memory."""
    import torch

    rng = np.random.default_rng(1)
    x = (rng.standard_normal((7, vocab)) * 2.5).astype(np.float32)
    _check(x, rng.random(7, dtype=np.float32), getattr(torch, dtype), **_some(rng, 7))


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [dict(top_k=700), dict(top_k=1), dict(top_p=0.97),
                                   dict(min_p=0.02), dict(temperature=0.0), dict()])
def test_many_rows_with_one_setting(cuda, limit) -> None:
    import torch

    rng = np.random.default_rng(2)
    x = (rng.standard_normal((700, 3001)) * 2).astype(np.float32)
    _check(x, rng.random(700, dtype=np.float32), torch.bfloat16, **limit)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [1, 2, 9, 63, 513, 4097, 8192, 50257, 150001])
def test_many_rows_without_limits(cuda, vocab, dtype) -> None:
    """One block a row; rows that are no ordinary ones among them."""
    import torch

    rng = np.random.default_rng(vocab)
    rows = 160
    x = (rng.standard_normal((rows, vocab)) * rng.choice([0.1, 1, 3], (rows, 1))).astype(np.float32)
    x[3, rng.random(vocab) < 0.9] = -np.inf
    x[4, :-1] = -np.inf
    x[5, 1:] = -np.inf
    x[6, vocab // 2] = np.nan
    x[7, vocab - 1] = np.inf
    x[8] = -np.inf
    x[9] = np.linspace(0, 2000, vocab)  # later ones 2^500 times as large, and more
    x[10] = x[9][::-1]
    x[11, :vocab // 3] = -np.inf
    x[12] = 7.0
    x[13] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[14] += 30000
    x[15] *= 1e4
    x[16, vocab // 2:] = 60000
    u = rng.random(rows, dtype=np.float32)
    u[20:30] = [0.0, -0.0, 1e-38, 2.0 ** -60, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan, 0.5]
    u[30:34], x[30:34, 0] = [0.0, 1e-38, 1e-30, 0.999], -np.inf
    t = rng.choice([0.3, 0.7, 1.0, 1.0, 1.5, 20.0], rows).astype(np.float32)
    t[40:50] = [0.0, 1e-38, 1e-45, 1e-6, 1e30, 3e38, np.inf, -1.0, np.nan, 1e6]
    _check(x, u, getattr(torch, dtype), vocab + 11, 3, temperature=t)
    _check(x, u, getattr(torch, dtype), temperature=0.9)


@pytest.mark.gpu
def test_a_captured_draw_without_limits(cuda) -> None:
    import torch

    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((300, 9001), device="cuda", generator=g).half()
    u = torch.rand(300, device="cuda", generator=g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sampling.sample(x, u)
    for _ in range(2):
        x.normal_(generator=g)
        u.uniform_(generator=g)
        graph.replay()
        want = sampling.sample(x, u, top_k=torch.zeros(300, dtype=torch.int32, device="cuda"))
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logp, want.logp)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "few values", "masked", "lowest", "one finite", "far",
                                  "tiny", "zeros of both signs", "one above"])
def test_rows_that_are_not_spread(cuda, kind) -> None:
    import torch

    rng = np.random.default_rng(3)
    rows, vocab = 30, 6007
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    if kind == "equal":
        x[:] = rng.standard_normal((rows, 1))
    elif kind == "few values":
        x = np.round(x)
    elif kind == "masked":
        x[rng.random(x.shape) < 0.9] = -np.inf
    elif kind == "lowest":
        x[rng.random(x.shape) < 0.9] = LOWEST
    elif kind == "one finite":
        x[:] = -np.inf
        x[np.arange(rows), rng.integers(0, vocab, rows)] = 5.0
    elif kind == "far":
        x *= np.float32(1e37)
    elif kind == "tiny":
        x *= np.float32(1e-42)
    elif kind == "zeros of both signs":
        x = np.where(rng.random(x.shape) < 0.5, 0.0, -0.0).astype(np.float32)
    else:
        x[np.arange(rows), rng.integers(0, vocab, rows)] = 80.0
    _check(x, rng.random(rows, dtype=np.float32), torch.float32, **_some(rng, rows))


@pytest.mark.gpu
def test_random_numbers_at_their_ends_and_on_borders(cuda) -> None:
    import torch

    u = np.array([0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, -0.0], dtype=np.float32)
    x = np.full((9, 1000), 2.0, dtype=np.float32)
    x[:, :4] = -np.inf
    x[:, 996:] = -np.inf
    _check(x, u, torch.float32)  # 992 equal weights: 0.25 of them is a whole number
    _check(x, u, torch.bfloat16, top_p=0.5)
    _check(x, u, torch.float16, top_k=128)


@pytest.mark.gpu
def test_rows_that_have_no_answer(cuda) -> None:
    import torch

    nan, inf = np.nan, np.inf
    x = np.zeros((9, 2000), dtype=np.float32)
    x[0, 1999], x[1, 3], x[2] = nan, inf, -inf
    f32 = np.float32
    u = np.array([.5, .5, .5, nan, .5, .5, .5, .5, .5], dtype=f32)
    _check(x, u, torch.float32,
           temperature=np.array([1, 1, 1, 1, -1, nan, 1, 1, inf], dtype=f32),
           top_p=np.array([1, 1, 1, 1, 1, 1, nan, 1, .5], dtype=f32),
           min_p=np.array([0, 0, 0, 0, 0, 0, 0, 1.5, .1], dtype=f32))


@pytest.mark.gpu
def test_settings_out_of_their_range_keep_all_or_one(cuda) -> None:
    import torch

    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 3000)).astype(np.float32)
    _check(x, rng.random(6, dtype=np.float32), torch.float32,
           top_k=np.array([-3, 0, 3000, 9999, 0, 0], dtype=np.int32),
           top_p=np.array([1, 1.5, 1, 1, 0, -2], dtype=np.float32))


@pytest.mark.gpu
def test_shares_of_the_draws_are_the_probabilities(cuda) -> None:
    """200000 draws of one row: each share within five standard deviations."""
    import torch

    n, x = 200000, np.log(np.array([0.4, 0.1, 0.3, 0.15, 0.05]))
    logits = torch.from_numpy(x.astype(np.float32)).cuda().expand(n, 5).contiguous()
    g = torch.Generator(device="cuda").manual_seed(5)
    u = torch.rand(n, device="cuda", generator=g)
    p = np.array([0.4, 0, 0.3, 0.15, 0]) / 0.85
    got = sampling.sample(logits, u, top_k=3).tokens.bincount(minlength=5).cpu().numpy() / n
    assert (np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / n)).all(), got


@pytest.mark.gpu
def test_captured_and_on_another_stream(cuda) -> None:
    import torch

    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((64, 40000), device="cuda", generator=g) * 3
    u = torch.rand(64, device="cuda", generator=g)
    t = torch.full((64,), 0.9, device="cuda")
    want = sampling.sample(x, u, temperature=t, top_p=0.9, top_k=900)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = sampling.sample(x, u, temperature=t, top_p=0.9, top_k=900, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logp, want.logp)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = sampling.sample(x, u, temperature=t, top_p=0.9, top_k=900)
    for seed in (7, 8):
        g.manual_seed(seed)
        x.normal_(generator=g)
        u.uniform_(generator=g)
        graph.replay()
        want = sampling.sample(x, u, temperature=t, top_p=0.9, top_k=900)
        assert torch.equal(again.tokens, want.tokens) and torch.equal(again.logp, want.logp)


@pytest.mark.gpu
def test_no_rows_and_refused_arguments(cuda) -> None:
    import torch

    x, u = torch.zeros((3, 50), device="cuda"), torch.zeros(3, device="cuda")
    none = sampling.sample(x[:0], u[:0], temperature=u[:0])
    assert none.tokens.shape == none.logp.shape == (0,)
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_p=0.0),
                dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=2.0), dict(top_k=-1)):
        with pytest.raises(LaunchError, match="pg_sample"):
            sampling.sample(x, u, **bad)
    for bad in (dict(top_k=2.5), dict(top_k=1 << 40), dict(temperature="warm"),
                dict(temperature=u[:2]), dict(top_k=u), dict(top_p=u.double()),
                dict(min_p=u.cpu())):
        with pytest.raises(ValueError):
            sampling.sample(x, u, **bad)
    for logits, uniform in ((x[0], u), (x.cpu(), u), (x.t(), u), (x.double(), u), (x, u[:2]),
                            (x, u.double())):
        with pytest.raises(ValueError):
            sampling.sample(logits, uniform)


def _args(**over) -> SampleArgs:
    a = SampleArgs(logits=16, uniform=16, tokens=16, logp=16, row_stride=100, dtype=3, rows=2,
                   vocab=100, temperature_all=1.0, top_p_all=1.0)
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over", [
    dict(dtype=0), dict(dtype=9), dict(rows=-1), dict(rows=1 << 30), dict(vocab=0),
    dict(vocab=1 << 30), dict(row_stride=99), dict(temperature_all=-1.0),
    dict(temperature_all=float("nan")), dict(top_p_all=0.0), dict(top_p_all=1.1),
    dict(min_p_all=-1.0), dict(min_p_all=1.1), dict(top_k_all=-1), dict(logits=0),
    dict(uniform=0), dict(tokens=0), dict(logp=0), dict(logits=18), dict(uniform=17),
    dict(tokens=20), dict(temperature=2), dict(top_k=2), dict(top_p=2), dict(min_p=2),
    dict(logp=2)], ids=str)
def test_refused_by_the_c_entry(over) -> None:
    build_library()
    assert library().pg_sample(_args(**over), 0) == PG_ERR_ARGUMENT
    assert b"pg_sample" in library().pg_last_error()


def test_no_rows_need_nothing() -> None:
    build_library()
    assert library().pg_sample(_args(rows=0, logits=0, tokens=0), 0) == 0
    assert library().pg_sample(None, 0) == PG_ERR_ARGUMENT
