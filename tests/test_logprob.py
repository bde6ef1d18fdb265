"""Log probabilities, entropy, top alternatives and their gradient against the definitions in 64
bits, and the gradient against differences.

Tolerances. The largest logit is exact and (x - m) rounds once (2^-24 relative); a thread adds
its share of the exponentials in order and shares join in a tree, so with n columns the sum s
carries at most (n / 512 / parts + 30) 2^-24 of itself, 3e-5 at the 200001 columns tested, with
exp's own error of a few 2^-24 times (1 + |x - m|) inside it; log s turns that into an absolute
error, and t / s carries it times the largest |x - m| that still has weight (about 20). So logp
and entropy are held to 4e-5 absolute plus 1e-6 relative. The gradient -p (a + b (log p + H)) has
p's relative error, 4e-5, plus the result's rounding: 2^-8 (bf16), 2^-11 (f16) of itself, and
what f16 cannot hold below 2^-25."""

from __future__ import annotations

import numpy as np
import pytest

from ptxgen import logprob
from ptxgen.build import build_library
from ptxgen.runtime import library

PG_ERR_ARGUMENT = -2
ROUND = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _definition(x, tokens, a, b):
    """In 64 bits: logp, entropy, log p of all columns, and the gradient."""
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        lp = x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))
        p = np.exp(lp)
        plp = np.where(p > 0, p * lp, np.where(np.isnan(p), np.nan, 0.0))
        h = -plp.sum(-1)
        rows = np.arange(len(x))
        has = tokens >= 0
        logp = np.where(has, lp[rows, np.maximum(tokens, 0)], 0.0)
        aa = np.where(has, a, 0.0)[:, None]
        g = -p * aa - b[:, None] * (plp + p * h[:, None])
        g[rows[has], tokens[has]] += aa[has, 0]
    return logp, h, lp, g


def _check(x, tokens, top, dtype, grad=True, stride=None, offset=0):
    import torch

    rows, vocab = x.shape
    wide = torch.full((rows, stride or vocab), float("nan"), device="cuda").to(dtype)
    logits = wide[:, offset:offset + vocab]
    logits.copy_(torch.from_numpy(x))
    exactly = logits.float().cpu().numpy()
    t = torch.from_numpy(tokens).cuda()
    rng = np.random.default_rng(vocab)
    a, b = rng.standard_normal((2, rows)).astype(np.float32)
    r = logprob.logprobs(logits, t, top=top)
    logp, h, lp, g = _definition(exactly, tokens, a.astype(np.float64), b.astype(np.float64))
    for got, want in ((r.logp, logp), (r.entropy, h)):
        np.testing.assert_allclose(got.cpu().numpy(), want, rtol=1e-6, atol=4e-5)
    if top:
        # NaN above all, then by value, ties to the lowest column
        order = np.lexsort((np.broadcast_to(np.arange(vocab), x.shape), -exactly,
                            ~np.isnan(exactly)))
        ids = order[:, :top]
        assert np.array_equal(r.top_ids.cpu().numpy(), ids)
        np.testing.assert_allclose(r.top_logp.cpu().numpy(), np.take_along_axis(lp, ids, 1),
                                   rtol=1e-6, atol=4e-5)
    if not grad:
        return
    got = logprob.logprobs_grad(logits, t, r, torch.from_numpy(a).cuda(),
                                torch.from_numpy(b).cuda())
    assert got.dtype == dtype and got.is_contiguous()
    unit = ROUND[str(dtype).split(".")[1]]
    # the terms that cancel in g carry p's error each
    scale = np.abs(g) + np.exp(lp) * (np.abs(a) + np.abs(b) * (np.abs(h) + 20))[:, None]
    bad = np.isnan(g)
    assert np.array_equal(np.isnan(got.float().cpu().numpy()), bad)
    err = np.abs(got.double().cpu().numpy() - g)
    bound = unit * np.abs(g) + 5e-5 * scale + (2.0 ** -24 if dtype == torch.float16 else 1e-37)
    assert (err <= bound)[~bad].all(), (err - bound)[~bad].max()


CASES = [(1, 1, 1), (3, 2, 2), (5, 7, 5), (2, 31, 31), (4, 513, 8), (3, 4096, 32), (300, 1000, 3),
         (2, 32001, 20), (1, 200001, 32), (7, 50257, 0), (160, 9001, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,top", CASES)
def test_against_64_bits(cuda, rows, vocab, top, dtype) -> None:
    import torch

    rng = np.random.default_rng(rows * vocab)
    x = (rng.standard_normal((rows, vocab)) * 4).astype(np.float32)
    tokens = rng.integers(0, vocab, rows)
    if rows > 2:
        tokens[1] = -1
    _check(x, tokens, min(top, vocab), getattr(torch, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("offset", [0, 1, 3, 8])
def test_strided_rows_at_any_alignment(cuda, dtype, offset) -> None:
    import torch

    rng = np.random.default_rng(offset)
    x = rng.standard_normal((9, 5003)).astype(np.float32)
    _check(x, rng.integers(0, 5003, 9).astype(np.int32), 4, getattr(torch, dtype), stride=5021,
           offset=offset)


@pytest.mark.gpu
def test_masks_infinities_and_equal_logits(cuda) -> None:
    """Columns masked with -inf or the lowest number, rows of one value, rows that have no
    distribution."""
    import torch

    rng = np.random.default_rng(3)
    vocab = 20011
    low = np.finfo(np.float32).min
    x = rng.standard_normal((12, vocab)).astype(np.float32)
    x[0, :] = -np.inf
    x[0, [5, 7, 19999]] = [1, 2, 3]      # three columns left
    x[1, :] = low
    x[1, 17] = 0
    x[2, :] = low                        # an even distribution
    x[3, :] = 0.5
    x[4, ::2] = -np.inf
    x[5, :] = -np.inf                    # nothing left: NaN
    x[6, 9] = np.nan
    x[7, 11] = np.inf
    x[8, :] = -0.0
    x[8, 3::7] = 0.0                     # equal to -0: ties to the lowest column
    x[9, 100:3000] = 9.0                 # more ties than there are candidates
    x[10, :] = np.arange(vocab) // 64    # ascending, with ties
    x[11, :] = -np.arange(vocab)
    tokens = rng.integers(0, vocab, 12)
    tokens[0] = 4
    for top in (5, 32):
        _check(x, tokens, top, torch.float32)
    one = np.zeros((1, 128), np.float32)
    _check(one, np.array([127]), 32, torch.bfloat16)


@pytest.mark.gpu
def test_token_out_of_range_gives_nan(cuda) -> None:
    import torch

    x = torch.randn((3, 100), device=cuda)
    t = torch.tensor([100, -2, 5], device=cuda)
    r = logprob.logprobs(x, t)
    assert r.logp.isnan().tolist() == [True, True, False]
    assert not r.entropy.isnan().any()
    g = logprob.logprobs_grad(x, t, r, torch.ones(3, device=cuda))
    assert g.isnan().any(-1).tolist() == [True, True, False]


@pytest.mark.gpu
def test_gradient_against_differences(cuda) -> None:
    """Central differences of the 64-bit definition in a random direction: with step 1e-4 their
    own error is the third derivative's 1e-9, so the bound is the kernel's 5e-5 of the terms."""
    import torch

    rng = np.random.default_rng(9)
    x = (rng.standard_normal((6, 301)) * 2).astype(np.float32)
    tokens = rng.integers(0, 301, 6)
    a, b = rng.standard_normal((2, 6)).astype(np.float32)
    xt, t = torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda()
    r = logprob.logprobs(xt, t)
    g = logprob.logprobs_grad(xt, t, r, torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda())
    g = g.double().cpu().numpy()

    def f(y):
        logp, h, _, _ = _definition(y, tokens, a, b)
        return (a * logp + b * h).sum()

    for _ in range(10):
        d = rng.standard_normal(x.shape)
        slope = (f(x + 1e-4 * d) - f(x - 1e-4 * d)) / 2e-4
        assert abs((g * d).sum() - slope) <= 5e-5 * (np.abs(g) * np.abs(d)).sum() + 1e-6
    # a missing gradient is a zero one, and the result may replace the logits
    zero = torch.zeros(6, device=cuda)
    only = logprob.logprobs_grad(xt, t, r, torch.from_numpy(a).cuda())
    assert torch.equal(only, logprob.logprobs_grad(xt, t, r, torch.from_numpy(a).cuda(), zero))
    logprob.logprobs_grad(xt, t, r, torch.from_numpy(a).cuda(), out=xt)
    assert torch.equal(xt, only)


@pytest.mark.gpu
def test_refusals_and_no_rows(cuda) -> None:
    import torch

    x = torch.zeros((2, 10), device=cuda)
    t = torch.zeros(2, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError, match="top 11"):
        logprob.logprobs(x, t, top=11)
    with pytest.raises(ValueError, match="tokens"):
        logprob.logprobs(x, t.float())
    with pytest.raises(ValueError, match="logits"):
        logprob.logprobs(x.t(), t)
    with pytest.raises(ValueError, match="dtype"):
        logprob.logprobs(x.double(), t)
    r = logprob.logprobs(x, t)
    with pytest.raises(ValueError, match="d_logp"):
        logprob.logprobs_grad(x, t, r, t)
    with pytest.raises(ValueError, match="out"):
        logprob.logprobs_grad(x, t, r, None, out=x.half())
    empty = logprob.logprobs(x[:0], t[:0], top=3)
    assert empty.logp.shape == (0,) and empty.top_ids.shape == (0, 3)


def test_bad_arguments_are_refused_before_any_cuda_call() -> None:
    build_library()
    lib = library()
    at = 1 << 20  # never dereferenced: every case fails its argument check first
    good = [at, 100, 3, at, 8, 4, 100, 5, at, at, at, at, at, 0]
    for i, bad in [(0, 0), (0, at + 2), (1, 99), (2, 0), (2, 4), (3, 0), (3, at + 4), (4, 2),
                   (5, -1), (6, 0), (7, 33), (7, -1), (8, 0), (9, at + 1), (10, 0), (11, 0),
                   (12, 0)]:
        args = list(good)
        args[i] = bad
        assert lib.pg_logprobs(*args) == PG_ERR_ARGUMENT, (i, bad)
    good = [at, 100, 1, at, 4, 4, 100, at, at, at, at, at, 100, 0]
    for i, bad in [(0, at + 1), (1, 50), (2, 9), (3, at + 2), (4, 1), (7, 0), (8, at + 2),
                   (9, at + 3), (11, 0), (11, at + 1), (12, 99)]:
        args = list(good)
        args[i] = bad
        assert lib.pg_logprobs_grad(*args) == PG_ERR_ARGUMENT, (i, bad)
    good[5] = 0  # no rows is no error and makes no CUDA call
    assert lib.pg_logprobs_grad(*good) == 0
