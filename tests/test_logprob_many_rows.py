"""Log probabilities and their gradient where the rows fill the GPU (more than eight an SM), on both
sides of 32768 columns with alternatives, against the definitions in 64 bits.

Tolerances. A block has 128 or 256 threads, each of which adds its n / 128 or fewer exponentials in
order, in two sums; the threads' sums join in a tree. So the sum s carries at most (n / 128 + 30) 2^-24
of itself, 1.8e-5 at the 32769 columns tested, and exp's own error is a few 2^-24 (1 + |x - m|). log s
turns that into an absolute error, and t / s carries it times the largest |x - m| that has weight (20):
logp and entropy are held to 4e-5 absolute plus 1e-6 relative, as with fewer rows, which random
roundings leave far below. The gradient -p (a + b (log p + H)) has p's relative error and the result's
rounding, 2^-8 (bf16) or 2^-11 (f16) of itself, and what f16 cannot hold below 2^-25."""

from __future__ import annotations

import pytest

from ptxgen import logprob

ROUND = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _rows(extra=37):
    import torch

    return 8 * torch.cuda.get_device_properties(0).multi_processor_count + extra


def _close(got, want, atol=4e-5, rtol=1e-6):
    import torch

    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    some = torch.isfinite(want)
    assert bool(((got - want).abs() <= atol + rtol * want.abs())[some].all()), \
        float((got - want)[some].abs().max())


def _check(logits, tokens, top, grad):
    import torch

    rows, vocab = logits.shape
    g = torch.Generator(device="cuda").manual_seed(vocab)
    a, b = torch.randn((2, rows), device="cuda", generator=g)
    r = logprob.logprobs(logits, tokens, top=top)
    x = logits.double()
    lp = x - x.amax(-1, keepdim=True)
    lp = lp - lp.exp().sum(-1, keepdim=True).log()
    p = lp.exp()
    plp = torch.where(p == 0, 0.0, p * lp)
    h = -plp.sum(-1)
    has = tokens >= 0
    at = tokens.long().clamp(min=0)[:, None]
    _close(r.logp, torch.where(has, lp.gather(1, at)[:, 0], 0.0))
    _close(r.entropy, h)
    if top:
        ids = logits.float().sort(dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids, ids.to(torch.int32))
        _close(r.top_logp, lp.gather(1, ids))
    if not grad:
        return
    got = logprob.logprobs_grad(logits, tokens, r, a, b).double()
    a, b = torch.where(has, a, 0.0).double()[:, None], b.double()[:, None]
    want = -p * a - b * (plp + p * h[:, None])
    want.scatter_add_(1, at, a)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    # the terms that cancel carry p's error each
    scale = want.abs() + p * (a.abs() + b.abs() * (h[:, None].abs() + 20))
    unit = ROUND[str(logits.dtype).split(".")[1]]
    bound = unit * want.abs() + 5e-5 * scale + \
        (2.0 ** -24 if logits.dtype is torch.float16 else 1e-37)
    assert bool(((got - want).abs() <= bound)[~torch.isnan(want)].all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(ROUND))
@pytest.mark.parametrize("vocab,top", [(1, 0), (1, 1), (33, 32), (127, 5), (1000, 0), (1001, 1),
                                       (1718, 0), (5003, 32), (32768, 5), (32768, 32), (32769, 5),
                                       (32769, 32), (32769, 0)])
def test_against_64_bits(cuda, vocab, top, dtype) -> None:
    import torch

    rows = _rows()
    g = torch.Generator(device="cuda").manual_seed(vocab + top)
    x = (torch.randn((rows, vocab), device="cuda", generator=g) * 4).to(getattr(torch, dtype))
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    tokens[::5] = -1
    _check(x, tokens, top, grad=top in (0, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(ROUND))
@pytest.mark.parametrize("offset", [0, 1, 3, 8])
@pytest.mark.parametrize("vocab", [5, 2003])
def test_strided_rows_at_any_alignment(cuda, vocab, offset, dtype) -> None:
    import torch

    rows = _rows(1)
    wide = torch.full((rows, vocab + 18), float("nan"), device="cuda").to(getattr(torch, dtype))
    x = wide[:, offset:offset + vocab]
    x.copy_(torch.randn((rows, vocab), device="cuda"))
    tokens = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda")
    _check(x, tokens, 4, grad=True)
    _check(x, tokens, 0, grad=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(ROUND))
@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("vocab", [4099, 32768, 33001])
def test_masks_and_equal_logits(cuda, vocab, top, dtype) -> None:
    """Rows of one value, with more equal logits than the selection looks at, mostly masked, with few
    columns left, or with nothing."""
    import torch

    rows = _rows(3)
    x = torch.randn((rows, vocab), device="cuda")
    low = torch.finfo(getattr(torch, dtype)).min
    x[0::11] = 0.5
    x[1::11, 100:3000] = 9.0
    x[2::11] = low
    x[3::11] = float("-inf")
    x[3::11, [5, 7, vocab - 1]] = torch.tensor([1.0, 2.0, 3.0], device="cuda")
    x[4::11, :-40] = float("-inf")
    x[5::11, 40:] = low
    x[6::11] = (torch.arange(vocab, device="cuda") // 64).float().clamp(max=500)
    x[7::11, ::2] = float("-inf")
    x[8] = float("-inf")
    x[19, 9] = float("nan")
    x[30, 11] = float("inf")
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    _check(x.to(getattr(torch, dtype)), tokens, top, grad=top == 0)
