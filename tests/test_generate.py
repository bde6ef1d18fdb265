"""Parallel sampling over the paged cache against the same model without one: every sample's log
probabilities and entropies recomputed from its tokens in 64 bits, each prompt on its own, with
whole-matrix attention.

Tolerance. In f32 a layer's projections and attention carry errors of some 2^-24 times the root
of their lengths (256 products, 500 keys), 1e-6 of numbers of order 1; two layers, logits of order
10 and the log probability's own 4e-5 leave 1e-3 as a safe bound."""

from __future__ import annotations

import pytest


def _scores(model, tokens):
    """log p and entropy of each token after the first, in 64 bits."""
    import torch

    x = model.embed[torch.tensor(tokens, device="cuda")].double()
    n = len(tokens)
    at = torch.arange(n, device="cuda")
    hidden = at[None] > at[:, None]
    if model.window:
        hidden |= (at[None] <= at[:, None] - model.window) & (at[None] >= model.sinks)
    group = model.heads // model.kv_heads
    for qkv, out in model.layers:
        y = (x @ qkv.double()).view(n, -1, model.dim)
        q, k, v = y.split([model.heads, model.kv_heads, model.kv_heads], 1)
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = torch.einsum("thd,shd->hts", q, k) * model.dim ** -0.5
        o = torch.softmax(s.masked_fill(hidden, float("-inf")), -1) @ v.transpose(0, 1)
        x = x + o.transpose(0, 1).reshape(n, -1) @ out.double()
    lp = torch.log_softmax(x @ model.unembed.double(), -1)
    logp = lp[:-1].gather(1, torch.tensor(tokens[1:], device="cuda")[:, None])[:, 0]
    return logp, -(lp.exp() * lp).sum(-1)[:-1]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (32, 3)])
def test_samples_score_as_without_a_cache(cuda, window, sinks) -> None:
    import torch

    from ptxgen.generate import Model, generate

    model = Model.random(dtype=torch.float32, window=window, sinks=sinks)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (33, 1, 300, 16)]
    out, cache = generate(model, prompts, samples=3, steps=20, page_size=8)
    assert len(out) == 12 and sum(s.dropped for s in out) == 4
    for s in out:
        assert len(s.tokens) == (11 if s.dropped else 20)
        n = len(prompts[s.prompt])
        logp, entropy = _scores(model, prompts[s.prompt] + s.tokens)
        for got, want in ((s.logps, logp[n - 1:]), (s.entropies, entropy[n - 1:])):
            assert float((torch.tensor(got, device="cuda") - want).abs().max()) < 1e-3
    # what is left of a prompt's samples shares its full pages, and no hole lies between pages
    live = cache.refs > 0
    held = sum(-(-int(n) // 8) for n in cache.lens.tolist())
    assert int(cache.refs.sum()) == held > int(live.sum())
    assert bool((cache.refs[: 4] > 0).all())


@pytest.mark.gpu
def test_16_bit_samples_and_the_command(cuda, capsys, monkeypatch) -> None:
    import sys

    from ptxgen import generate

    monkeypatch.setattr(sys, "argv", ["generate", "--samples", "3", "--steps", "10"])
    generate.main()
    text = capsys.readouterr().out
    assert text.count("prompt ") == 9 and text.count("(dropped)") == 3 and "pages in use" in text
