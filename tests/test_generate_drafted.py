"""Drawing, the cache in 8 bits, drafted trees and what is kept of them, run together as a serving
program does.

Greedy tokens are whole numbers and must be those of one token at a time: in f32 the two ways differ by
some 1e-6 of logits of order 10, and the largest two are further apart than that at every token tested
(1e-4, asserted). In 8 bits a row is off by half a step of its largest number's 127th, so log
probabilities move: keys and values of order 1 by 2^-8 a coordinate, the scores by 2^-8 64^(1/2) 8^-1 and
the weights as much, and logits of order 10 by a few hundredths a layer; 0.5 is a safe bound for two."""

from __future__ import annotations

import pytest

from test_generate import _scores


def _prompts():
    import torch

    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (33, 1, 300, 16)]


def _greedy(model, prompt, steps):
    """One token at a time without a cache, in 64 bits; the least lead of a largest logit."""
    import torch

    tokens, lead = list(prompt), float("inf")
    for _ in range(steps):
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
        top = (x[-1] @ model.unembed.double()).topk(2)
        lead = min(lead, float(top.values[0] - top.values[1]))
        tokens.append(int(top.indices[0]))
    return tokens[len(prompt):], lead


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_drafted_greedy_tokens_are_those_of_one_at_a_time(cuda, window, sinks) -> None:
    import torch

    from ptxgen.generate import Model, drafted

    model = Model.random(dtype=torch.float32, window=window, sinks=sinks)
    prompts = _prompts()
    out, cache = drafted(model, prompts, rounds=9, page_size=8, temperature=0.0)
    for p, tokens in zip(prompts, out):
        assert 10 <= len(tokens) <= 28
        want, lead = _greedy(model, p, len(tokens))
        assert lead > 1e-4
        assert tokens == want
    # the cache holds all of them but the last, in pages that no other slot has
    assert cache.lens.tolist() == [len(p) + len(t) - 1 for p, t in zip(prompts, out)]
    held = sum(-(-n // 8) for n in cache.lens.tolist())
    assert int((cache.refs > 0).sum()) == int(cache.refs.sum()) == held


@pytest.mark.gpu
def test_guesses_are_taken(cuda) -> None:
    """A model without layers is what guesses are made of, so every one is right."""
    import torch

    from ptxgen.generate import Model, drafted

    model = Model.random(dtype=torch.float32)
    for _, out in model.layers:
        out.zero_()
    out, _ = drafted(model, _prompts(), rounds=5, temperature=0.0)
    assert [len(t) for t in out] == [16] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_samples_over_a_cache_in_8_bits(cuda, dtype) -> None:
    import torch

    from ptxgen.generate import Model, drafted, generate

    model = Model.random(dtype=getattr(torch, dtype))
    prompts = _prompts()
    out, cache = generate(model, prompts, samples=3, steps=16, page_size=8, bits8=True, top_p=0.9,
                          temperature=0.8)
    assert cache.k.dtype is torch.int8
    for s in out:
        n = len(prompts[s.prompt])
        logp, _ = _scores(model, prompts[s.prompt] + s.tokens)
        err = (torch.tensor(s.logps, device="cuda") - logp[n - 1:]).abs().max()
        assert float(err) < 0.5
    texts, cache = drafted(model, prompts, rounds=6, bits8=True, top_k=40, min_p=0.01)
    assert cache.lens.tolist() == [len(p) + len(t) - 1 for p, t in zip(prompts, texts)]


@pytest.mark.gpu
def test_limits_hold_for_every_token(cuda) -> None:
    import torch

    from ptxgen.generate import Model, generate

    model = Model.random(dtype=torch.float32)
    prompts = _prompts()[:2]
    out, _ = generate(model, prompts, samples=2, steps=10, top_k=1)
    for s in out:  # one token is kept: the samples of a prompt are the same, and its likeliest
        want, lead = _greedy(model, prompts[s.prompt], len(s.tokens))
        assert lead > 1e-4 and s.tokens == want


@pytest.mark.gpu
@pytest.mark.parametrize("argv", [["--draft", "--steps", "5"], ["--bits8", "--top-p", "0.9", "--steps", "6"],
                                  ["--draft", "--bits8", "--temperature", "0.7", "--top-k", "50"]],
                         ids=" ".join)
def test_the_command(cuda, capsys, monkeypatch, argv) -> None:
    import sys

    from ptxgen import generate

    monkeypatch.setattr(sys, "argv", ["generate", *argv])
    generate.main()
    text = capsys.readouterr().out
    assert "prompt 2" in text and ("rounds" in text) == ("--draft" in argv)


@pytest.mark.parametrize("prompts,rounds", [([], 2), ([[1], []], 2), ([[1]], 0)])
def test_refused(prompts, rounds) -> None:
    from ptxgen.generate import drafted

    with pytest.raises(ValueError, match="at least one"):
        drafted(None, prompts, rounds)
