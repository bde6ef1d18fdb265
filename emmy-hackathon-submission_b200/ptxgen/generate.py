"""Parallel sampling over a paged cache: the cache, the attention that reads it and the scores of
what comes out, as a serving program calls them.

    python emmy-hackathon-submission_b200/ptxgen/generate.py --samples 4 --steps 24

A small attention-only model with random weights reads a few prompts of different lengths at once
(``PagedCache.extend`` and ``write``, ``attention.prompt``), each prompt is forked into several
samples that share its full pages (``fork``), and the samples are continued token by token
(``attention.decode``), every token drawn from the distribution whose log probability, entropy and
best alternatives ``logprobs`` gives. Halfway the worst sample of each prompt is dropped (``free``)
and the cache compacted. Nothing in the loop waits for the GPU; the result comes back at the end.

With ``--temperature``, ``--top-k``, ``--top-p`` or ``--min-p`` tokens are drawn by ``sampling.sample``, with
``--bits8`` the cache is in 8 bits. ``--draft`` continues each prompt by drafted trees instead
(``drafted``): a small tree of guesses a sequence goes through the model at once (``attention.tree``),
a token is drawn at each of its nodes, and the branch that the draws follow stays in the cache
(``PagedCache.keep``). The tokens have the distribution that one at a time would have.
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path
from typing import Any

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch

from ptxgen import attention, sampling
from ptxgen.cache import PagedCache
from ptxgen.logprob import logprobs


@dataclass
class Model:
    """Random weights: an embedding, attention layers and an output projection."""

    embed: Any  # [vocab, heads * dim]
    unembed: Any  # [heads * dim, vocab]
    layers: list[tuple[Any, Any]]  # (q, k, v projection; output projection)
    heads: int
    kv_heads: int
    dim: int
    window: int = 0
    sinks: int = 0

    @classmethod
    def random(cls, vocab: int = 1000, layers: int = 2, heads: int = 4, kv_heads: int = 2,
               dim: int = 64, dtype: torch.dtype = torch.bfloat16, seed: int = 0, window: int = 0,
               sinks: int = 0, device: Any = "cuda") -> Model:
        g = torch.Generator(device=device).manual_seed(seed)
        width = heads * dim

        def weights(rows: int, columns: int) -> Any:
            w = torch.randn((rows, columns), device=device, generator=g)
            return (w * rows ** -0.5).to(dtype)

        embed = torch.randn((vocab, width), device=device, generator=g).to(dtype)
        return cls(embed, weights(width, vocab) * 2,
                   [(weights(width, (heads + 2 * kv_heads) * dim), weights(width, width))
                    for _ in range(layers)], heads, kv_heads, dim, window, sinks)

    def forward(self, tokens: Any, slots: Any, starts: Any, cache: PagedCache, workspace: Any,
                prompts: bool, mask: Any = None) -> Any:
        """The hidden states [tokens, width] of each slot's new tokens, which get room in the
        cache: rows ``starts[i]`` to ``starts[i + 1]``, or row i alone where not ``prompts``. With a
        ``mask`` (``attention.branches``) they are trees."""
        cache.extend(slots, starts)
        x = self.embed[tokens]
        for i, (qkv, out) in enumerate(self.layers):
            y = (x @ qkv).view(-1, self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], 1)
            cache.write(i, slots, starts, k, v)
            at = dict(slots=slots, window=self.window, sinks=self.sinks, workspace=workspace)
            if cache.k_scale is not None:
                at |= dict(k_scale=cache.k_scale[i], v_scale=cache.v_scale[i])
            if mask is not None:
                o = attention.tree(q, starts, mask, cache.k[i], cache.v[i], cache.table, cache.lens,
                                   **at)
            elif prompts:
                o = attention.prompt(q, starts, cache.k[i], cache.v[i], cache.table, cache.lens,
                                     **at)
            else:
                o = attention.decode(q, cache.k[i], cache.v[i], cache.table, cache.lens, **at)
            x = x + o.reshape(-1, self.heads * self.dim) @ out
        return x


@dataclass
class Sample:
    prompt: int  # which prompt it continues
    tokens: list[int]
    logps: list[float]  # of each token
    entropies: list[float]  # of the distributions that they were drawn from
    dropped: bool


def generate(model: Model, prompts: list[list[int]], samples: int = 4, steps: int = 24,
             page_size: int = 16, seed: int = 0, bits8: bool = False,
             **limits: Any) -> tuple[list[Sample], PagedCache]:
    """``samples`` continuations of each prompt by ``steps`` tokens; after half of them each
    prompt's least likely sample is dropped and keeps what it has. Every prompt has a token: the
    samples begin from the hidden state of its last one. ``limits`` are ``sampling.sample``'s; the
    scores are those of the whole distribution."""
    if not prompts or not all(prompts) or samples < 1 or steps < 1:
        raise ValueError(f"prompts of {[len(p) for p in prompts]} tokens, {samples} samples, {steps} "
                         "steps: want at least one of each")
    dev = model.embed.device
    g = torch.Generator(device=dev).manual_seed(seed)

    def ints(values: Any) -> Any:
        return torch.tensor(list(values), dtype=torch.int32, device=dev)

    count, total = len(prompts), sum(map(len, prompts))
    longest = max(map(len, prompts)) + steps
    width = -(-longest // page_size)
    cache = PagedCache.allocate(len(model.layers), count * (samples + 1) * width, model.kv_heads,
                                page_size, model.dim, count * (samples + 1), width,
                                dtype=torch.int8 if bits8 else model.embed.dtype, device=dev)
    workspace = attention.Workspace(dev)

    # the prompts, at once: slot i holds prompt i; the last hidden state of each begins its samples
    ends = torch.tensor([len(p) for p in prompts]).cumsum(0).tolist()
    tokens = torch.tensor([t for p in prompts for t in p], device=dev)
    hidden = model.forward(tokens, ints(range(count)), ints([0, *ends]), cache, workspace, True)
    assert hidden.shape[0] == total
    hidden = hidden[[e - 1 for e in ends]].repeat_interleave(samples, 0)
    parents = ints(range(count)).repeat_interleave(samples)
    slots = ints(range(count, count * (samples + 1)))
    cache.fork(parents, slots)
    cache.free(ints(range(count)))

    live = torch.arange(count * samples, device=dev)
    made, scores = [], []
    likely = torch.zeros(count * samples, device=dev)
    for step in range(steps):
        logits = hidden @ model.unembed
        if limits:
            uniform = torch.rand(logits.shape[0], device=dev, generator=g)
            drawn = sampling.sample(logits, uniform, **limits).tokens
        else:
            noise = torch.rand(logits.shape, device=dev, generator=g).clamp_(1e-9)
            drawn = (logits.float() - noise.log().neg_().log_()).argmax(-1)
        r = logprobs(logits, drawn)
        made.append((live, drawn))
        scores.append((r.logp, r.entropy))
        likely[live] += r.logp
        if step == steps // 2 and samples > 1:
            # the least likely sample of each prompt goes; the others' pages close up
            worst = likely.view(count, samples).argmin(-1) + torch.arange(count, device=dev) * samples
            cache.free(slots[worst])
            keep = torch.ones(count * samples, dtype=torch.bool, device=dev)
            keep[worst] = False
            order = (~keep).to(torch.int32).argsort(stable=True)[:count * (samples - 1)]
            live, slots, drawn = live[order], slots[order], drawn[order]
            cache.compact()
        if step + 1 < steps:
            one_each = torch.arange(live.numel() + 1, dtype=torch.int32, device=dev)
            hidden = model.forward(drawn, slots, one_each, cache, workspace, False)
    cache.check()
    workspace.check()
    out = [Sample(i // samples, [], [], [], True) for i in range(count * samples)]
    for (who, drawn), (logp, entropy) in zip(made, scores):
        for i, t, a, b in zip(who.tolist(), drawn.tolist(), logp.tolist(), entropy.tolist()):
            out[i].tokens.append(t)
            out[i].logps.append(a)
            out[i].entropies.append(b)
    for i in live.tolist():
        out[i].dropped = False
    return out, cache


# A tree of guesses: the last token, three that may follow it, and one that may follow each of them.
_PARENTS = [-1, 0, 0, 0, 1, 2, 3]


def drafted(model: Model, prompts: list[list[int]], rounds: int = 12, page_size: int = 16,
            seed: int = 0, bits8: bool = False, **limits: Any) -> tuple[list[list[int]], PagedCache]:
    """Each prompt continued by one to three tokens a round, as ``sampling.sample`` with ``limits`` draws
    them. Guesses are what the embedding alone makes of a token."""
    if not prompts or not all(prompts) or rounds < 1:
        raise ValueError(f"prompts of {[len(p) for p in prompts]} tokens, {rounds} rounds: want at least "
                         "one of each")
    dev, nodes = model.embed.device, len(_PARENTS)
    g = torch.Generator(device=dev).manual_seed(seed)

    def ints(values: Any, dtype: torch.dtype = torch.int32) -> Any:
        return torch.tensor(list(values), dtype=dtype, device=dev)

    def draw(hidden: Any) -> Any:
        uniform = torch.rand(hidden.shape[0], device=dev, generator=g)
        return sampling.sample(hidden @ model.unembed, uniform, **limits).tokens

    count = len(prompts)
    width = -(-(max(map(len, prompts)) + 3 * rounds + nodes) // page_size)
    cache = PagedCache.allocate(len(model.layers), count * width, model.kv_heads, page_size, model.dim,
                                count, width, dtype=torch.int8 if bits8 else model.embed.dtype,
                                device=dev)
    workspace = attention.Workspace(dev)
    slots = ints(range(count))
    ends = torch.tensor([len(p) for p in prompts]).cumsum(0).tolist()
    tokens = torch.tensor([t for p in prompts for t in p], device=dev)
    hidden = model.forward(tokens, slots, ints([0, *ends]), cache, workspace, True)
    last = draw(hidden[[e - 1 for e in ends]])
    starts = ints(range(0, nodes * (count + 1), nodes))
    branches = ints(attention.branches(_PARENTS), torch.int64)
    mask = branches.repeat(count)
    made = [(last, None, None)]
    for _ in range(rounds):
        likely = (model.embed[last] @ model.unembed).topk(3).indices
        after = (model.embed[likely] @ model.unembed).argmax(-1)
        tree = torch.cat([last[:, None], likely, after], 1)
        hidden = model.forward(tree.reshape(-1), slots, starts, cache, workspace, True, mask)
        drawn = draw(hidden).view(count, nodes)
        # from the root to the guess that is what was drawn there, and on to the guess after it
        hit = likely == drawn[:, :1]
        at = torch.where(hit.any(1), hit.int().argmax(1) + 1, 0)
        guess = after.gather(1, (at - 1).clamp(min=0)[:, None])
        more = (at > 0) & (guess == drawn.gather(1, at[:, None]))[:, 0]
        at = torch.where(more, at + 3, at)
        cache.keep(slots, starts, branches[at])
        last = drawn.gather(1, at[:, None])[:, 0]
        made.append((last, tree, at))
    cache.check()
    workspace.check()
    out: list[list[int]] = [[] for _ in prompts]
    for drawn, tree, at in made:
        for i, t in enumerate(drawn.tolist()):
            if tree is not None:
                path, node = [], int(at[i])
                while node > 0:
                    path.append(int(tree[i, node]))
                    node = _PARENTS[node]
                out[i] += reversed(path)
            out[i].append(t)
    return out, cache


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--samples", type=int, default=4)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--bits8", action="store_true", help="a cache in 8 bits")
    ap.add_argument("--draft", action="store_true", help="drafted trees, --steps rounds of them")
    for name, kind in (("temperature", float), ("top-k", int), ("top-p", float), ("min-p", float)):
        ap.add_argument(f"--{name}", type=kind)
    args = ap.parse_args()
    limits = {n: v for n in ("temperature", "top_k", "top_p", "min_p")
              if (v := getattr(args, n)) is not None}
    model = Model.random(window=64, sinks=4)
    g = torch.Generator().manual_seed(args.seed)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (40, 133, 7)]
    if args.draft:
        texts, cache = drafted(model, prompts, args.steps, seed=args.seed, bits8=args.bits8, **limits)
        for i, t in enumerate(texts):
            print(f"prompt {i}: {len(t)} tokens in {args.steps} rounds: "
                  f"{' '.join(map(str, t[:8]))} ...")
        return
    out, cache = generate(model, prompts, args.samples, args.steps, seed=args.seed,
                          bits8=args.bits8, **limits)
    for i, s in enumerate(out):
        mean = sum(s.entropies) / len(s.entropies)
        print(f"prompt {s.prompt} sample {i % args.samples}: log p {sum(s.logps):8.2f}, mean "
              f"entropy {mean:.2f}, {len(s.tokens)} tokens{' (dropped)' if s.dropped else ''}: "
              f"{' '.join(map(str, s.tokens[:8]))} ...")
    pages = int((cache.refs > 0).sum())
    print(f"{pages} of {cache.refs.numel()} pages in use, the highest "
          f"{int((cache.refs > 0).nonzero().max())}")


if __name__ == "__main__":
    main()
