"""Cases for the serving operators: a paged key-value cache, the attention that reads it, and the
log probabilities of the tokens that come out.

Five operators, each a user's call of ``ptxgen``:

* ``admit``: finished sequences free their pages, the next prompts take pages, and one layer's new
  keys and values are written into them (``PagedCache.free``, ``extend``, ``write``);
* ``pages``: beams are dropped and forked from other parents, or a fragmented cache is compacted
  (``PagedCache.free``, ``fork``, ``compact``);
* ``decode``: attention of one new token a sequence over its pages (``attention.decode``);
* ``prompt``: causal attention of several new tokens a sequence over its pages, with a sliding
  window and sinks (``attention.prompt``);
* ``logprob``: log probabilities of given tokens with the entropy and the top alternatives, and
  the gradient of both for training (``logprob.logprobs``, ``logprobs_grad``).

``run`` is the plain form where ``own`` is false and the framework's calls where it is true.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # a few short chat turns arrive: the calls' latency counts
        {"name": "admit_small", "op": "admit", "dtype": "bf16", "batch": 6, "most": 70,
         "page": 16, "heads": 2, "dim": 64, "ragged": 1},
        # a full prefill batch of one layer
        {"name": "admit_large", "op": "admit", "dtype": "bf16", "batch": 48, "most": 4096,
         "page": 16, "heads": 8, "dim": 128, "ragged": 2},
        # parallel sampling: eight continuations of a handful of prompts in a shallow model
        {"name": "fork_small", "op": "pages", "what": "fork", "dtype": "bf16", "parents": 3,
         "children": 8, "most": 300, "layers": 4, "page": 16, "heads": 4, "dim": 64,
         "ragged": 3},
        # a beam step of a busy server: every beam re-forked, all layers' open pages copied
        {"name": "fork_beams", "op": "pages", "what": "fork", "dtype": "f16", "parents": 40,
         "children": 250, "most": 700, "layers": 24, "page": 64, "heads": 4, "dim": 128,
         "ragged": 4},
        # half the sequences have left a long-running cache: the live pages move to its front
        {"name": "compact", "op": "pages", "what": "compact", "dtype": "bf16", "parents": 96,
         "children": 0, "most": 900, "layers": 16, "page": 16, "heads": 8, "dim": 128,
         "ragged": 5},
        # interactive decoding: few, short sequences
        {"name": "decode_small", "op": "decode", "dtype": "f16", "batch": 4, "most": 777,
         "page": 16, "heads": 4, "group": 4, "dim": 128, "window": 0, "sinks": 0, "ragged": 6},
        # a serving batch over long, ragged contexts
        {"name": "decode_long", "op": "decode", "dtype": "bf16", "batch": 48, "most": 32768,
         "page": 16, "heads": 8, "group": 8, "dim": 128, "window": 0, "sinks": 0, "ragged": 7},
        # a few drafted tokens are checked against a long context with a window and sinks
        {"name": "prompt_draft", "op": "prompt", "dtype": "f16", "batch": 7, "new": 5,
         "most": 20000, "page": 32, "heads": 4, "group": 5, "dim": 64, "window": 4096,
         "sinks": 4, "ragged": 8},
        # chunked prefill of two long documents
        {"name": "prompt_long", "op": "prompt", "dtype": "bf16", "batch": 2, "new": 4096,
         "most": 8192, "page": 16, "heads": 8, "group": 4, "dim": 128, "window": 0, "sinks": 0,
         "ragged": 9},
        # one answer token at a time: the sampled token's score and its alternatives
        {"name": "logprob_step", "op": "logprob", "what": "serve", "dtype": "f32", "rows": 4,
         "vocab": 32001, "top": 5},
        # scoring a batch with a large vocabulary
        {"name": "logprob_score", "op": "logprob", "what": "serve", "dtype": "bf16",
         "rows": 1000, "vocab": 128256, "top": 20},
        # a policy-gradient step: log probability and entropy with their gradient
        {"name": "logprob_train", "op": "logprob", "what": "train", "dtype": "bf16",
         "rows": 4096, "vocab": 50257, "top": 0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("admit", "pages", "decode", "prompt", "logprob"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    ragged = rng.randrange(1 << 20)
    if op == "logprob":
        what = rng.choice(("serve", "train"))
        vocab = _log(rng, 1000, 150000)
        rows = _log(rng, 1, max(1, 100_000_000 // vocab))
        return {"op": op, "what": what, "dtype": dtype, "rows": min(rows, 8192), "vocab": vocab,
                "top": rng.randint(1, 32) if what == "serve" else 0}
    page = rng.choice((8, 16, 16, 32, 64, 24))
    dim = rng.choice((64, 128, 128, 96))
    if op == "admit":
        most = _log(rng, 8, 4096)
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, max(1, min(64, 100_000 // most))),
                "most": most, "page": page, "heads": rng.randint(1, 8), "dim": dim, "ragged": ragged}
    if op == "pages":
        what = rng.choice(("fork", "compact"))
        parents = _log(rng, 2, 64)
        return {"op": op, "what": what, "dtype": dtype, "parents": parents,
                "children": _log(rng, 1, 4 * parents) if what == "fork" else 0,
                "most": _log(rng, 20, 600), "layers": rng.randint(1, 16), "page": page,
                "heads": rng.randint(1, 4), "dim": dim, "ragged": ragged}
    window = rng.choice((0, _log(rng, 16, 4096)))
    case = {"op": op, "dtype": dtype, "page": page, "dim": dim, "window": window,
            "sinks": rng.choice((0, 4, 64)) if window else 0, "ragged": ragged}
    if op == "decode":
        most = _log(rng, 16, 65536)
        case |= {"batch": _log(rng, 1, max(1, min(128, 400_000 // most))), "most": most,
                 "heads": rng.randint(1, 8), "group": rng.choice((1, 2, 4, 7, 8, 16))}
    else:
        new = _log(rng, 1, 4096)
        case |= {"batch": _log(rng, 1, max(1, min(16, 4096 // new))), "new": new,
                 "most": _log(rng, new, 8192), "heads": rng.randint(1, 4),
                 "group": rng.choice((1, 2, 4, 5, 8))}
    return case


# --- what a case's sequences look like (from the case alone: work() goes by them) ------------


def _lens(case, count, lo=1):
    """Ragged lengths up to the case's longest, one of them the longest itself."""
    rng = random.Random(case["ragged"])
    most = case["most"]
    lens = [int(round(lo + (most - lo) * rng.random() ** 1.5)) for _ in range(count)]
    lens[rng.randrange(count)] = most
    return lens


def _news(case, lens):
    """New tokens of each sequence of a prompt batch: up to the case's, never past its length."""
    rng = random.Random(case["ragged"] + 1)
    news = [min(n, case["new"] if i == 0 else rng.randint((case["new"] + 1) // 2, case["new"]))
            for i, n in enumerate(lens)]
    return news


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _pool(case, layers, pages, g):
    """Keys and values of every page: [layers, pages, heads, page, dim]."""
    shape = (layers, pages, case["heads"], case["page"], case["dim"])
    return [torch.randn(shape, device="cuda", dtype=DTYPES[case["dtype"]], generator=g)
            for _ in range(2)]


def _tables(case, counts, pages, g):
    """A table of scattered pages: row i holds counts[i] pages, -1 past them."""
    width = max(1, max(counts))
    ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = ids[at:at + n]
        at += n
    return table


def _pages_of(tokens, page):
    return -(-tokens // page)


def _cache(state):
    """The framework's cache over the tensors in hand."""
    from ptxgen.cache import PagedCache

    return PagedCache(state["k"], state["v"], state["refs"], state["table"], state["lens"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if own:
        package = str(Path(__file__).resolve().parents[1] / "emmy-hackathon-submission_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
    s = {"case": case}
    if case["op"] == "logprob":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab), device="cuda", generator=g) * 3
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["tokens"] = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
        s["d_logp"] = torch.randn(rows, device="cuda", generator=g) / rows
        s["d_entropy"] = torch.full((rows,), 0.01 / rows, device="cuda")
        return s
    page, heads, dim, dtype = case["page"], case["heads"], case["dim"], DTYPES[case["dtype"]]
    if case["op"] in ("decode", "prompt"):
        lens = _lens(case, case["batch"], 0 if case["op"] == "decode" else 1)
        counts = [_pages_of(n, page) for n in lens]
        k, v = _pool(case, 1, sum(counts) + 3, g)
        s |= {"k": k[0], "v": v[0], "table": _tables(case, counts, sum(counts) + 3, g),
              "lens": _ints(lens)}
        news = [1] * len(lens) if case["op"] == "decode" else _news(case, lens)
        hq = heads * case["group"]
        # queries as a model has them: the first heads of a fused projection's rows
        fused = torch.randn((sum(news), hq + 2 * heads, dim), device="cuda", generator=g)
        s["q"] = fused.to(dtype)[:, :hq]
        s["starts"] = _ints(_starts(news))
        s["scale"] = dim ** -0.5
        if own:
            from ptxgen.attention import Workspace

            s["workspace"] = Workspace()
        return s
    if case["op"] == "admit":
        # the cache's slots hold the finished batch; the next one has the lengths reversed
        old = _lens(case, case["batch"])
        new = old[::-1]
        counts = [_pages_of(n, page) for n in old]
        pages = sum(counts) + 5
        k, v = _pool(case, 1, pages, g)
        table = _tables(case, counts, pages, g)
        lens = _ints(old)
        slots = torch.arange(len(old), dtype=torch.int32, device="cuda")
        fused = torch.randn((sum(new), 2 * heads, dim), device="cuda", generator=g).to(dtype)
        s |= {"slots": slots, "starts": _ints(_starts(new)), "new_k": fused[:, :heads],
              "new_v": fused[:, heads:]}
    else:
        parents = case["parents"]
        lens = _lens(case, parents)
        counts = [_pages_of(n, page) for n in lens]
        if case["what"] == "compact":
            # every other sequence has gone: its pages are the holes
            pages = sum(counts)
            table = _tables(case, counts, pages, g)
            lens = [0 if i % 2 else n for i, n in enumerate(lens)]
            table[1::2] = -1
            k, v = _pool(case, case["layers"], pages, g)
        else:
            # the children were forked earlier: one open page each, their parents' other pages
            rng = random.Random(case["ragged"] + 2)
            children = case["children"]
            old = [rng.randrange(parents) for _ in range(children)]
            s["parents"] = _ints([rng.randrange(parents) for _ in range(children)])
            s["children"] = torch.arange(parents, parents + children, dtype=torch.int32,
                                         device="cuda")
            pages = sum(counts) + children + 5
            rows = _tables(case, counts + [1] * children, pages, g)
            share = rows[_ints(old).long()].clone()
            full = [lens[p] // page for p in old]
            open_ = [i for i, p in enumerate(old) if lens[p] % page]
            share[open_, [full[i] for i in open_]] = rows[[parents + i for i in open_], 0]
            table = torch.cat([rows[:parents], share])
            lens = lens + [lens[p] for p in old]
            k, v = _pool(case, case["layers"], pages, g)
        lens = _ints(lens)
    refs = torch.zeros(k.shape[1], dtype=torch.int32, device="cuda")
    held = table[table >= 0].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    s |= {"k": k, "v": v, "refs": refs, "table": table, "lens": lens}
    s |= {"refs0": refs.clone(), "table0": table.clone()}
    if own:
        s["cache"] = _cache(s)
    return s


# --- the plain forms --------------------------------------------------------------------------


def _plain_attention(q, pos, k, v, table, lens, case, scale):
    """softmax(q k^T scale + mask) v for queries q [batch, rows, group, heads, dim] at positions
    pos [batch, rows] of their sequences; a row that sees no key gives zeros."""
    b, width = table.shape
    heads, page, dim = k.shape[1:]
    span = width * page
    at = torch.arange(span, device=q.device)
    inside = at[None] < lens[:, None]
    ids = table.clamp(min=0).long()
    kk = k[ids].permute(0, 2, 1, 3, 4).reshape(b, heads, span, dim).float()
    vv = v[ids].permute(0, 2, 1, 3, 4).reshape(b, heads, span, dim).float()
    vv = torch.where(inside[:, None, :, None], vv, 0.0)
    rows, group = q.shape[1:3]
    qq = q.permute(0, 3, 1, 2, 4).reshape(b, heads, rows * group, dim).float()
    s = (qq @ kk.transpose(-1, -2)) * scale
    seen = inside[:, None] & (at <= pos[:, :, None])
    if case["window"]:
        seen = seen & ((at > pos[:, :, None] - case["window"]) | (at < case["sinks"]))
    seen = seen[:, None, :, None].expand(b, 1, rows, group, span).reshape(b, 1, -1, span)
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.where(total > 0, (s @ vv) / total, 0.0)
    return o.reshape(b, heads, rows, group, dim).permute(0, 2, 3, 1, 4)


def _run_decode(s):
    case, q = s["case"], s["q"]
    if own:
        from ptxgen import attention

        return attention.decode(q, s["k"], s["v"], s["table"], s["lens"], scale=s["scale"],
                                window=case["window"], sinks=case["sinks"],
                                workspace=s["workspace"])
    b, hq, dim = q.shape
    qq = q.reshape(b, 1, case["heads"], case["group"], dim).transpose(2, 3)
    pos = s["lens"][:, None] - 1
    o = _plain_attention(qq, pos, s["k"], s["v"], s["table"], s["lens"], case, s["scale"])
    return o.transpose(2, 3).reshape(b, hq, dim).to(q.dtype)


def _run_prompt(s):
    case, q = s["case"], s["q"]
    if own:
        from ptxgen import attention

        return attention.prompt(q, s["starts"], s["k"], s["v"], s["table"], s["lens"],
                                scale=s["scale"], window=case["window"], sinks=case["sinks"],
                                workspace=s["workspace"])
    starts, hq, dim = s["starts"], q.shape[1], q.shape[2]
    rows = torch.arange(case["new"], device=q.device)
    news = starts[1:] - starts[:-1]
    real = rows[None] < news[:, None]
    at = (starts[:-1, None] + rows[None]).clamp(max=q.shape[0] - 1).long()
    qq = q[at].reshape(*at.shape, case["heads"], case["group"], dim).transpose(2, 3)
    pos = s["lens"][:, None] - news[:, None] + rows[None]
    o = _plain_attention(qq, pos, s["k"], s["v"], s["table"], s["lens"], case, s["scale"])
    return o.transpose(2, 3).reshape(*at.shape, hq, dim)[real].to(q.dtype)


def _plain_free(s, slots):
    """Drops the slots' hold on their pages: refs down, rows -1, lengths 0."""
    rows = s["table"][slots.long()]
    held = rows[rows >= 0].long()
    s["refs"].index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    s["table"][slots.long()] = -1
    s["lens"][slots.long()] = 0


def _run_admit(s):
    case = s["case"]
    if own:
        cache = s["cache"]
        cache.free(s["slots"])
        cache.extend(s["slots"], s["starts"])
        cache.write(0, s["slots"], s["starts"], s["new_k"], s["new_v"])
        return {n: s[n] for n in ("k", "v", "table", "lens", "refs")}
    _plain_free(s, s["slots"])
    page, slots, starts = case["page"], s["slots"].long(), s["starts"].long()
    news = starts[1:] - starts[:-1]
    counts = (news + page - 1) // page
    ends = counts.cumsum(0)
    free = (s["refs"] == 0).nonzero()[:, 0]
    j = torch.arange(s["table"].shape[1], device=slots.device)
    real = j[None] < counts[:, None]
    ids = free[((ends - counts)[:, None] + j[None]).clamp(max=free.numel() - 1)]
    s["table"][slots] = torch.where(real, ids, -1).to(torch.int32)
    s["refs"][ids[real]] = 1
    s["lens"][slots] = news.to(torch.int32)
    t = torch.arange(s["new_k"].shape[0], device=slots.device)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    pos = t - starts[seq]
    where = s["table"][slots[seq], pos // page].long()
    s["k"][0][where, :, pos % page] = s["new_k"]
    s["v"][0][where, :, pos % page] = s["new_v"]
    return {n: s[n] for n in ("k", "v", "table", "lens", "refs")}


def _run_fork(s):
    case = s["case"]
    if own:
        cache = s["cache"]
        cache.free(s["children"])
        cache.fork(s["parents"], s["children"])
        return {n: s[n] for n in ("k", "v", "table", "lens", "refs")}
    page, parents, children = case["page"], s["parents"].long(), s["children"].long()
    _plain_free(s, children)
    lens = s["lens"][parents].long()
    full, part = lens // page, lens % page
    rows = s["table"][parents].clone()
    j = torch.arange(rows.shape[1], device=rows.device)
    shared = rows[j[None] < full[:, None]].long()
    s["refs"].index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    which = (part > 0).nonzero()[:, 0]
    fresh = (s["refs"] == 0).nonzero()[:which.numel(), 0]
    source = rows[which, full[which]].long()
    rows[which, full[which]] = fresh.to(torch.int32)
    s["refs"][fresh] = 1
    s["table"][children] = rows
    s["lens"][children] = lens.to(torch.int32)
    live = (torch.arange(page, device=rows.device)[None] < part[which][:, None])
    live = live[None, :, None, :, None]
    s["k"][:, fresh] = torch.where(live, s["k"][:, source], s["k"][:, fresh])
    s["v"][:, fresh] = torch.where(live, s["v"][:, source], s["v"][:, fresh])
    return {n: s[n] for n in ("k", "v", "table", "lens", "refs")}


def _run_compact(s):
    # the same fragmented cache each time: its table and counts as they were (the pages that
    # move stay behind in place, so the data is the fragmented cache's too)
    s["refs"].copy_(s["refs0"])
    s["table"].copy_(s["table0"])
    if own:
        s["cache"].compact()
        return {n: s[n] for n in ("k", "v", "table", "refs")}
    refs, table = s["refs"], s["table"]
    live = refs > 0
    ids = torch.arange(refs.numel(), device=refs.device)
    front = ids < live.sum()
    holes = (front & ~live).nonzero()[:, 0]
    movers = (~front & live).nonzero()[:, 0]
    s["k"][:, holes] = s["k"][:, movers]
    s["v"][:, holes] = s["v"][:, movers]
    place = ids.to(torch.int32)
    place[movers] = holes.to(torch.int32)
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], -1))
    refs[holes] = refs[movers]
    refs[movers] = 0
    return {n: s[n] for n in ("k", "v", "table", "refs")}


def _run_logprob(s):
    case, logits, tokens = s["case"], s["logits"], s["tokens"]
    if own:
        from ptxgen import logprob

        if case["what"] == "serve":
            r = logprob.logprobs(logits, tokens, top=case["top"])
            return {"logp": r.logp, "entropy": r.entropy, "top_logp": r.top_logp,
                    "top_ids": r.top_ids}
        r = logprob.logprobs(logits, tokens)
        grad = logprob.logprobs_grad(logits, tokens, r, s["d_logp"], s["d_entropy"])
        return {"logp": r.logp, "entropy": r.entropy, "grad": grad}
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    total = (x - top).exp().sum(-1, keepdim=True)
    logp = x - (top + total.log())
    p = logp.exp()
    entropy = -(p * logp).sum(-1)
    out = {"logp": logp.gather(1, tokens[:, None])[:, 0], "entropy": entropy}
    if case["what"] == "serve":
        ids = logits.sort(dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        return out | {"top_logp": logp.gather(1, ids), "top_ids": ids.to(torch.int32)}
    g = -p * (s["d_logp"][:, None] + s["d_entropy"][:, None] * (logp + entropy[:, None]))
    g.scatter_add_(1, tokens[:, None], s["d_logp"][:, None])
    return out | {"grad": g.to(logits.dtype)}


def run(state):
    case = state["case"]
    name = case["what"] if case["op"] == "pages" else case["op"]
    return {"admit": _run_admit, "fork": _run_fork, "compact": _run_compact,
            "decode": _run_decode, "prompt": _run_prompt, "logprob": _run_logprob}[name](state)


# --- what a pass cannot do without ------------------------------------------------------------


def _seen(case, length, new):
    """(keys that some of the sequence's new tokens see, pairs of a new token and a key)."""
    window, sinks = case["window"], case["sinks"]
    if not new or not length:
        return 0, 0
    first = length - new
    if not window:
        return length, sum(range(first + 1, length + 1))
    start = max(0, first - window + 1)  # the first new token's oldest key but the sinks
    keys = length - start + min(sinks, start)
    pairs = 0
    for p in range(first, length):
        low = max(0, p - window + 1)
        pairs += p - low + 1 + min(sinks, low)
    return keys, pairs


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "logprob":
        n, rows, top = case["rows"] * case["vocab"], case["rows"], case["top"]
        if case["what"] == "serve":
            return {"bytes": n * size + rows * (8 + 8 + 8 * top), "flops": 5 * n}
        return {"bytes": 2 * n * size + rows * (2 * 8 + 4 * 8), "flops": 13 * n}
    page, heads, dim = case["page"], case["heads"], case["dim"]
    token = heads * dim * size  # one token's keys (or values) of one layer
    if case["op"] in ("decode", "prompt"):
        lens = _lens(case, case["batch"], 0 if case["op"] == "decode" else 1)
        news = [1] * len(lens) if case["op"] == "decode" else _news(case, lens)
        seen = [_seen(case, n, m) for n, m in zip(lens, news)]
        keys, pairs = sum(a for a, _ in seen), sum(b for _, b in seen)
        q = sum(news) * heads * case["group"] * dim * size
        return {"bytes": 2 * keys * token + 2 * q + 4 * (-(-keys // page) + 2 * len(lens)),
                "flops": 4 * pairs * heads * case["group"] * dim}
    if case["op"] == "admit":
        lens = _lens(case, case["batch"])
        counts = sum(_pages_of(n, page) for n in lens)
        # keys and values read and written; tables read and written; counts down and up
        return {"bytes": 4 * sum(lens) * token + 4 * (2 * counts + 4 * counts + 4 * len(lens)),
                "flops": 0}
    lens = _lens(case, case["parents"])
    if case["what"] == "fork":
        rng = random.Random(case["ragged"] + 2)
        old = [rng.randrange(case["parents"]) for _ in range(case["children"])]
        new = [rng.randrange(case["parents"]) for _ in range(case["children"])]
        rows = sum(lens[p] % page for p in new)
        held = sum(_pages_of(lens[p], page) for p in old + new)
        return {"bytes": 4 * rows * token * case["layers"] + 4 * (2 * held + 2 * held),
                "flops": 0}
    counts = [_pages_of(n, page) for n in lens]
    live = sum(counts[::2])
    # of the live pages, scattered at random, those past the front move
    moved = live * (sum(counts) - live) // sum(counts)
    return {"bytes": 4 * moved * page * token * case["layers"]
            + 4 * (4 * sum(counts) + 4 * len(lens) * max(counts)), "flops": 0}


# --- the definitions in 64 bits -----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprob":
        return _exact_logprob(s)
    if case["op"] in ("decode", "prompt"):
        return _exact_attention(s)
    return None  # copies and whole numbers


def _exact_attention(s):
    case, q, starts = s["case"], s["q"], s["starts"].tolist()
    heads, group, page = case["heads"], case["group"], case["page"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i, n in enumerate(s["lens"].tolist()):
        a, b = starts[i], starts[i + 1]
        if n == 0 or a == b:
            continue
        ids = s["table"][i, :_pages_of(n, page)].long()
        pos = torch.arange(n - (b - a), n, device=q.device)[:, None]
        at = torch.arange(n, device=q.device)[None]
        hidden = at > pos
        if case["window"]:
            hidden |= (at <= pos - case["window"]) & (at >= case["sinks"])
        for h in range(heads):
            k = s["k"][ids, h].reshape(-1, case["dim"])[:n].double()
            v = s["v"][ids, h].reshape(-1, case["dim"])[:n].double()
            for r in range(h * group, (h + 1) * group):
                w = torch.einsum("td,sd->ts", q[a:b, r].double(), k) * s["scale"]
                w[hidden] = -math.inf
                out[a:b, r] = torch.softmax(w, -1) @ v
    return out


def _exact_logprob(s):
    case, logits, tokens = s["case"], s["logits"], s["tokens"]
    rows, vocab = logits.shape
    logp = torch.empty(rows, dtype=torch.float64, device=logits.device)
    entropy = torch.empty_like(logp)
    grad = torch.empty((rows, vocab), dtype=torch.float64, device=logits.device) \
        if case["what"] == "train" else None
    tops = []
    for a in range(0, rows, 256):
        b = min(rows, a + 256)
        lp = torch.log_softmax(logits[a:b].double(), -1)
        p = lp.exp()
        logp[a:b] = lp[torch.arange(b - a), tokens[a:b]]
        entropy[a:b] = -(p * lp).sum(-1)
        if grad is None:
            tops.append(lp.topk(case["top"], -1).values)
            continue
        d1, d2 = s["d_logp"][a:b, None].double(), s["d_entropy"][a:b, None].double()
        hot = torch.zeros_like(p)
        hot[torch.arange(b - a), tokens[a:b]] = 1
        grad[a:b] = d1 * (hot - p) - d2 * p * (lp + entropy[a:b, None])
    out = {"logp": logp, "entropy": entropy}
    if grad is None:
        return out | {"top_logp": torch.cat(tops), "top_ids": None}
    return out | {"grad": grad}
