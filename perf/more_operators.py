"""Cases for operators around the paged cache: drawing the next token, a cache in 8 bits with the
attention that reads it, and trees of drafted tokens.

Five operators, each a user's call of ``ptxgen``:

* ``sample``: a token of each row from temperature, top-k, top-p and min-p, by a given random number
  (``sampling.sample``);
* ``store``: new keys and values are quantised into the pages of a cache in 8 bits and read back as a
  16-bit or f32 user sees them (``PagedCache.write``, ``read``);
* ``attend``: attention over such a cache, of one new token a sequence or of several
  (``attention.decode``, ``attention.prompt``);
* ``tree``: attention of a tree of drafted tokens a sequence, each of which sees its ancestors only
  (``attention.tree``);
* ``keep``: the accepted branch of each tree stays in the cache, the rest leaves it
  (``PagedCache.keep``).

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
NODES = 64  # the most drafted tokens of a tree


def listed():
    return [
        # interactive decoding: a few rows with all limits, where latency counts
        {"name": "sample_step", "op": "sample", "dtype": "f32", "rows": 4, "vocab": 32001,
         "limits": "mixed", "spread": 2.5},
        # a busy server's step: a large vocabulary, each request with settings of its own
        {"name": "sample_batch", "op": "sample", "dtype": "bf16", "rows": 256, "vocab": 128256,
         "limits": "mixed", "spread": 3.0},
        # samples for training: the whole distribution, many rows
        {"name": "sample_rollout", "op": "sample", "dtype": "bf16", "rows": 2000, "vocab": 50257,
         "limits": "none", "spread": 2.0},
        # a few chat turns are written into the 8-bit cache and one layer is read back
        {"name": "store_small", "op": "store", "dtype": "f16", "batch": 5, "most": 60, "page": 16,
         "heads": 2, "dim": 64, "ragged": 1},
        # a full prefill batch of one layer
        {"name": "store_large", "op": "store", "dtype": "bf16", "batch": 40, "most": 4096,
         "page": 16, "heads": 8, "dim": 128, "ragged": 2},
        # interactive decoding over an 8-bit cache: few, short sequences
        {"name": "attend_small", "op": "attend", "dtype": "f16", "batch": 4, "new": 1, "most": 777,
         "page": 16, "heads": 4, "group": 4, "dim": 128, "window": 0, "sinks": 0, "ragged": 3},
        # a serving batch over long, ragged contexts
        {"name": "attend_long", "op": "attend", "dtype": "bf16", "batch": 48, "new": 1,
         "most": 32768, "page": 16, "heads": 8, "group": 8, "dim": 128, "window": 0, "sinks": 0,
         "ragged": 4},
        # the next chunk of two long documents
        {"name": "attend_chunk", "op": "attend", "dtype": "bf16", "batch": 2, "new": 2048,
         "most": 8192, "page": 16, "heads": 8, "group": 4, "dim": 128, "window": 0, "sinks": 0,
         "ragged": 5},
        # small trees of drafted tokens, a few users
        {"name": "tree_small", "op": "tree", "dtype": "f16", "batch": 3, "new": 7, "most": 1500,
         "page": 16, "heads": 4, "group": 5, "dim": 64, "window": 0, "sinks": 0, "ragged": 6},
        # full trees over long contexts
        {"name": "tree_large", "op": "tree", "dtype": "bf16", "batch": 16, "new": 64,
         "most": 16384, "page": 16, "heads": 8, "group": 4, "dim": 128, "window": 0, "sinks": 0,
         "ragged": 7},
        # the accepted branches of a few users in a shallow model
        {"name": "keep_small", "op": "keep", "dtype": "bf16", "batch": 3, "new": 7, "most": 300,
         "layers": 4, "page": 16, "heads": 4, "dim": 64, "ragged": 8},
        # ... of a busy server in a deep one
        {"name": "keep_large", "op": "keep", "dtype": "f16", "batch": 96, "new": 64, "most": 900,
         "layers": 32, "page": 16, "heads": 8, "dim": 128, "ragged": 9},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("sample", "store", "attend", "tree", "keep"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    ragged = rng.randrange(1 << 20)
    if op == "sample":
        vocab = _log(rng, 500, 150000)
        return {"op": op, "dtype": dtype, "rows": _log(rng, 1, min(4000, 33_000_000 // vocab)),
                "vocab": vocab, "spread": rng.uniform(0.5, 4.0),
                "limits": rng.choice(("none", "top_k", "top_p", "min_p", "mixed", "mixed"))}
    page = rng.choice((8, 16, 16, 32, 64, 24))
    dim = rng.choice((64, 128, 128, 96))
    if op == "store":
        most = _log(rng, 8, 4096)
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, max(1, min(64, 80_000 // most))),
                "most": most, "page": page, "heads": rng.randint(1, 8), "dim": dim,
                "ragged": ragged}
    if op == "keep":
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, 96), "new": rng.randint(2, NODES),
                "most": _log(rng, 64, 900), "layers": rng.randint(1, 16), "page": page,
                "heads": rng.randint(1, 8), "dim": dim, "ragged": ragged}
    window = rng.choice((0, _log(rng, 16, 4096)))
    case = {"op": op, "dtype": dtype, "page": page, "dim": dim, "window": window,
            "sinks": rng.choice((0, 4, 64)) if window else 0, "ragged": ragged}
    if op == "tree":
        new, most = rng.randint(2, NODES), _log(rng, NODES, 16384)
        return case | {"batch": _log(rng, 1, max(1, min(32, 100_000 // most))), "new": new,
                       "most": most, "heads": rng.randint(1, 8),
                       "group": rng.choice((1, 2, 4, 5, 8))}
    if rng.random() < 0.6:
        most = _log(rng, 16, 65536)
        return case | {"batch": _log(rng, 1, max(1, min(128, 400_000 // most))), "new": 1,
                       "most": most, "heads": rng.randint(1, 8),
                       "group": rng.choice((1, 2, 4, 7, 8, 16))}
    new = _log(rng, 2, 2048)
    return case | {"batch": _log(rng, 1, max(1, min(16, 2048 // new))), "new": new,
                   "most": _log(rng, new, 8192), "heads": rng.randint(1, 4),
                   "group": rng.choice((1, 2, 4, 5, 8))}


# --- what a case's sequences look like (from the case alone: work() goes by them) ------------


def _lens(case, lo=1):
    """Ragged lengths up to the case's longest, one of them the longest itself."""
    rng = random.Random(case["ragged"])
    most, count = case["most"], case["batch"]
    lens = [int(round(lo + (most - lo) * rng.random() ** 1.5)) for _ in range(count)]
    lens[rng.randrange(count)] = most
    return lens


def _news(case, lens):
    """New tokens of each sequence: up to the case's, never past its length."""
    if case["new"] == 1:
        return [1] * len(lens)
    rng = random.Random(case["ragged"] + 1)
    return [min(n, case["new"] if i == 0 else rng.randint((case["new"] + 1) // 2, case["new"]))
            for i, n in enumerate(lens)]


def _sequences(case):
    """(lengths, new tokens of each): what every operator over a cache goes by."""
    if case["op"] == "store":
        lens = _lens(case)
        return lens, lens
    lens = _lens(case, 0 if case["op"] == "attend" and case["new"] == 1 else 1)
    return lens, _news(case, lens)


def _parents(case, news):
    """A random tree over each sequence's new tokens: node 0 is the last accepted token, a node's
    parent is one of the few before it (so that trees are some levels deep), -1 for the root."""
    rng = random.Random(case["ragged"] + 2)
    return [[-1] + [rng.randint(max(0, (i - 1) // 3 - 1), (i - 1) // 2) for i in range(1, n)]
            for n in news]


def _ancestors(parents):
    """Bit j of a node's mask: node j is an ancestor of it, or the node itself."""
    masks = []
    for i, p in enumerate(parents):
        masks.append(1 << i | (masks[p] if p >= 0 else 0))
    return masks


def _signed(mask):
    return mask - (1 << 64) if mask >> 63 else mask


def _kept(case, news):
    """The accepted nodes of each sequence: the root and a few of the later nodes."""
    rng = random.Random(case["ragged"] + 3)
    out = []
    for n in news:
        more = min(rng.randint(0, 6), (n - 1) // 2)
        out.append([0] + sorted(rng.sample(range(more + 1, n), more)))
    return out


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _pages_of(tokens, page):
    return -(-tokens // page)


def _tables(counts, pages, g):
    """A table of scattered pages: row i holds counts[i] pages, -1 past them."""
    width = max(1, max(counts))
    ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = ids[at:at + n]
        at += n
    return table


def _settings(case, g, s):
    """Each row's temperature, top-k, top-p and min-p, as the requests of a batch have them."""
    rows, limits = case["rows"], case["limits"]

    def some(values):
        pick = torch.randint(0, len(values), (rows,), device="cuda", generator=g)
        return torch.tensor(values, device="cuda")[pick]

    s["temperature"] = some([0.6, 0.8, 1.0, 1.2] + ([0.0] if limits == "mixed" else []))
    k = some([20, 50, 200, 5000]) if limits == "top_k" else some([0, 0, 40, 1000])
    s["top_k"] = k.to(torch.int32) if limits in ("top_k", "mixed") else None
    s["top_p"] = some([0.5, 0.8, 0.9, 0.95, 0.99]) if limits in ("top_p", "mixed") else None
    s["min_p"] = some([0.0, 0.05, 0.01]) if limits in ("min_p", "mixed") else None


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if own:
        package = str(Path(__file__).resolve().parents[1] / "emmy-hackathon-submission_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "sample":
        x = torch.randn((case["rows"], case["vocab"]), device="cuda", generator=g)
        s["logits"] = (x * case["spread"]).to(dtype)
        s["uniform"] = torch.rand(case["rows"], device="cuda", generator=g)
        _settings(case, g, s)
        return s
    page, heads, dim = case["page"], case["heads"], case["dim"]
    lens, news = _sequences(case)
    counts = [_pages_of(n, page) for n in lens]
    pages = sum(counts) + 3
    shape = (case.get("layers", 1), pages, heads, page, dim)
    s |= {"lens": _ints(lens), "starts": _ints(_starts(news)), "table": _tables(counts, pages, g),
          "slots": _ints(list(range(len(lens))))}
    if op in ("store", "attend"):
        s["k"], s["v"] = (torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda",
                                        generator=g) for _ in range(2))
        # rows of unlike size: a scale of about 1 / 40, as normal rows have, and up to e^2 off
        s["k_scale"], s["v_scale"] = (
            (torch.randn(shape[:-1], device="cuda", generator=g).clamp_(-2, 2)).exp_() / 60
            for _ in range(2))
    else:
        s["k"], s["v"] = (torch.randn(shape, device="cuda", dtype=dtype, generator=g)
                          for _ in range(2))
    tokens = sum(news)
    if op == "store":
        fused = torch.randn((tokens, 2 * heads, dim), device="cuda", generator=g)
        fused *= torch.randn((tokens, 2 * heads, 1), device="cuda", generator=g).exp_()
        fused = fused.to(dtype)
        s |= {"new_k": fused[:, :heads], "new_v": fused[:, heads:]}
    elif op in ("attend", "tree"):
        hq = heads * case["group"]
        # queries as a model has them: the first heads of a fused projection's rows
        fused = torch.randn((tokens, hq + 2 * heads, dim), device="cuda", generator=g)
        s |= {"q": fused.to(dtype)[:, :hq], "scale": dim ** -0.5}
    if op == "tree":
        s["mask"] = _ints([_signed(m) for p in _parents(case, news) for m in _ancestors(p)],
                          torch.int64)
    if op == "keep":
        s["kept"] = _ints([_signed(sum(1 << i for i in k)) for k in _kept(case, news)],
                          torch.int64)
    if op in ("store", "keep"):
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        held = s["table"][s["table"] >= 0].long()
        refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
        s["refs"] = refs
        s |= {"refs0": refs.clone(), "table0": s["table"].clone(), "lens0": s["lens"].clone()}
    if own:
        if op in ("store", "keep"):
            from ptxgen.cache import PagedCache

            s["cache"] = PagedCache(s["k"], s["v"], s["refs"], s["table"], s["lens"],
                                    k_scale=s.get("k_scale"), v_scale=s.get("v_scale"))
        else:
            from ptxgen.attention import Workspace

            s["workspace"] = Workspace()
    return s


# --- the plain forms --------------------------------------------------------------------------


def _run_sample(s):
    x = s["logits"]
    if own:
        from ptxgen import sampling

        limits = {n: s[n] for n in ("top_k", "top_p", "min_p") if s[n] is not None}
        r = sampling.sample(x, s["uniform"], temperature=s["temperature"], **limits)
        return {"tokens": r.tokens, "logp": r.logp}
    # in 64 bits: a token next to a border must not depend on how sums are rounded
    rows, vocab = x.shape
    t = s["temperature"].double()[:, None]
    greedy = t == 0
    x = x.float()
    top = x.amax(-1, keepdim=True)
    z = (x.double() - top.double()) / torch.where(greedy, 1.0, t)
    if s["top_k"] is None and s["top_p"] is None and s["min_p"] is None:
        w = z.exp_()
    else:
        values, ids = x.sort(dim=-1, descending=True, stable=True)
        w = z.exp().gather(1, ids)
        place = torch.arange(vocab, device=x.device)[None]
        keep = torch.ones((rows, vocab), dtype=torch.bool, device=x.device)
        if s["top_k"] is not None:
            k = s["top_k"][:, None]
            keep &= (place < k) | (k <= 0)
        if s["top_p"] is not None:
            p = s["top_p"].double()[:, None]
            upto = torch.where(keep, w, 0.0).cumsum(-1)
            keep &= (upto - w < p * upto[:, -1:]) | (p >= 1)
        if s["min_p"] is not None:
            keep &= w >= s["min_p"].double()[:, None]
        keep &= ~greedy
        keep[:, 0] = True
        kept = torch.zeros_like(keep).scatter_(1, ids, keep)
        w = torch.where(kept, z.exp_(), 0.0)
    upto = w.cumsum(-1)
    total = upto[:, -1:].contiguous()
    tokens = torch.searchsorted(upto, s["uniform"].double()[:, None] * total, right=True)
    tokens.clamp_(max=vocab - 1)
    logp = (w.gather(1, tokens) / total).log()
    return {"tokens": tokens[:, 0], "logp": logp[:, 0].float()}


def _run_store(s):
    case = s["case"]
    tokens, dtype = s["new_k"].shape[0], DTYPES[case["dtype"]]
    if own:
        cache = s["cache"]
        cache.write(0, s["slots"], s["starts"], s["new_k"], s["new_v"])
        k, v = cache.read(0, s["slots"], s["starts"], tokens, dtype=dtype)
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    page, starts = case["page"], s["starts"].long()
    t = torch.arange(tokens, device=starts.device)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    pos = s["lens"].long()[seq] - starts[seq + 1] + t
    where, row = s["table"][seq, pos // page].long(), pos % page
    out = {}
    for name in ("k", "v"):
        x = s["new_" + name].float()
        scale = x.abs().amax(-1) / 127
        # in 64 bits, where a quotient between two whole numbers is seen as it is
        q = (x.double() / torch.where(scale > 0, scale, 1.0).double()[..., None]).round()
        s[name][0][where, :, row] = q.to(torch.int8)
        s[name + "_scale"][0][where, :, row] = scale
        back = s[name][0][where, :, row].float() * s[name + "_scale"][0][where, :, row][..., None]
        out[name] = back.to(dtype)
    return out | {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(q, seen, k, v, k_scale, v_scale, table, lens, scale):
    """softmax(q k^T scale) v for queries q [batch, rows, group, heads, dim] over the keys that seen
    [batch, rows, keys] names; a row that sees no key gives zeros."""
    b, width = table.shape
    heads, page, dim = k.shape[1:]
    span = width * page
    inside = torch.arange(span, device=q.device)[None] < lens[:, None]
    ids = table.clamp(min=0).long()

    def rows_of(x, x_scale):
        y = x[ids].float()
        if x_scale is not None:
            y = y * x_scale[ids][..., None]
        return y.permute(0, 2, 1, 3, 4).reshape(b, heads, span, dim)

    kk = rows_of(k, k_scale)
    vv = torch.where(inside[:, None, :, None], rows_of(v, v_scale), 0.0)
    rows, group = q.shape[1:3]
    qq = q.permute(0, 3, 1, 2, 4).reshape(b, heads, rows * group, dim).float()
    s = (qq @ kk.transpose(-1, -2)) * scale
    seen = seen[:, None, :, None].expand(b, 1, rows, group, span).reshape(b, 1, -1, span)
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.where(total > 0, (s @ vv) / total, 0.0)
    return o.reshape(b, heads, rows, group, dim).permute(0, 2, 3, 1, 4)


def _run_attention(s):
    """``attend`` and ``tree``."""
    case, q, tree = s["case"], s["q"], s["case"]["op"] == "tree"
    k, v = s["k"][0], s["v"][0]
    if own:
        from ptxgen import attention

        more = dict(scale=s["scale"], window=case["window"], sinks=case["sinks"],
                    workspace=s["workspace"])
        if tree:
            return attention.tree(q, s["starts"], s["mask"], k, v, s["table"], s["lens"], **more)
        more |= dict(k_scale=s["k_scale"][0], v_scale=s["v_scale"][0])
        if case["new"] == 1:
            return attention.decode(q, k, v, s["table"], s["lens"], **more)
        return attention.prompt(q, s["starts"], k, v, s["table"], s["lens"], **more)
    starts, lens, hq, dim = s["starts"], s["lens"], q.shape[1], q.shape[2]
    rows = torch.arange(case["new"], device=q.device)
    news = starts[1:] - starts[:-1]
    real = rows[None] < news[:, None]
    at = (starts[:-1, None] + rows[None]).clamp(max=q.shape[0] - 1).long()
    qq = q[at].reshape(*at.shape, case["heads"], case["group"], dim).transpose(2, 3)
    keys = torch.arange(s["table"].shape[1] * case["page"], device=q.device)
    base = lens - news
    if tree:
        mask = s["mask"][at]
        bit = keys[None] - base[:, None]  # the new token that a key is
        mine = (mask[:, :, None] >> bit.clamp(0, NODES - 1)[:, None]) & 1 == 1
        # where a token stands is how many of the query's ancestors come before it
        bits = (mask[:, :, None] >> torch.arange(NODES, device=q.device)) & 1
        pos = base[:, None] + bits.sum(-1) - 1
        order = (bits.cumsum(-1) - bits).gather(2, bit.clamp(0, NODES - 1)[:, None].expand(
            -1, bits.shape[1], -1))
        place = torch.where(bit[:, None] < 0, keys, base[:, None, None] + order)
        seen = (bit < 0)[:, None] | (mine & (bit < news[:, None])[:, None])
    else:
        pos = base[:, None] + rows[None]
        place = keys[None, None]
        seen = place <= pos[:, :, None]
        seen = seen & (keys < lens[:, None])[:, None]
    if case["window"]:
        seen = seen & ((place > pos[:, :, None] - case["window"]) | (place < case["sinks"]))
    scales = (None, None) if tree else (s["k_scale"][0], s["v_scale"][0])
    o = _plain_attention(qq, seen, k, v, *scales, s["table"], lens, s["scale"])
    return o.transpose(2, 3).reshape(*at.shape, hq, dim)[real].to(q.dtype)


def _run_keep(s):
    # the same drafts each time: lengths, table and counts as they were (what has moved comes from
    # rows that no other move reaches, so the data is the drafts' too)
    for n in ("refs", "table", "lens"):
        s[n].copy_(s[n + "0"])
    names = ("k", "v", "table", "lens", "refs")
    if own:
        s["cache"].keep(s["slots"], s["starts"], s["kept"])
        return {n: s[n] for n in names}
    page, table, lens = s["case"]["page"], s["table"], s["lens"]
    starts = s["starts"].long()
    news = starts[1:] - starts[:-1]
    bits = ((s["kept"][:, None] >> torch.arange(NODES, device=lens.device)) & 1) == 1
    base = lens.long() - news
    rank = bits.long().cumsum(-1) - 1
    who, node = bits.nonzero(as_tuple=True)
    source, target = base[who] + node, base[who] + rank[who, node]
    a, b = table[who, source // page].long(), table[who, target // page].long()
    for x in (s["k"], s["v"]):
        x[:, b, :, target % page] = x[:, a, :, source % page]
    new_lens = base + bits.sum(-1)
    old, now = (lens.long() + page - 1) // page, (new_lens + page - 1) // page
    entry = torch.arange(table.shape[1], device=lens.device)[None]
    gone = (entry >= now[:, None]) & (entry < old[:, None])
    held = table[gone].long()
    s["refs"].index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    table[gone] = -1
    lens.copy_(new_lens)
    return {n: s[n] for n in names}


def run(state):
    return {"sample": _run_sample, "store": _run_store, "attend": _run_attention,
            "tree": _run_attention, "keep": _run_keep}[state["case"]["op"]](state)


# --- what a pass cannot do without ------------------------------------------------------------


def _seen(case, length, new, parents=None):
    """(keys that some of the sequence's new tokens see, pairs of a new token and a key)."""
    window, sinks = case["window"], case["sinks"]
    if not new or not length:
        return 0, 0
    base = length - new
    depths = [bin(m).count("1") for m in _ancestors(parents)] if parents else range(1, new + 1)
    if not window:
        return length, sum(base + d for d in depths)
    low = max(0, base - window + 1)  # the first new token's oldest key but the sinks
    pairs = 0
    for d in depths:
        first = max(0, base + d - window)
        pairs += base + d - first + min(sinks, first)
    return length - low + min(sinks, low), pairs


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "sample":
        n, rows = case["rows"] * case["vocab"], case["rows"]
        return {"bytes": n * size + rows * (12 + 4 + 4 * 4), "flops": 10 * n}
    page, heads, dim = case["page"], case["heads"], case["dim"]
    lens, news = _sequences(case)
    if case["op"] == "store":
        rows = 2 * sum(lens) * heads  # of keys and values
        moved = rows * (dim * size + dim + 4)  # read and quantised, then the other way
        return {"bytes": 2 * moved + 4 * (sum(_pages_of(n, page) for n in lens) + 2 * len(lens)),
                "flops": 5 * rows * dim}
    if case["op"] == "keep":
        moves = sum(sum(1 for r, i in enumerate(k) if r != i) for k in _kept(case, news))
        return {"bytes": 4 * moves * heads * dim * size * case["layers"] + 4 * 8 * len(lens),
                "flops": 0}
    tree = case["op"] == "tree"
    parents = _parents(case, news) if tree else [None] * len(lens)
    seen = [_seen(case, n, m, p) for n, m, p in zip(lens, news, parents)]
    keys, pairs = sum(a for a, _ in seen), sum(b for _, b in seen)
    token = heads * (dim * size if tree else dim + 4)  # one token's keys (or values)
    q = sum(news) * heads * case["group"] * dim * size
    return {"bytes": 2 * keys * token + 2 * q + 4 * (-(-keys // page) + 2 * len(lens))
            + (8 * sum(news) if tree else 0), "flops": 4 * pairs * heads * case["group"] * dim}


# --- the definitions in 64 bits -----------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "keep":
        return None  # copies and whole numbers
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "store":
        return _exact_store(s)
    return _exact_attention(s)


def _exact_sample(s):
    x, u = s["logits"], s["uniform"].tolist()

    def setting(name, none):
        return [none] * len(u) if s[name] is None else s[name].tolist()

    out = torch.empty(len(u), dtype=torch.float64, device=x.device)
    settings = zip(setting("temperature", 1.0), setting("top_k", 0), setting("top_p", 1.0),
                   setting("min_p", 0.0))
    for i, (t, k, p, least) in enumerate(settings):
        if t == 0:
            out[i] = 0.0
            continue
        row = x[i].double()
        best, order = torch.sort(row, descending=True, stable=True)
        if k > 0:
            best, order = best[:k], order[:k]
        prob = torch.softmax(best / t, 0)
        n = prob.numel()
        if p < 1:
            reached = (prob.cumsum(0) >= p).nonzero()
            n = min(n, int(reached[0]) + 1 if reached.numel() else n)
        if least > 0:
            n = min(n, int((prob >= least * prob[0]).sum()))
        n = max(n, 1)
        columns, sorted_at = order[:n].sort()
        prob = prob[:n][sorted_at] / prob[:n].sum()
        at = min(int((prob.cumsum(0) <= u[i]).sum()), n - 1)
        out[i] = prob[at].log()
    return {"tokens": None, "logp": out}


def _exact_store(s):
    """The quantised rows of each token in turn; the scale is the f32 number that the cache holds."""
    out = {}
    for name in ("k", "v"):
        x = s["new_" + name].double()
        scale = (s["new_" + name].float().abs().max(-1).values / 127).double()
        steps = torch.where(scale[..., None] > 0, x / scale[..., None], 0.0)
        out[name] = torch.round(steps) * scale[..., None]
    page, starts = s["case"]["page"], s["starts"].tolist()
    for name in ("k", "v"):
        scales = s[name + "_scale"].double()
        new = (s["new_" + name].float().abs().max(-1).values / 127).double()
        for i, n in enumerate(s["lens"].tolist()):
            ids = s["table"][i, :_pages_of(n, page)].long()
            rows = scales[0, ids].transpose(1, 2).reshape(-1, new.shape[1]).clone()
            rows[:n] = new[starts[i]:starts[i + 1]]
            scales[0, ids] = rows.reshape(-1, page, new.shape[1]).transpose(1, 2)
        out[name + "_scale"] = scales
    return out


def _exact_attention(s):
    case, q, starts = s["case"], s["q"], s["starts"].tolist()
    heads, group, page, dim = case["heads"], case["group"], case["page"], case["dim"]
    tree = case["op"] == "tree"
    lens, news = _sequences(case)
    trees = _parents(case, news) if tree else None
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if n == 0 or a == b:
            continue
        base = n - (b - a)
        hidden = torch.zeros((b - a, n), dtype=torch.bool)
        at = torch.arange(n)
        for r in range(b - a):
            if tree:
                path = [r]  # from the node up to the root
                while trees[i][path[-1]] >= 0:
                    path.append(trees[i][path[-1]])
                sees = list(range(base)) + [base + t for t in reversed(path)]
            else:
                sees = list(range(base + r + 1)) if case["window"] == 0 else None
            if sees is None:
                p = base + r
                hidden[r] = (at > p) | ((at <= p - case["window"]) & (at >= case["sinks"]))
                continue
            sees = torch.tensor(sees)
            if case["window"]:
                place = torch.arange(len(sees))
                sees = sees[(place > len(sees) - 1 - case["window"]) | (place < case["sinks"])]
            hidden[r] = True
            hidden[r, sees] = False
        hidden = hidden.to(q.device)
        ids = s["table"][i, :_pages_of(n, page)].long()
        for h in range(heads):
            k = s["k"][0][ids, h].reshape(-1, dim)[:n].double()
            v = s["v"][0][ids, h].reshape(-1, dim)[:n].double()
            if not tree:
                k = k * s["k_scale"][0][ids, h].reshape(-1)[:n, None].double()
                v = v * s["v_scale"][0][ids, h].reshape(-1)[:n, None].double()
            for r in range(h * group, (h + 1) * group):
                w = (q[a:b, r].double() @ k.T) * s["scale"]
                w[hidden] = -math.inf
                out[a:b, r] = torch.softmax(w, -1) @ v
    return out
