"""Attention over a paged key-value cache: one new token a sequence, or several.

    ws = Workspace()                                     # once, one per stream
    out = decode(q, k, v, table, lens, workspace=ws)     # q [batch, heads, dim]
    out = prompt(q, starts, k, v, table, lens, workspace=ws)   # q [tokens, heads, dim]
    out = tree(q, starts, mask, k, v, table, lens, workspace=ws)   # drafted tokens of several branches

``k`` and ``v`` are one layer's pages [pages, kv_heads, page_size, dim] (``PagedCache.k[layer]``),
``table`` [slots, width] and ``lens`` [slots] the cache's; sequence b of the batch is row
``slots[b]`` of them, or row b. The queries are a sequence's last tokens, already written to the
cache: row b of q for ``decode``, rows ``starts[b]`` to ``starts[b + 1]`` for ``prompt``. A query
at position p sees key j when j <= p and, with a ``window``, j > p - window or j < ``sinks``. A
query that sees no key gives zeros; what lies past a sequence's length or in a masked place is
never part of a result. A visible value that is not finite makes its column of the result so: an
infinity, where all such values are that one (or NaN, where its weight is below 2^-126). Each group of heads / kv_heads query heads reads one kv head.

The new tokens of a sequence may be a ``tree``, 64 at most: each sees the tokens before them and those
of its own branch, which ``mask`` names (``branches`` makes it of the tokens' parents).

Over a cache in 8 bits, ``k_scale`` and ``v_scale`` [pages, kv_heads, page_size] are one layer's scales
(``PagedCache.k_scale[layer]``) and k and v int8. For few rows keys and values are what they stand for, and
only the weights' products with the values' scales are rounded, to f16 numbers (one each for bf16 results,
else two). Prompts of many rows, as below, with bf16 results have keys and values rounded to f16, too, as
have f16 ones (and one number a weight) where the workspace has no room for one kv head's keys
and values in 16 bits (96000 tokens of heads of 128 in all, by ``max_len`` or the table's width, in one of
the default size). What is below 2^-22 of the largest scale loses digits there. A key or value whose scale is not finite makes the results
that see it NaN. ``max_len`` must not be below a length then: such a sequence is cut, and ``Workspace.check``
raises for it.

q, k and v have one dtype (f32, bf16 or f16; k and v may be int8) and a head size of up to 256 whose rows are a
multiple of 16 bytes; q may be a slice of a fused projection. Scores, maxima and sums are held in 32
bits. bf16 and f16 results are rounded to their type; prompts of more than 48 rows (tokens times heads
/ kv_heads) a sequence on average with heads of up to 128 round each weight to it as well, before its
product with a value. Rows of q that no sequence has leave theirs of the result as they are. Nothing waits for the GPU; where only the device can see that a slot, page id or length is
out of range, nothing is read, that sequence's result is not defined, and bits are set that
``Workspace.check`` raises as ``CacheError``. Calls run on the current stream, or on ``stream`` (a
``cudaStream_t`` as an integer), whose memory a new result then comes from: other streams wait for
it and call ``record_stream``, as for any tensor of another stream. The kernels are ``csrc/attention*.cu``
(``pg_attention``).
"""

from __future__ import annotations

import ctypes
import struct
from typing import Any

import torch

from .cache import CacheError
from .launch import call, dtype_code, empty, int32_list, take_status, wait_until_set
from .runtime import AttentionArgs, AttentionMore, library

WORKSPACE_BYTES = 64 << 20  # PG_ATTENTION_WORKSPACE
DIM_MAX = 256  # PG_ATTENTION_DIM
TREE_MAX = 64  # PG_ATTENTION_TREE
# pg_attention_args at once: setting its fields one by one takes longer than a short call
_PACK = struct.Struct("=9Q10q13if")
assert _PACK.size == ctypes.sizeof(AttentionArgs)
_PACK_MORE = struct.Struct("=2Q4qQ")  # pg_attention_more
assert _PACK_MORE.size == ctypes.sizeof(AttentionMore)


class Workspace:
    """The device memory in which attention leaves the parts of a long sequence's result until
    they are joined, and widens the keys and values of prompts over 8 bits. One per stream: calls that
    overlap on the GPU must not share it. It has to live until the calls that were given it have run.
    ``size`` in bytes may be more than the default: trees and long prompts over 8 bits make use of it."""

    def __init__(self, device: Any = None, size: int = WORKSPACE_BYTES):
        if size < WORKSPACE_BYTES:
            raise ValueError(f"size {size}: want {WORKSPACE_BYTES} bytes at least")
        self.buffer = torch.zeros(size // 4, dtype=torch.int32,
                                  device="cuda" if device is None else device)
        self.size = size // 4 * 4
        self.device = self.buffer.device  # with an index, as a call's tensors have it
        wait_until_set(self.device)

    def check(self) -> None:
        """Wait for the GPU, all its streams, and raise ``CacheError`` if an earlier call met a slot,
        page id or starts out of range (the bits are cleared)."""
        bits = take_status(self.buffer[:1])
        if bits:
            raise CacheError(bits)


def _call(q: Any, starts: Any, k: Any, v: Any, table: Any, lens: Any, slots: Any,
          scale: float | None, window: int, sinks: int, max_len: int | None, workspace: Workspace,
          out: Any, stream: int | None, k_scale: Any, v_scale: Any, mask: Any = None) -> Any:
    dev, dtype, size = q.device, q.dtype, q.element_size()
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if len(qs) != 3 or not q.is_cuda or qs[2] != 1:
        raise ValueError(f"q: want [tokens, heads, dim] on a CUDA device with contiguous rows, "
                         f"got {tuple(q.shape)} {q.stride()} on {dev}")
    tokens, hq, dim = q.shape
    shape, of = k.shape, dtype if k_scale is None else torch.int8
    for name, t, s in (("k", k, ks), ("v", v, vs)):
        if len(s) != 4 or t.dtype is not of or t.device != dev or t.shape != shape or \
                shape[3] != dim or s[3] != 1 or s[2] != dim:
            raise ValueError(f"{name}: want {of} [pages, kv_heads, page_size, {dim}] on {dev} "
                             f"with a head's rows of one page one after another, got {t.dtype} "
                             f"{tuple(t.shape)} {t.stride()} on {t.device}")
    pages, heads, page_size, _ = shape
    if not heads or hq % heads:
        raise ValueError(f"{hq} query heads are no multiple of {heads} kv heads")
    if table.dtype is not torch.int32 or table.dim() != 2 or table.stride(1) != 1 or \
            table.device != dev:
        raise ValueError(f"table: want int32 [slots, width] on {dev} with contiguous rows")
    rows, width = table.shape
    if slots is not None:
        batch = slots.shape[0]
        slots = int32_list("slots", slots, dev)
    else:
        batch = rows if starts is None else starts.shape[0] - 1
        slots = 0
        if batch > rows:
            raise ValueError(f"{batch} sequences, but table has {rows} rows")
    if starts is None:
        if batch != tokens:
            raise ValueError(f"q has {tokens} tokens for {batch} sequences")
    else:
        starts = int32_list("starts", starts, dev, batch + 1)
    if workspace.device != dev:
        raise ValueError(f"the workspace is on {workspace.device}, q on {dev}")
    if out is None:
        out = empty((tokens, hq, dim), dtype, dev, stream)
    elif out.shape != q.shape or out.dtype != dtype or out.device != dev or out.stride(2) != 1:
        raise ValueError(f"out: want {dtype} {tuple(q.shape)} on {dev} with contiguous rows")
    os_ = out.stride()
    size_kv = size if k_scale is None else 1
    args = AttentionArgs()
    try:
        _PACK.pack_into(
            args, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), starts or 0, slots,
            table.data_ptr(), int32_list("lens", lens, dev, rows), workspace.buffer.data_ptr(),
            workspace.size, qs[0] * size, qs[1] * size, os_[0] * size, os_[1] * size,
            ks[0] * size_kv, ks[1] * size_kv, vs[0] * size_kv, vs[1] * size_kv, table.stride(0),
            dtype_code(dtype), batch, tokens, heads, hq // heads, dim, page_size, pages, width, rows,
            window, sinks, max_len or 0, dim ** -0.5 if scale is None else scale)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"window, sinks, max_len, scale or a size is out of range: {e}") from e
    if k_scale is None and v_scale is None and mask is None:
        call(library().pg_attention, dev, stream, args)
    else:
        call(library().pg_attention_ex, dev, stream, args,
             _more(dev, tokens, shape[:3], k_scale, v_scale, mask))
    return out


def _more(dev: Any, tokens: int, rows: Any, k_scale: Any, v_scale: Any, mask: Any) -> AttentionMore:
    scales, at = (0, 0, 0, 0, 0, 0), 0
    if k_scale is not None or v_scale is not None:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is None or t.dtype is not torch.float32 or t.shape != rows or t.device != dev or \
                    (rows[2] > 1 and t.stride(2) != 1):
                raise ValueError(f"{name}: want float32 {tuple(rows)} on {dev} with a page's rows one "
                                 f"after another, got {t if t is None else (t.dtype, t.shape)}")
        ks, vs = k_scale.stride(), v_scale.stride()
        scales = (k_scale.data_ptr(), v_scale.data_ptr(), 4 * ks[0], 4 * ks[1], 4 * vs[0], 4 * vs[1])
    if mask is not None:
        if mask.dtype is not torch.int64 or mask.shape != (tokens,) or not mask.is_contiguous() or \
                mask.device != dev:
            raise ValueError(f"mask: want contiguous int64 [{tokens}] on {dev}, got {mask.dtype} "
                             f"{tuple(mask.shape)} on {mask.device}")
        at = mask.data_ptr()
    more = AttentionMore()
    _PACK_MORE.pack_into(more, 0, *scales, at)
    return more


def decode(q: Any, k: Any, v: Any, table: Any, lens: Any, *, workspace: Workspace,
           slots: Any = None, scale: float | None = None, window: int = 0, sinks: int = 0,
           max_len: int | None = None, out: Any = None, k_scale: Any = None, v_scale: Any = None,
           stream: int | None = None) -> Any:
    """Attention of one new token a sequence, ``q`` [batch, heads, dim]: the last of each
    sequence's ``lens`` tokens. ``max_len`` may name the longest length (it only shapes the
    launch); ``scale`` is dim ** -0.5 by default."""
    return _call(q, None, k, v, table, lens, slots, scale, window, sinks, max_len, workspace, out,
                 stream, k_scale, v_scale)


def prompt(q: Any, starts: Any, k: Any, v: Any, table: Any, lens: Any, *, workspace: Workspace,
           slots: Any = None, scale: float | None = None, window: int = 0, sinks: int = 0,
           max_len: int | None = None, out: Any = None, k_scale: Any = None, v_scale: Any = None,
           stream: int | None = None) -> Any:
    """Causal attention of each sequence's last tokens, ``q`` [tokens, heads, dim] with sequence
    b's in rows ``starts[b]`` to ``starts[b + 1]`` (int32, on the device)."""
    return _call(q, starts, k, v, table, lens, slots, scale, window, sinks, max_len, workspace,
                 out, stream, k_scale, v_scale)


def tree(q: Any, starts: Any, mask: Any, k: Any, v: Any, table: Any, lens: Any, *,
         workspace: Workspace, slots: Any = None, scale: float | None = None, window: int = 0,
         sinks: int = 0, max_len: int | None = None, out: Any = None, k_scale: Any = None,
         v_scale: Any = None, stream: int | None = None) -> Any:
    """Attention of each sequence's last tokens, at most 64, as a tree: bit t of ``mask[i]`` (int64
    [tokens], on the device) says whether token i sees the t-th of its sequence's new tokens, itself
    among them. Those n stand one behind the other from base on, the length less the new tokens, and
    token i at base + n - 1; window and sinks go by that. All see the tokens before base."""
    if mask is None:
        raise ValueError("mask: a tree of tokens wants one")
    return _call(q, starts, k, v, table, lens, slots, scale, window, sinks, max_len, workspace,
                 out, stream, k_scale, v_scale, mask)


def branches(parents: list[int]) -> list[int]:
    """The masks of one sequence's new tokens (as signed 64-bit numbers, for ``torch.tensor``) from
    their parents' indices, -1 for one that has none: each token's bit and those of its ancestors. Parents
    come before their children."""
    if len(parents) > TREE_MAX:
        raise ValueError(f"{len(parents)} tokens, want {TREE_MAX} at most")
    masks: list[int] = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"parent {p} of token {i}: want -1 to {i - 1}")
        masks.append(1 << i | (masks[p] if p >= 0 else 0))
    return [m - (1 << 64) if m >> 63 else m for m in masks]
