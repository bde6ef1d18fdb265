"""A paged key-value cache: the pages a batch of sequences keeps its keys and values in.

``PagedCache`` holds the cache's tensors and calls the page operations of the C ABI
(``pg_cache_*`` in ``include/ptxgen_b200.h``) on them:

    cache = PagedCache.allocate(layers=2, pages=1024, heads=8, page_size=16, dim=128, slots=64,
                                width=256)
    cache.extend(slots, starts)                  # room for each sequence's new tokens
    cache.write(layer, slots, starts, k, v)      # their keys and values, layer by layer
    cache.fork(parents, children)                # continuations that share full pages
    cache.free(slots)                            # finished sequences let go of their pages
    cache.compact()                              # the live pages move to the front
    cache.check()                                # raises CacheError if a call could not be met

``ptxgen.attention`` reads the cache's ``k``, ``v``, ``table`` and ``lens``. Slots, starts and page
ids are int32 device tensors, and nothing here waits for the GPU but ``check`` and the making of a
cache: what only the device can see (no page left, a slot listed twice) sets bits of ``status``, and an ``extend`` or
``fork`` that cannot be met changes nothing. A ``write`` that was queued behind a refused ``extend``
leaves out that call's slots, since their last tokens are older ones, until an ``extend`` of them is
met (by no tokens, if need be) or they are freed. Calls run on the current stream, or on ``stream``
(a ``cudaStream_t`` as an integer); a cache's calls belong on one stream at a time, and the cache
has to live until they have run.
"""

from __future__ import annotations

import ctypes
from typing import Any

import torch

from .launch import call, int32_list, take_status, wait_until_set
from .runtime import Cache, LaunchError, Rows, library

NO_PAGES, BAD_SLOT, BAD_PAGE, TOO_LONG, WAIT, REFUSED = 1, 2, 4, 8, 16, 32
_WHY = {NO_PAGES: "fewer free pages than a call needed",
        BAD_SLOT: "a slot out of range, listed twice, or a fork's child in use",
        BAD_PAGE: "a page id or count out of range",
        TOO_LONG: "more tokens than a table row has pages for, or than there are rows",
        WAIT: "a bounded wait inside an attention kernel gave up",
        REFUSED: "rows of a slot whose last extend could not be met were not written"}


class CacheError(LaunchError):
    """A page operation could not be met; ``bits`` are those of the cache's status word."""

    def __init__(self, bits: int):
        self.bits = bits
        super().__init__("; ".join(w for b, w in _WHY.items() if bits & b))


class PagedCache:
    """The cache over ``k`` and ``v`` [layers, pages, heads, page_size, dim], ``refs`` [pages],
    ``table`` [slots, width] and ``lens`` [slots] (int32). A head's rows of one page lie one
    after another; the other strides are free but multiples of 16 bytes and the same for both."""

    def __init__(self, k: Any, v: Any, refs: Any, table: Any, lens: Any):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v: want one shape [layers, pages, heads, page_size, dim], "
                             f"dtype and strides, got {k.dtype} {tuple(k.shape)} {k.stride()} "
                             f"and {v.dtype} {tuple(v.shape)} {v.stride()}")
        layers, pages, heads, page_size, dim = k.shape
        size = k.element_size()
        if (dim > 1 and k.stride(4) != 1) or (page_size > 1 and k.stride(3) != dim):
            raise ValueError(f"k and v: strides {k.stride()}: a head's rows of one page must lie "
                             "one after another")
        if not k.is_cuda or any(t.device != k.device for t in (v, refs, table, lens)):
            raise ValueError("the cache's tensors must be on one CUDA device")
        if table.dtype is not torch.int32 or table.dim() != 2 or table.stride(1) != 1:
            raise ValueError("table: want int32 [slots, width] with contiguous rows")
        self.k, self.v, self.refs, self.table, self.lens = k, v, refs, table, lens
        self.device, self._size, self._row_shape = k.device, size, torch.Size((heads, dim))
        slots, width = table.shape
        words = 4 + 3 * pages + 2 * slots + 2
        self._scratch = torch.empty(words, dtype=torch.int32, device=k.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._refused = torch.zeros(slots, dtype=torch.int32, device=k.device)
        self._c = Cache(
            k.data_ptr(), v.data_ptr(), k.stride(0) * size, k.stride(1) * size,
            k.stride(2) * size, int32_list("refs", refs, k.device, pages), table.data_ptr(),
            int32_list("lens", lens, k.device, slots), self.status.data_ptr(),
            self._scratch.data_ptr(), self._refused.data_ptr(), max(table.stride(0), width), words, layers, pages, heads,
            page_size, dim * size, slots, width)
        wait_until_set(self.device)
        self._ref = ctypes.byref(self._c)
        self._lib = library()

    @classmethod
    def allocate(cls, layers: int, pages: int, heads: int, page_size: int, dim: int, slots: int,
                 width: int, dtype: Any = None, device: Any = None) -> PagedCache:
        """An empty cache: ``pages`` free pages, ``slots`` empty slots of up to ``width`` pages."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        shape = (layers, pages, heads, page_size, dim)
        k, v = (torch.empty(shape, dtype=dtype or torch.bfloat16, device=dev) for _ in range(2))
        refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        table = torch.full((slots, width), -1, dtype=torch.int32, device=dev)
        return cls(k, v, refs, table, torch.zeros(slots, dtype=torch.int32, device=dev))

    def _rows(self, name: str, t: Any) -> Rows:
        if t.dtype is not self.k.dtype or t.dim() != 3 or t.shape[1:] != self._row_shape or \
                t.device != self.device or t.stride(2) != 1:
            raise ValueError(f"{name}: want {self.k.dtype} [tokens, {self._row_shape[0]}, "
                             f"{self._row_shape[1]}] on {self.device} with contiguous rows, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        size = self._size
        return Rows(t.data_ptr(), t.stride(0) * size, t.stride(1) * size)

    def extend(self, slots: Any, starts: Any, stream: int | None = None) -> None:
        """Make room for new tokens: ``slots[i]`` grows by ``starts[i + 1] - starts[i]`` tokens."""
        n, dev = slots.shape[0], self.device
        call(self._lib.pg_cache_extend, dev, stream, self._ref, int32_list("slots", slots, dev),
             int32_list("starts", starts, dev, n + 1), n)

    def write(self, layer: int, slots: Any, starts: Any, k: Any, v: Any,
              stream: int | None = None) -> None:
        """Write one layer's ``k`` and ``v`` [tokens, heads, dim] of the slots' last tokens:
        rows ``starts[i]`` to ``starts[i + 1]`` are the last ones of ``slots[i]``. Rows past the last
        of ``starts`` belong to none."""
        n, dev = slots.shape[0], self.device
        if k.shape[0] != v.shape[0]:
            raise ValueError(f"k has {k.shape[0]} tokens, v has {v.shape[0]}")
        call(self._lib.pg_cache_write, dev, stream, self._ref, layer,
             int32_list("slots", slots, dev), int32_list("starts", starts, dev, n + 1), n,
             k.shape[0], self._rows("k", k), self._rows("v", v))

    def free(self, slots: Any, stream: int | None = None) -> None:
        """Let go of the slots' pages: their lengths become 0."""
        call(self._lib.pg_cache_free, self.device, stream, self._ref,
             int32_list("slots", slots, self.device), slots.shape[0])

    def fork(self, parents: Any, children: Any, stream: int | None = None) -> None:
        """Make each empty slot ``children[i]`` a continuation of ``parents[i]``: it shares the
        full pages and gets a copy of a last page that is not full, in every layer."""
        n, dev = parents.shape[0], self.device
        call(self._lib.pg_cache_fork, dev, stream, self._ref,
             int32_list("parents", parents, dev), int32_list("children", children, dev, n), n)

    def copy_pages(self, source: Any, destination: Any, stream: int | None = None) -> None:
        """Copy whole pages in every layer; counts and tables stay as they are. No page may be
        both a source and a destination, nor a destination twice."""
        n, dev = source.shape[0], self.device
        call(self._lib.pg_cache_copy, dev, stream, self._ref, int32_list("source", source, dev),
             int32_list("destination", destination, dev, n), n)

    def compact(self, stream: int | None = None) -> None:
        """Move the live pages to the lowest ids, with the tables and counts."""
        call(self._lib.pg_cache_compact, self.device, stream, self._ref)

    def check(self) -> None:
        """Wait for the GPU, all its streams, and raise ``CacheError`` if an earlier call could not
        be met (the status word is cleared)."""
        bits = take_status(self.status)
        if bits:
            raise CacheError(bits)
