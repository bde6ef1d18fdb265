"""Drawing the next token of each row of logits by a given random number.

    r = sample(logits, uniform, temperature=0.8, top_k=50, top_p=0.95, min_p=0.02)
    r.tokens, r.logp

For a row x of ``logits`` [rows, vocab] (f32, bf16 or f16; rows may lie apart), m = max x and w =
exp((x - m) / temperature), the kept tokens are a prefix of the tokens ordered by logit, the largest
first and ties by the lowest column: the shortest of the first ``top_k`` (0: all), the fewest whose
weights reach ``top_p`` of the sum of the top_k ones' (1: all), and those with w >= ``min_p``; one at
least. The token drawn is the lowest kept column up to which the kept weights add up to more than
``uniform`` (f32 [rows], from 0 to below 1) of their sum, and ``logp`` the log of its share of it, in
the distribution that it was drawn from. Temperature 0 takes the first of the largest logits.

Each setting is a number for all rows or a device tensor of one a row (float32; ``top_k`` int32).
Weights and sums are held in 64 bits, so the token does not hang on the order of a sum. A column of
-inf is never drawn. A row with a NaN, a +inf or nothing but -inf gives token -1 and a logp of NaN, as
does one whose own settings are NaN, its temperature negative or its min_p above 1; a row's top_k below
1 or top_p of 1 and more keeps all.

The kernel is ``csrc/sample.cu`` (``pg_sample``); calls run on the current stream, or on ``stream`` (a
``cudaStream_t`` as an integer), whose memory new results then come from: other streams wait for
them and call ``record_stream``, as for any tensor of another stream.
"""

from __future__ import annotations

import ctypes
import struct
from typing import Any

import torch

from .launch import call, dtype_code, empty
from .runtime import SampleArgs, library

_PACK = struct.Struct("=8Qq4i3fi")
assert _PACK.size == ctypes.sizeof(SampleArgs)


class Samples:
    """What ``sample`` returns; its tensors are parts of one allocation, made when asked for."""

    __slots__ = ("_all", "_rows")

    def __init__(self, device: torch.device, rows: int, stream: int | None = None):
        self._all = empty((rows + (rows + 1) // 2,), torch.int64, device, stream)
        self._rows = rows

    @property
    def tokens(self) -> Any:
        """[rows] int64: the columns drawn."""
        return self._all.narrow(0, 0, self._rows)

    @property
    def logp(self) -> Any:
        """[rows] f32: the log of their probabilities among the kept tokens."""
        return self._all.narrow(0, self._rows, (self._rows + 1) // 2).view(
            torch.float32).narrow(0, 0, self._rows)


def _per_row(name: str, t: Any, dtype: torch.dtype, logits: Any) -> int:
    if t.dtype is not dtype or t.shape != logits.shape[:1] or not t.is_contiguous() or \
            t.device != logits.device:
        raise ValueError(f"{name}: want contiguous {dtype} [{logits.shape[0]}] on "
                         f"{logits.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def sample(logits: Any, uniform: Any, *, temperature: Any = 1.0, top_k: Any = 0, top_p: Any = 1.0,
           min_p: Any = 0.0, stream: int | None = None) -> Samples:
    """One token of each row of ``logits`` [rows, vocab], by ``uniform`` [rows]."""
    if logits.dim() != 2 or not logits.is_cuda or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits: want [rows, vocab] on a CUDA device with contiguous rows, got "
                         f"{tuple(logits.shape)} {logits.stride()} on {logits.device}")
    rows, vocab = logits.shape
    at, all_ = [0, 0, 0, 0], [temperature, top_k, top_p, min_p]
    for i, name in enumerate(("temperature", "top_k", "top_p", "min_p")):
        if isinstance(all_[i], torch.Tensor):
            at[i] = _per_row(name, all_[i], torch.int32 if i == 1 else torch.float32, logits)
            # an empty tensor has no address
            all_[i], at[i] = (1, 0, 1, 0)[i], at[i] if rows else 0
    u = _per_row("uniform", uniform, torch.float32, logits)
    r = Samples(logits.device, rows, stream)
    to = r._all.data_ptr()
    args = SampleArgs()
    try:
        _PACK.pack_into(args, 0, logits.data_ptr(), u, *at, to, to + 8 * rows, logits.stride(0),
                        dtype_code(logits.dtype), rows, vocab, all_[1], all_[0], all_[2], all_[3],
                        0)
    except (struct.error, OverflowError, TypeError) as e:
        raise ValueError(f"temperature {temperature}, top_k {top_k}, top_p {top_p} or min_p "
                         f"{min_p} is out of range: {e}") from e
    call(library().pg_sample, logits.device, stream, args)
    return r
