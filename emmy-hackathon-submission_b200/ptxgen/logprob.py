"""Log probabilities of given tokens, with the distribution's entropy and its top alternatives.

    r = logprobs(logits, tokens, top=5)          # r.logp, r.entropy, r.top_logp, r.top_ids
    d_logits = logprobs_grad(logits, tokens, r, d_logp, d_entropy)

For a row x of ``logits`` [rows, vocab] (f32, bf16 or f16; rows may lie apart) and p =
softmax(x): ``logp`` = log p[token], ``entropy`` = -sum p log p, ``norm`` = (max x, log sum
exp(x - max x)), and the ``top`` largest log probabilities with their columns, ties to the lowest
column. All are f32 from 32-bit sums. Token -1 means there is none: its ``logp`` is 0 and has no gradient. A token outside
[-1, vocab) gives NaN, as does a row with a NaN, a +inf or nothing but -inf; a column of -inf has
probability 0. ``logprobs_grad`` is the gradient of ``logp`` and ``entropy`` with respect to the
logits, in their type; either incoming gradient may be None.

The kernels are ``csrc/logprob.cu`` (``pg_logprobs``, ``pg_logprobs_grad``); calls run on the
current stream, or on ``stream`` (a ``cudaStream_t`` as an integer), whose memory new results then
come from: other streams wait for them and call ``record_stream``, as for any tensor of another
stream.
"""

from __future__ import annotations

from typing import Any

import torch

from .launch import call, dtype_code, empty
from .runtime import library

TOP_MAX = 32  # PG_LOGPROB_TOP


class LogProbs:
    """What ``logprobs`` returns. Its tensors are parts of one allocation, made when asked for: five
    allocations would take the host longer than a short call takes the GPU."""

    __slots__ = ("_all", "_rows", "_top")

    def __init__(self, device: torch.device, rows: int, top: int, stream: int | None = None):
        # norm, logp, entropy, top_logp, top_ids
        self._all = empty((4 + 2 * top) * rows, torch.float32, device, stream)
        self._rows, self._top = rows, top

    @property
    def logp(self) -> Any:
        """[rows] f32: log p[token]."""
        return self._all.narrow(0, 2 * self._rows, self._rows)

    @property
    def entropy(self) -> Any:
        """[rows] f32."""
        return self._all.narrow(0, 3 * self._rows, self._rows)

    @property
    def norm(self) -> Any:
        """[rows, 2] f32: the largest logit m, and log sum exp(x - m)."""
        return self._all.as_strided((self._rows, 2), (2, 1))

    @property
    def top_logp(self) -> Any:
        """[rows, top] f32, largest first."""
        return self._all.as_strided((self._rows, self._top), (self._top, 1), 4 * self._rows)

    @property
    def top_ids(self) -> Any:
        """[rows, top] int32: their columns."""
        return self._all.as_strided((self._rows, self._top), (self._top, 1),
                                    (4 + self._top) * self._rows).view(torch.int32)


def _inputs(logits: Any, tokens: Any) -> tuple[int, int, int, int, int, int, int]:
    if logits.dim() != 2 or not logits.is_cuda or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits: want [rows, vocab] on a CUDA device with contiguous rows, got "
                         f"{tuple(logits.shape)} {logits.stride()} on {logits.device}")
    rows, vocab = logits.shape
    if tokens.dtype not in (torch.int64, torch.int32) or tokens.shape != logits.shape[:1] or \
            not tokens.is_contiguous() or tokens.device != logits.device:
        raise ValueError(f"tokens: want contiguous int64 or int32 [{rows}] on {logits.device}, "
                         f"got {tokens.dtype} {tuple(tokens.shape)} on {tokens.device}")
    return (logits.data_ptr(), logits.stride(0), dtype_code(logits.dtype), tokens.data_ptr(),
            tokens.element_size(), rows, vocab)


def _per_row(name: str, t: Any, logits: Any) -> int:
    if t is None:
        return 0
    if t.dtype is not torch.float32 or t.shape != logits.shape[:1] or not t.is_contiguous() or \
            t.device != logits.device:
        raise ValueError(f"{name}: want contiguous float32 [{logits.shape[0]}] on "
                         f"{logits.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def logprobs(logits: Any, tokens: Any, top: int = 0, stream: int | None = None) -> LogProbs:
    """``LogProbs`` of ``tokens`` [rows] under ``logits`` [rows, vocab], with the ``top`` (at
    most 32) largest log probabilities of each row."""
    args = _inputs(logits, tokens)
    rows, vocab = logits.shape
    if not 0 <= top <= min(TOP_MAX, vocab):
        raise ValueError(f"top {top}: want 0 to {min(TOP_MAX, vocab)}")
    result = LogProbs(logits.device, rows, top, stream)
    at = result._all.data_ptr()
    call(library().pg_logprobs, logits.device, stream, *args, top, at + 8 * rows, at + 12 * rows,
         at, at + 16 * rows, at + (16 + 4 * top) * rows)
    return result


def logprobs_grad(logits: Any, tokens: Any, result: LogProbs, d_logp: Any, d_entropy: Any = None,
                  out: Any = None, stream: int | None = None) -> Any:
    """The gradient of sum(d_logp * logp + d_entropy * entropy) with respect to ``logits``, given
    ``result`` = ``logprobs(logits, tokens)``; into ``out`` (which may be ``logits``) if given."""
    args = _inputs(logits, tokens)
    if out is None:
        out = empty(logits.shape, logits.dtype, logits.device, stream)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device \
            or (out.shape[1] > 1 and out.stride(1) != 1):
        raise ValueError(f"out: want {logits.dtype} {tuple(logits.shape)} on {logits.device} "
                         "with contiguous rows")
    rows, of = logits.shape[0], result._all
    if result._rows != rows or of.device != logits.device:
        raise ValueError(f"result: of {result._rows} rows on {of.device}, logits have {rows} on "
                         f"{logits.device}")
    at = of.data_ptr()
    call(library().pg_logprobs_grad, logits.device, stream, *args, at, at + 12 * rows,
         _per_row("d_logp", d_logp, logits), _per_row("d_entropy", d_entropy, logits),
         out.data_ptr(), out.stride(0))
    return out
