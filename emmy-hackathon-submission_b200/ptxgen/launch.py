"""Calling the C ABI's operators on PyTorch tensors: the checks of arguments that
``ptxgen.cache``, ``ptxgen.attention`` and ``ptxgen.logprob`` share, and the call itself.

Single-token calls last a few microseconds on the GPU, so the host's part counts: the stream is
asked for as a plain integer, and the device is only switched where it has to be.
"""

from __future__ import annotations

from collections.abc import Callable
from typing import Any

import torch

from .runtime import _check

_DTYPES = {torch.float16: 1, torch.bfloat16: 2, torch.float32: 3}  # PG_DT_*


def dtype_code(dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"dtype {dtype}: want float32, bfloat16 or float16")
    return code


def int32_list(name: str, t: Any, device: torch.device, n: int | None = None) -> int:
    """The address of a contiguous 1-D int32 tensor on ``device`` (with ``n`` entries)."""
    if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: want a contiguous 1-D int32 tensor on {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name}: {t.shape[0]} entries, want {n}")
    return t.data_ptr()


def call(fn: Callable[..., int], device: torch.device, stream: int | None, *args: Any) -> None:
    """``fn(*args, stream)`` with ``device`` current, on its current stream where ``stream`` is
    None; raises ``LaunchError`` where it fails."""
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return call(fn, device, stream, *args)
    rc = fn(*args, torch._C._cuda_getCurrentRawStream(index) if stream is None else stream)
    if rc:
        _check(rc, fn.__name__)
