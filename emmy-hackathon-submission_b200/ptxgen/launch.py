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

# torch's own ways to the current device and to a device's current stream as an integer, which make no
# stream object; the public ones where a torch has no such names
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                          lambda index: torch.cuda.current_stream(index).cuda_stream)
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


def empty(shape: Any, dtype: torch.dtype, device: torch.device, stream: int | None) -> Any:
    """A new tensor for a call on ``stream``, from that stream's memory: what the current stream
    has let go of may still be read there, and what this tensor lets go of is not the current
    stream's to write while the call runs."""
    if stream is None or stream == _current_stream(device.index):
        return torch.empty(shape, dtype=dtype, device=device)
    # a null handle is the default stream, of which ExternalStream would make a new one
    of = torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device)
    with torch.cuda.stream(of):
        return torch.empty(shape, dtype=dtype, device=device)


def wait_until_set(device: torch.device) -> None:
    """Wait for the current stream, which has set what calls on any stream will read. Under capture
    nothing runs yet, and the graph's own order holds."""
    if not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(device).synchronize()


def take_status(word: Any) -> int:
    """The bits of a status word (a one-element int32 tensor), which is cleared. The calls that set
    it may have been on any stream, so this waits for the whole device, before it reads the word and
    until it is cleared."""
    torch.cuda.synchronize(word.device)
    bits = int(word.item())
    if bits:
        word.zero_()
        torch.cuda.synchronize(word.device)
    return bits


def call(fn: Callable[..., int], device: torch.device, stream: int | None, *args: Any) -> None:
    """``fn(*args, stream)`` with ``device`` current, on its current stream where ``stream`` is
    None; raises ``LaunchError`` where it fails."""
    index = device.index
    if _current_device() != index:
        with torch.cuda.device(index):
            return call(fn, device, stream, *args)
    rc = fn(*args, _current_stream(index) if stream is None else stream)
    if rc:
        _check(rc, fn.__name__)
