"""Per-(device, stream) scratch buffers handed to the C-ABI as workspaces.

The kernels keep a status word and atomic tickets in their workspace and leave
both zero when they finish, so a buffer is zero-filled once, when it is first
allocated or grown, and then reused by every later call on the same stream.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_cache: dict[tuple[str, int, int], torch.Tensor] = {}


def get(kind: str, nbytes: int, device: torch.device) -> torch.Tensor:
    stream = torch.cuda.current_stream(device).cuda_stream
    key = (kind, device.index if device.index is not None else torch.cuda.current_device(), stream)
    buf = _cache.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 4096), dtype=torch.uint8, device=device)
        _cache[key] = buf
    return buf


# The raw handle of a device's current stream, without building a Stream object around it (2 us of a 5 us launch).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream(index: int) -> int:
    """Handle of the current stream of device ``index``."""
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _capturing(index: int) -> bool:
    """Whether the current stream of device ``index``, which need not be the current device, is being captured."""
    if torch.cuda.current_device() == index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def scratch(kind: str, nbytes: int, head: int, device: torch.device, handle: int) -> torch.Tensor:
    """Like :func:`get` for kernels of which only the first ``head`` bytes must be zero, and safe under graph capture.

    ``device`` has an index, ``handle`` is its current stream (:func:`stream`).  A call that is being captured gets a buffer
    of the graph's own, whose head is cleared by a node of the graph: two graphs, or a graph and eager calls, never share
    one, however their replays overlap."""
    if _capturing(device.index):
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        buf[:head].zero_()
        return buf
    buf = _cache.get((kind, device.index, handle))
    return buf if buf is not None and buf.numel() >= nbytes else get(kind, nbytes, device)


def all_of(kind: str, device: torch.device) -> list[torch.Tensor]:
    """Every cached workspace of one kind on a device (one per stream that has launched with it)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    return [buf for (k, d, _), buf in _cache.items() if k == kind and d == index]


def status(buf: torch.Tensor) -> int:
    """Read (and synchronise on) the device status word of a workspace."""
    out = C.c_int(0)
    dev = buf.device.index
    st = torch.cuda.current_stream(buf.device).cuda_stream
    _lib.check(_lib.load().skv_workspace_status(buf.data_ptr(), dev, st, C.byref(out)), "skv_workspace_status")
    return out.value


def clear() -> None:
    _cache.clear()
