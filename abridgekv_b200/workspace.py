"""Caller-side device workspace for libabkv entry points.

The C ABI never allocates: every call receives a workspace whose first four
bytes hold the device error word.  This helper keeps one zero-initialised,
256-byte aligned buffer per device and grows it on demand (growth happens
outside any kernel and keeps the error word; a buffer that a captured call used
stays allocated as long as the workspace, for the graph's replays).  Give a
workspace its size before a capture: one that grows inside is zeroed by the
replays only.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import threading

import torch

from . import _lib


class Workspace:
    def __init__(self, device: torch.device | int | str | None = None, nbytes: int = 1 << 20,
                 zeroed: int | None = None):
        """``zeroed``: leading bytes that start at zero (None: all)."""
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self._buf = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=self.device)
        self._buf[:zeroed].zero_()
        self._in_graph = False  # a CUDA graph holds the buffer's address
        self._kept: list[torch.Tensor] = []

    @property
    def on(self) -> torch.device:
        """The device of the buffer (``device`` may leave its index open)."""
        return self._buf.device

    @property
    def nbytes(self) -> int:
        return self._buf.numel()

    def ensure(self, nbytes: int) -> "Workspace":
        if nbytes > self._buf.numel():
            # keep the error word of the old buffer visible to the caller
            old_err = self._buf[:4].clone()
            if self._in_graph:  # its replays go on writing there: the memory is not given back
                self._kept.append(self._buf)
                self._in_graph = False
            self._buf = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
            self._buf[:4].copy_(old_err)
        return self

    def ptr(self) -> int:
        if not self._in_graph:
            self._in_graph = torch._C._cuda_isCurrentStreamCapturing()
        return self._buf.data_ptr()

    def read_error(self, stream: torch.cuda.Stream | None = None) -> int:
        """Device error word (ABKV_DEVERR_* bits); clears it.  Synchronises."""
        s = torch.cuda.current_stream(self.device) if stream is None else stream
        v = C.c_int32(0)
        _lib.check("abkv_workspace_error", _lib.lib().abkv_workspace_error(
            C.c_void_p(self.ptr()), C.c_void_p(s.cuda_stream), C.byref(v)))
        return int(v.value)


_per_device: dict[int, Workspace] = {}


def default_workspace(device: torch.device) -> Workspace:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    ws = _per_device.get(idx)
    if ws is None:
        ws = _per_device[idx] = Workspace(torch.device("cuda", idx))
    return ws


_here = contextlib.nullcontext()


def call_scope(device: torch.device, stream: torch.cuda.Stream | None):
    """The context of one call's allocations and launches: ``device`` current, and ``stream`` (when
    given) its current stream, so that what the call allocates belongs to the stream that uses it.
    No context is entered where both hold already (a context costs a few microseconds)."""
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the call's tensors are on {device}")
        return torch.cuda.stream(stream)
    return _here if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


_own = threading.local()  # .table: {(device index, raw stream): Workspace} of this thread


def stream_workspace(device: torch.device | str, stream: torch.cuda.Stream | None = None) -> Workspace:
    """The workspace that this thread's calls without one of their own use on ``stream`` (None: the current
    stream) outside a capture.  Its error word is theirs: ``stream_workspace(device, s).read_error(s)``."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    with call_scope(device, stream):
        return _stream_workspace(device, torch._C._cuda_getCurrentRawStream(device.index), 256)


def _stream_workspace(device: torch.device, raw: int, nbytes: int) -> Workspace:
    table = _own.__dict__.setdefault("table", {})
    ws = table.get((device.index, raw))
    if ws is None:
        ws = table[(device.index, raw)] = Workspace(device, nbytes)
    return ws.ensure(nbytes)


def call_workspace(device: torch.device, nbytes: int, workspace: Workspace | None = None) -> tuple[Workspace, int]:
    """(workspace, raw current stream) of one call, inside its ``call_scope``: the caller's workspace,
    else one that no other stream, no other thread and no CUDA graph uses.

    A call may be several launches with data in the workspace between them, and another thread's launches may
    come in between on the same stream, so every thread has a buffer per stream (``stream_workspace``), apart
    from ``default_workspace``, which other entries use on any stream.  A call under stream capture gets a
    fresh one from the graph's memory pool, its header zeroed at every replay (the entries that come here write
    the rest before they read it): two graphs never share it, and no later growth frees it under them.  (To read
    the error word of a captured call, pass a workspace of your own.)"""
    raw = torch._C._cuda_getCurrentRawStream(device.index)
    if workspace is not None:
        if workspace.on != device:
            raise ValueError(f"the workspace is on {workspace.on}, the call's tensors are on {device}")
        return workspace.ensure(nbytes), raw
    if torch._C._cuda_isCurrentStreamCapturing():
        return Workspace(device, nbytes, zeroed=256), raw
    return _stream_workspace(device, raw, nbytes), raw
