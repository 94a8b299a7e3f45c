"""Device workspaces that calls on torch tensors keep for the next: one a thread and stream.

Work on one stream runs in order, and a thread enqueues one call's kernels before the next one's, so calls that share a
workspace here do not overlap. A call that is captured into a graph gets one of its own from the graph's memory (None
here), as its replays may run beside anything. So does a call on a stream that is not torch's: such a stream's address may be
another's later, while the last kernels of the first still run."""

from __future__ import annotations

import threading
import weakref

from .attention import torch

# (torch.cuda's functions of these names, without their checks that the device was used before: a tensor of it is there)
_capturing = getattr(getattr(torch, "_C", None), "_cuda_isCurrentStreamCapturing", None)
_current = getattr(getattr(torch, "_C", None), "_cuda_getDevice", None)

_KEEP = 64 << 20   # larger ones live as long as their call
_LEAST = 1 << 20
_STREAMS = 8       # a thread keeps workspaces for so many, the newest


class _Streams(dict):
    __slots__ = ("__weakref__",)
    __eq__, __hash__ = object.__eq__, object.__hash__


_threads = weakref.WeakSet()  # every living thread's
_threads_lock = threading.Lock()


class _Kept(threading.local):
    def __init__(self):
        self.by_stream = _Streams()
        with _threads_lock:
            _threads.add(self.by_stream)


_kept = _Kept()


def _shared(device: int) -> bool:
    """Whether a call may use a kept workspace: its stream, the device's current one, is not being captured."""
    if _capturing is None or _current is None:
        return not torch.cuda.is_current_stream_capturing() and torch.cuda.current_device() == device
    return not _capturing() and _current() == device


def _lasting(device: int) -> bool:
    """Whether the device's current stream is the default one or of torch's pool, which are never destroyed. (The id of a stream
    from elsewhere, torch.cuda.ExternalStream, is its address.)"""
    s = torch.cuda.current_stream(device)
    return s.cuda_stream == 0 or s.stream_id != s.cuda_stream


def kept_workspace(device: int, stream: int):
    """The thread's workspace for the stream as (address, bytes, tensor); None if there is none yet, or a call must not use it."""
    return _kept.by_stream.get((device, stream)) if _shared(device) else None


def new_workspace(like, device: int, stream: int, nbytes: int):
    """A workspace of at least ``nbytes`` for a call on ``stream``, the current one: (address, bytes, the tensor to hold until
    the call was made). It is kept for the thread's next calls unless it is large, the call is being captured or the stream may be
    destroyed."""
    if nbytes > _KEEP or not _shared(device) or not _lasting(device):
        ws = like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        return (ws.data_ptr() if ws is not None else None), nbytes, ws
    n = max(_LEAST, 1 << (nbytes - 1).bit_length()) if nbytes else _LEAST
    ws = like.new_empty(n, dtype=torch.uint8)
    mine = _kept.by_stream
    mine.pop((device, stream), None)
    while len(mine) >= _STREAMS:  # (its memory goes to its stream's next allocations, which run behind the calls that used it)
        try:
            mine.pop(next(iter(mine)), None)
        except (StopIteration, RuntimeError):  # another thread released them
            break
    mine[(device, stream)] = k = (ws.data_ptr(), n, ws)
    return k


def release_workspaces() -> None:
    """Gives back to torch's allocator what all threads keep for their next calls (up to 64 MiB a thread and stream, for at most
    eight streams a thread); those allocate again. Calls under way are not disturbed."""
    with _threads_lock:
        every = list(_threads)
    for s in every:
        s.clear()
