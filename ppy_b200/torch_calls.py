"""Calls with torch tensors: where they launch, and checks of what they are given.

The library launches on the thread's stream (`runtime.set_stream`); torch allocates and orders by its
own current stream. A function that takes torch tensors brackets its launches with `begin` and
`end`: where both streams are the same one, the usual case, they cost next to nothing.
"""

from __future__ import annotations

import functools
import threading

import torch

from . import runtime
from .runtime import B200Error

__all__ = ["Beside", "begin", "element_rows", "end", "whole"]

# torch.cuda.current_device and current_stream(...).cuda_stream without the Python around them,
# which costs as much as a launch
_current_device = torch._C._cuda_getDevice
_current_raw_stream = torch._C._cuda_getCurrentRawStream
_external_stream = functools.lru_cache(maxsize=256)(torch.cuda.ExternalStream)


class _Thread(threading.local):
    def __init__(self) -> None:
        self.events = {}  # an event of each device


_thread = _Thread()


def _order(index: int, before, after) -> None:
    """What comes on `after` waits for what `before` holds by now. One event a thread and device:
    a wait keeps to the record before it, so the next record may follow at once."""
    event = _thread.events.get(index)
    if event is None:
        event = _thread.events[index] = torch.cuda.Event()
    event.record(before)
    after.wait_event(event)


class Beside:
    """A call whose launches go to another stream than torch's current one, or to another device
    than the current one. `side` is the stream when it is another. Tensors made within the call
    belong to torch's current stream, which is behind the launches from `end` on, so they need no
    record on the side stream."""

    __slots__ = ("_guard", "_index", "side")

    def __init__(self, index: int) -> None:
        lib = runtime.library()
        bound = lib.ppyb200_current_device()
        if bound != index and bound >= 0:
            raise B200Error(f"tensors on cuda:{index}, but this thread's device is {bound} "
                            "(runtime.init)")
        self._index, self._guard, self.side = index, None, None
        if torch.cuda.current_device() != index:
            self._guard = torch.cuda.device(index)
            self._guard.__enter__()
        try:
            if bound < 0:
                runtime.init(index)
            handle = lib.ppyb200_stream() or 0
            current = torch.cuda.current_stream(index)
            if handle != (current.cuda_stream or runtime._LEGACY_STREAM):
                self.side = (torch.cuda.default_stream(index) if handle == runtime._LEGACY_STREAM
                             else _external_stream(handle, index))
                _order(index, current, self.side)
        except BaseException:
            self._leave()
            raise

    def wait_for_torch(self) -> None:
        """The launches that follow wait for what torch's stream holds by now."""
        if self.side is not None:
            _order(self._index, torch.cuda.current_stream(self._index), self.side)

    def end(self) -> None:
        try:
            if self.side is not None:
                _order(self._index, self.side, torch.cuda.current_stream(self._index))
        finally:
            self._leave()

    def _leave(self) -> None:
        if self._guard is not None:
            self._guard.__exit__(None, None, None)


def begin(index: int) -> Beside | None:
    """Before launches with tensors of device `index`: the thread's device has to be theirs (a thread
    without one is bound to it). None when it is the current device and torch's current stream is
    the thread's; else the launches are ordered behind the work on torch's stream so far, and `end`
    orders torch's stream behind them, so that the tensors are the caller's to use as if the call had
    run on torch's stream."""
    lib = runtime.library()
    if (lib.ppyb200_current_device() == index and _current_device() == index
            and (lib.ppyb200_stream() or 0) == (_current_raw_stream(index)
                                                or runtime._LEGACY_STREAM)):
        return None
    return Beside(index)


def end(beside: Beside | None) -> None:
    if beside is not None:
        beside.end()


def element_rows(name: str, t, shape, dtype, device: int):
    """The strides of a tensor of `shape` and `dtype` on CUDA device `device` with unit stride along
    its last axis."""
    strides = t.stride()
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device or (
            strides[-1] != 1 and shape[-1] > 1):
        raise B200Error(f"{name}: {dtype} {list(shape)} on cuda:{device}, unit stride along the last "
                        f"axis (not {t.dtype} {list(t.shape)} on {t.device}, strides "
                        f"{list(strides)})")
    return strides


def whole(name: str, t, shape, dtype, device: int) -> int:
    """The address of a contiguous tensor of `shape` and `dtype` on CUDA device `device`."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device or (
            not t.is_contiguous()):
        raise B200Error(f"{name}: contiguous {dtype} {list(shape)} on cuda:{device} (not {t.dtype} "
                        f"{list(t.shape)} on {t.device}, strides {list(t.stride())})")
    return t.data_ptr()
