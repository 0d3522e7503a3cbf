"""What a KVCache keeps between calls, as far as that needs no GPU."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from ppy_b200 import decode, runtime  # noqa: E402


def _cache(**more):
    return decode.KVCache(1, 2, 2, 64, 16, device="cpu", **more)


def test_evict_refuses_while_an_extension_is_pending():
    cache = _cache()
    cache.pending = pending = (torch.zeros(1, 2, 3, 2, 64), torch.zeros(1, 2, 2, 3))
    with pytest.raises(runtime.B200Error, match="pending"):
        cache.evict(4)
    assert cache.pending is pending and cache.lengths.tolist() == [0, 0]
    cache.reset()  # forgets the extension too
    with pytest.raises(runtime.B200Error, match="CUDA device"):
        cache.evict(4)


def _part(**changes):
    values = dict(counts=0, taken_before=0, taken=0, first=0, path_steps=2, path_stride=2)
    values.update(changes)
    return decode._PART.pack(*values.values())


@pytest.mark.parametrize("part", [
    dict(first=-1), dict(first=1, taken_before=64), dict(first=64, path_steps=66),
    dict(path_steps=1), dict(path_stride=-1), dict(path_steps=1 << 31),
])
def test_pieces_of_a_path_that_are_refused(part):
    lib = runtime.library()
    args = decode._ACCEPT.pack(*(0,) * 11, 1, 1, 1, 4, 2, 4, 2, 64, 128, *(64,) * 15, 0.125)
    assert lib.ppyb200_accept_part(args, _part(**part)) == runtime.STATUS_RAISED
    assert "piece" in runtime.last_error()
    assert lib.ppyb200_accept_part(args, None) == runtime.STATUS_RAISED


def test_accept_refuses_paths_of_other_shapes():
    cache = _cache()
    cache.pending = (torch.zeros(1, 2, 3, 2, 64), torch.zeros(1, 2, 2, 3))
    with pytest.raises(runtime.B200Error, match="path"):
        cache.accept(torch.zeros(3, dtype=torch.int32))
    assert cache.pending is not None


def test_a_call_that_fails_leaves_the_current_device(monkeypatch):
    """A call with tensors of another device than the current one makes that the current one until
    it ends, also when the order of the streams cannot be set up or restored."""
    from ppy_b200 import torch_calls

    left = []

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            left.append(("enter", self.index))

        def __exit__(self, *_):
            left.append(("exit", self.index))

    class Library:
        @staticmethod
        def ppyb200_current_device():
            return -1

        @staticmethod
        def ppyb200_stream():
            return 64

    class Stream:
        cuda_stream = 128

    def refuse(*_):
        raise runtime.B200Error("no")

    monkeypatch.setattr(runtime, "library", lambda: Library)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: Stream)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(runtime, "init", refuse)
    with pytest.raises(runtime.B200Error):
        torch_calls.Beside(1)
    assert left == [("enter", 1), ("exit", 1)]
    left.clear()
    orders = iter((None, refuse))
    monkeypatch.setattr(runtime, "init", lambda index: None)
    monkeypatch.setattr(torch_calls, "_external_stream", lambda *_: Stream)
    monkeypatch.setattr(torch_calls, "_order", lambda *_: (next(orders) or (lambda: None))())
    beside = torch_calls.Beside(1)
    with pytest.raises(runtime.B200Error):
        beside.end()
    assert left == [("enter", 1), ("exit", 1)]
