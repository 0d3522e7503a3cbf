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
