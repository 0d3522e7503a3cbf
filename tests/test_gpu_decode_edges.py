"""The decoding operators where their sizes, masks and orders of calls are odd. Inputs, plain forms and
tolerances are those of test_gpu_decode.py unless a test says otherwise."""

from __future__ import annotations

import math

import pytest

from test_gpu_decode import BF16, F16, Inputs, bound  # noqa: F401 - the fixture

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# ---------------------------------------------------------------- workspaces


@pytest.mark.parametrize("lengths,nodes,heads,kv,d,cap,tree", [
    ((5,), 1, 1, 1, 8, 64, False),
    ((100,), 3, 2, 1, 8, 192, True),
    ((180,), 8, 2, 1, 32, 192, True),
    ((0, 40), 1, 1, 1, 16, 64, False),
    ((20,), 4, 3, 3, 24, 64, True),
    ((60,), 20, 8, 1, 64, 128, True),    # 160 rows of one key head: the tensor-core kernel, one CTA
    ((0,), 70, 2, 1, 128, 100, False),
    ((0,), 1, 1, 1, 64, 1, False),
])
def test_small_caches_keep_to_their_workspace(lengths, nodes, heads, kv, d, cap, tree):
    """Caches so small that one CTA does the call, which takes no workspace then: what lies
    behind the bytes that the library asks for stays as it was."""
    from ppy_b200 import decode, runtime

    x = Inputs(lengths, nodes, heads, kv, d, tree=tree, spare=cap - max(lengths) - nodes)
    x.check(*x.call())
    for b, n in enumerate(lengths):
        x.keys[b, :, n:] = math.nan
        x.values[b, :, n:] = math.nan
    out, lse = torch.empty_like(x.q, memory_format=torch.contiguous_format), torch.empty(
        len(lengths), heads, nodes, device="cuda")
    strides = [s for t in (x.q, x.k_new, x.v_new, x.keys, x.values, out) for s in t.stride()[:3]]
    sizes = (1, len(lengths), nodes, heads, kv, d, cap)
    lib = runtime.library()
    size = lib.ppyb200_tree_attention_workspace(decode._ATTENTION.pack(
        *(0,) * 13, *sizes, *strides, nodes if tree else 0, 1.0))
    guarded = torch.full(((size + 15) // 16 * 16 + (1 << 20),), 77, dtype=torch.uint8,
                         device="cuda")
    status = lib.ppyb200_tree_attention(decode._ATTENTION.pack(
        x.q.data_ptr(), x.k_new.data_ptr(), x.v_new.data_ptr(), x.keys.data_ptr(),
        x.values.data_ptr(), x.lengths.data_ptr(), x.parents.data_ptr() if tree else 0, 0,
        out.data_ptr(), lse.data_ptr(), 0, guarded.data_ptr(), size, *sizes, *strides,
        nodes if tree else 0, d ** -0.5))
    assert status == runtime.STATUS_OK, runtime.last_error()
    x.check(out, lse)
    assert bool((guarded[size:] == 77).all())


# ---------------------------------------------------------------- the order of calls


def _model_and_cache(batch, capacity, layers=1, seed=5):
    from ppy_b200 import gpt2

    model = gpt2.GPT2(gpt2.Config(layers=layers), seed=seed)
    return model, model.new_cache(batch, capacity=capacity)


def _ids(batch, length, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, 50257, (batch, length), device="cuda", generator=g)


def test_evict_waits_for_the_pending_extension():
    """A cache cut between an extension and its acceptance would take other rows for the nodes'."""
    from ppy_b200.runtime import B200Error

    model, cache = _model_and_cache(2, 64)
    model.extend(cache, _ids(2, 30))
    cache.accept()
    model.extend(cache, _ids(2, 3, seed=1))
    nodes = cache.keys[:, :, :, 30:33].clone()
    with pytest.raises(B200Error, match="pending"):
        cache.evict(16)
    assert cache.lengths.tolist() == [30, 30]
    cache.accept(accepted=torch.tensor([2, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.keys[:, 0, :, 30:32], nodes[:, 0, :, :2])
    cache.evict(16)
    cache.check()
    assert cache.lengths.tolist() == [16, 16] and cache.seen.tolist() == [32, 30]
