"""What the decoding and scoring entry points refuse, before any GPU is needed."""

from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

from ppy_b200 import decode, runtime, scoring, torch_calls  # noqa: E402

ATTENTION = ("q k_new v_new keys values lengths parents counts out lse status workspace "
             "workspace_bytes dtype batch nodes heads kv_heads head_dim capacity").split()
ACCEPT = ("q lse keys values weights positions lengths seen path accepted status dtype layers "
          "batch nodes steps heads kv_heads head_dim capacity").split()
EVICT = ("keys values weights positions weights_out positions_out kept lengths seen status "
         "workspace workspace_bytes layers batch kv_heads head_dim capacity budget "
         "recent").split()


def _packed(struct, names, strides, values, scale=()):
    return struct.pack(*(values.get(n, 0) for n in names), *strides, *scale)


def _attention(strides=None, **changes):
    values = dict(dtype=1, batch=1, nodes=1, heads=4, kv_heads=2, head_dim=64, capacity=128)
    values.update(changes)
    return _packed(decode._ATTENTION, ATTENTION, strides or (64,) * 18 + (0,), values, (0.125,))


def _accept(strides=None, **changes):
    values = dict(dtype=1, layers=1, batch=1, nodes=4, steps=2, heads=4, kv_heads=2, head_dim=64,
                  capacity=128)
    values.update(changes)
    return _packed(decode._ACCEPT, ACCEPT, strides or (64,) * 15, values, (0.125,))


def _evict(strides=None, **changes):
    values = dict(layers=1, batch=1, kv_heads=2, head_dim=64, capacity=128, budget=64)
    values.update(changes)
    return _packed(decode._EVICT, EVICT, strides or (64,) * 14, values)


@pytest.mark.parametrize("changes,why", [
    (dict(dtype=0), "bf16 or f16"), (dict(dtype=3), "bf16 or f16"),
    (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"),
    (dict(batch=-1), "negative"), (dict(nodes=-1), "negative"),
    (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(head_dim=0), "head_dim"),
    (dict(parents=64, nodes=257), "PPYB200_TREE_NODES"),
    (dict(batch=70000), "65535"), (dict(capacity=1 << 31), "2^31"),
    (dict(q=8), "16-byte"), (dict(keys=24), "16-byte"), (dict(out=2), "16-byte"),
])
def test_tree_attention_refusals(changes, why):
    lib = runtime.library()
    assert lib.ppyb200_tree_attention(_attention(**changes)) == runtime.STATUS_RAISED
    assert why in runtime.last_error()
    assert lib.ppyb200_tree_attention_workspace(_attention(**changes)) == 0


def test_tree_attention_refuses_strides_off_16_bytes_and_null():
    lib = runtime.library()
    for at in range(18):
        strides = [64] * 18 + [0]
        strides[at] = 68
        assert lib.ppyb200_tree_attention(_attention(strides)) == runtime.STATUS_RAISED
    assert lib.ppyb200_tree_attention(None) == runtime.STATUS_RAISED
    assert lib.ppyb200_tree_attention(_attention(batch=0)) == runtime.STATUS_OK  # nothing to do
    assert lib.ppyb200_tree_attention(_attention(nodes=0)) == runtime.STATUS_OK


@pytest.mark.parametrize("changes,why", [
    (dict(dtype=0), "bf16 or f16"), (dict(heads=5), "multiple of kv_heads"),
    (dict(steps=-1), "negative"), (dict(head_dim=12), "head_dim"),
    (dict(steps=65), "64 steps"), (dict(steps=64, heads=18), "512"),
    (dict(layers=300, batch=300), "65535"), (dict(keys=8), "16-byte"),
    (dict(weights=16, q=8, lse=4), "16-byte"), (dict(weights=16), "q and lse"),
])
def test_accept_refusals(changes, why):
    lib = runtime.library()
    assert lib.ppyb200_accept(_accept(**changes)) == runtime.STATUS_RAISED
    assert why in runtime.last_error()
    assert lib.ppyb200_accept(_accept(steps=0)) == runtime.STATUS_OK


@pytest.mark.parametrize("changes,why", [
    (dict(kv_heads=0), "negative"), (dict(budget=0), "budget"), (dict(budget=129), "budget"),
    (dict(recent=-1), "recent"), (dict(head_dim=20), "head_dim"), (dict(values=8), "16-byte"),
    (dict(batch=40000), "65535"), (dict(), "workspace"),
    (dict(workspace=16, workspace_bytes=16), "workspace"),
])
def test_evict_refusals(changes, why):
    lib = runtime.library()
    assert lib.ppyb200_evict(_evict(**changes)) == runtime.STATUS_RAISED
    assert why in runtime.last_error()
    assert lib.ppyb200_evict(_evict(batch=0)) == runtime.STATUS_OK
    # counts, holes and sources of 2 heads: at most 64 rows move
    assert lib.ppyb200_evict_workspace(_evict()) >= 2 * (1 + 2 * 64) * 4


@pytest.mark.parametrize("changes", [
    dict(dtype=3), dict(rows=-1), dict(vocab=0), dict(pitch=9), dict(top=65), dict(top=11),
    dict(given=-1), dict(logits=6),
])
def test_token_logprobs_refusals(changes):
    lib = runtime.library()
    v = dict(logits=64, dtype=0, rows=2, vocab=10, pitch=10, given=1, top=3)
    v.update(changes)
    assert lib.ppyb200_token_logprobs(v["logits"], v["dtype"], v["rows"], v["vocab"], v["pitch"],
                                      64, v["given"], v["top"], 64, 64, 64,
                                      64) == runtime.STATUS_RAISED
    assert "ppyb200_token_logprobs" in runtime.last_error()
    assert lib.ppyb200_token_logprobs(64, 0, 0, 10, 10, 64, 1, 3, 64, 64, 64, 64) == 0


def test_operators_refuse_host_tensors_and_wrong_types():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16)
    lengths = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(runtime.B200Error):
        decode.tree_attention(q, q[:, :, :2], q[:, :, :2], cache, cache, lengths)
    with pytest.raises(runtime.B200Error):
        decode.tree_attention(q.float(), q, q, cache, cache, lengths)
    with pytest.raises(runtime.B200Error):
        decode.evict(cache[None], cache[None], None, None, lengths, lengths, 4)
    with pytest.raises(runtime.B200Error):
        scoring.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(runtime.B200Error):
        decode.KVCache(1, 1, 2, 64, 8, dtype=torch.float32, device="cpu")
    with pytest.raises(runtime.B200Error):
        decode.KVCache(1, 1, 2, 64, 8, device="cpu").accept()
    with pytest.raises(runtime.B200Error):
        decode.KVCache(1, 1, 2, 64, 8, device="cpu", weights=False).evict(4)


def test_argument_checks_name_the_tensor():
    x = torch.zeros(2, 3, 8, dtype=torch.bfloat16)
    on = x.get_device()  # -1: host memory
    assert torch_calls.element_rows("x", x.transpose(0, 1), (3, 2, 8), torch.bfloat16, on) == (8, 24, 1)
    for bad in (x.transpose(1, 2), x.float(), x[:1]):
        with pytest.raises(runtime.B200Error, match="x:"):
            torch_calls.element_rows("x", bad, (2, 3, 8), torch.bfloat16, on)
    with pytest.raises(runtime.B200Error, match="x:"):
        torch_calls.element_rows("x", x, (2, 3, 8), torch.bfloat16, 0)
    with pytest.raises(runtime.B200Error, match="n:"):
        torch_calls.whole("n", torch.zeros(4, dtype=torch.int32)[::2], (2,), torch.int32, on)


def test_logits_rows_layout():
    rows = lambda t: scoring._rows(t.shape, t.stride())  # noqa: E731
    assert rows(torch.empty(4, 10)) == (4, 10)
    assert rows(torch.empty(2, 3, 16)[:, :, :10]) == (6, 16)
    assert rows(torch.empty(2, 3, 16)[:, 1]) == (2, 48)
    assert rows(torch.empty(2, 3, 16)[:, :2])[1] == -1  # unevenly spaced
    assert rows(torch.empty(16)) == (1, 16)
    assert rows(torch.empty(5, 1, 16)) == (5, 16)
    assert rows(torch.empty(4, 10).expand(2, 4, 10))[1] == -1


def test_structures_are_as_large_as_the_headers():
    """The packed arguments against the header's fields, 8 bytes each."""
    import re

    from conftest import REPO

    text = (REPO / "include" / "ppyb200.h").read_text()
    for name, struct in (("tree_attention", decode._ATTENTION), ("accept", decode._ACCEPT),
                         ("evict", decode._EVICT)):
        body = re.search(r"typedef struct ppyb200_%s_args \{(.*?)\}" % name, text, re.S).group(1)
        size = 0
        for line in body.split(";"):
            for field in line.strip().split(","):
                if field.strip():
                    array = re.search(r"\[(\d+)\]", field)
                    size += 8 * (int(array.group(1)) if array else 1)
        assert size == struct.size, name
    assert ctypes.sizeof(ctypes.c_void_p) == 8
