"""Decoding with a cache: attention of drafted trees, acceptance, eviction.

    cache = KVCache(layers, batch, heads, head_dim, capacity)
    out, lse = tree_attention(q, k, v, cache.keys[i], cache.values[i], cache.lengths, parents)
    cache.accept(path, accepted)        # the verified path of the last attention joins the cache
    cache.evict(budget, recent=64)      # entries of least accumulated attention weight give way

`tree_attention`, `accept_nodes` and `evict` are the operators, on torch CUDA tensors (storage
only: the work is this package's kernels, through ppyb200_tree_attention, ppyb200_accept and
ppyb200_evict); `KVCache` holds the state that belongs together. A single token is a tree of one
node, and a piece of a prompt is a chain (`parents=None`).

Calls are asynchronous on the thread's stream (`runtime.set_stream`), ordered with torch's current
stream (`torch_calls.begin`), and read sequence lengths on the device, so that they can
be captured into a CUDA graph and replayed as the cache grows. Each call's workspace is a torch
allocation of its own: calls on several streams and captured graphs share none.
"""

from __future__ import annotations

import functools
import math
import struct
from typing import NamedTuple

import torch

from . import runtime
from .runtime import B200Error
from .torch_calls import begin, element_rows, end, whole

__all__ = ["Extension", "KVCache", "accept_nodes", "evict", "tree_attention"]

#: The header's limits (include/ppyb200.h).
TREE_NODES, PATH_STEPS, PATH_ROWS = 256, 64, 512

_ATTENTION = struct.Struct("=39qd")  # ppyb200_tree_attention_args
_ACCEPT = struct.Struct("=35qd")  # ppyb200_accept_args
_PART = struct.Struct("=6q")  # ppyb200_accept_part_args
_EVICT = struct.Struct("=33q")  # ppyb200_evict_args


#: Element types, as the header numbers them.
_KINDS = {torch.bfloat16: 1, torch.float16: 2}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise B200Error(what)


def _address(t) -> int:
    return 0 if t is None else t.data_ptr()


@functools.lru_cache(maxsize=4096)
def _attention_workspace(device, dtype, batch, nodes, heads, kv_heads, head_dim,
                         capacity) -> int:
    return runtime.library().ppyb200_tree_attention_workspace(_ATTENTION.pack(
        *(0,) * 13, dtype, batch, nodes, heads, kv_heads, head_dim, capacity, *(0,) * 19, 1.0))


def tree_attention(q, k_new, v_new, keys, values, lengths, parents=None, counts=None, scale=None,
                   out=None, lse=None, status=None):
    """Attend from drafted nodes to their sequences' caches and to their own ancestors, and append
    the nodes to the caches. Returns (out, lse).

    q [batch, nodes, heads, head_dim], k_new and v_new [batch, nodes, kv_heads, head_dim]; keys and
    values [batch, kv_heads, capacity, head_dim], any strides (a view of a token-major cache, one
    layer of a KVCache); lengths int32 [batch], the entries of each cache; parents int32 [batch,
    nodes] or [nodes]: parents[b, i] < i is node i's parent, -1 hangs it off the last entry; None
    makes the nodes a chain. counts int32 [batch] gives each sequence's real nodes (all without
    it). Scores are scale * q . k (1 / sqrt(head_dim) by default).

    out [batch, nodes, heads, head_dim] of q's type and lse f32 [batch, heads, nodes], the natural
    log of the sum of e^score of each row (made here unless given; behind a sequence's nodes they
    are left as they were, zeros when made here, and zeros for nodes that do not fit in the cache). Node i is written to slot lengths[b] + i of keys
    and values; `lengths` stay as they are (`accept_nodes` says which nodes join).

    bf16 or f16; head_dim a multiple of 8 up to 128; rows on 16-byte boundaries; up to 256 nodes
    with parents. `status` (int32 [1], optional) is raised to 2 when a length, count or parent is out of
    range: the call then keeps to the buffers, and takes such a parent for -1. It is raised, too,
    when a wait inside the kernel was given up: rows without a result are NaN then."""
    dtype, device = q.dtype, q.get_device()
    kind = _KINDS.get(dtype)
    if kind is None or device < 0 or q.dim() != 4 or keys.dim() != 4:
        raise B200Error("q: bf16 or f16 [batch, nodes, heads, head_dim], keys [batch, kv_heads, "
                        "capacity, head_dim], on a CUDA device")
    batch, nodes, heads, d = shape = q.shape
    cache = keys.shape
    kv_heads, capacity = cache[1], cache[2]
    new, entries = (batch, nodes, kv_heads, d), (batch, kv_heads, capacity, d)
    q_strides = element_rows("q", q, shape, dtype, device)
    k_strides = element_rows("k_new", k_new, new, dtype, device)
    v_strides = element_rows("v_new", v_new, new, dtype, device)
    keys_strides = element_rows("keys", keys, entries, dtype, device)
    values_strides = element_rows("values", values, entries, dtype, device)
    lengths_at = whole("lengths", lengths, (batch,), torch.int32, device)
    parents_stride = parents_at = counts_at = status_at = workspace_at = 0
    if parents is not None:
        shared = parents.dim() == 1
        parents_at = whole("parents", parents, (nodes,) if shared else (batch, nodes),
                           torch.int32, device)
        parents_stride = 0 if shared else nodes
    if counts is not None:
        counts_at = whole("counts", counts, (batch,), torch.int32, device)
    if status is not None:
        status_at = whole("status", status, (1,), torch.int32, device)
    beside = begin(device)
    try:
        if out is None or lse is None:
            make = torch.empty if counts is None else torch.zeros
            if out is None:
                out = make(shape, dtype=dtype, device=q.device)
            if lse is None:
                lse = make((batch, heads, nodes), dtype=torch.float32, device=q.device)
            if beside is not None:  # zeros were written on torch's stream
                beside.wait_for_torch()
        out_strides = element_rows("out", out, shape, dtype, device)
        lse_at = whole("lse", lse, (batch, heads, nodes), torch.float32, device)
        size = _attention_workspace(device, kind, batch, nodes, heads, kv_heads, d, capacity)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
            workspace_at = workspace.data_ptr()
        if runtime.library().ppyb200_tree_attention(_ATTENTION.pack(
                q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), keys.data_ptr(),
                values.data_ptr(), lengths_at, parents_at, counts_at, out.data_ptr(), lse_at,
                status_at, workspace_at, size, kind, batch, nodes, heads, kv_heads, d, capacity,
                *q_strides[:3], *k_strides[:3], *v_strides[:3], *keys_strides[:3],
                *values_strides[:3], *out_strides[:3], parents_stride,
                1.0 / math.sqrt(d) if scale is None else scale)) != runtime.STATUS_OK:
            raise B200Error(runtime.last_error())
    finally:
        end(beside)
    return out, lse


def accept_nodes(q, lse, keys, values, weights, positions, lengths, seen, path, accepted,
                 scale=None, status=None, taken=None, counts=None) -> None:
    """The verified path of the last attention joins the caches of every layer, in place.

    q [layers, batch, nodes, heads, head_dim] and lse f32 [layers, batch, heads, nodes] are that
    attention's; keys and values [layers, batch, kv_heads, capacity, head_dim] hold its nodes
    behind `lengths` (int32 [batch]). path int32 [batch, steps]: the accepted nodes in ascending
    order, the first accepted[b] (int32 [batch]) of row b; up to 64 steps, steps times query heads
    a key head up to 512 (`KVCache.accept` takes longer ones in pieces).

    weights f32 [layers, batch, kv_heads, capacity] (None: not kept) grow by the attention that
    the path's rows paid to each entry, summed over the query heads of the key head; the path's
    keys and values move to slots lengths[b], lengths[b] + 1, ..., their weights start with what
    the path paid them, and positions (int32, laid out as weights; None: not kept) get seen[b],
    seen[b] + 1, ... (`seen` int32 [batch]: the tokens before them). lengths and seen are the
    caller's to advance, by `taken` (int32 [batch], optional), which gets the steps that were taken:
    a path is cut before a step that is out of order, behind the capacity, or no node of the
    sequence (`counts`, int32 [batch], as the attention had them). `status` as in tree_attention:
    raised when a path was cut, or a length or count is out of range."""
    _need(path.dim() == 2, "path: int32 [batch, steps]")
    _accept(q, lse, keys, values, weights, positions, lengths, seen, path, accepted, scale, status,
            taken, counts)


def _accept(q, lse, keys, values, weights, positions, lengths, seen, path, accepted, scale, status,
            taken, counts, first=0, steps=None, before=None) -> None:
    """`accept_nodes` for `steps` steps from step `first` on, all without them; path as there, or
    [steps] for every sequence. `before` is what the piece of the path before this one left in
    `taken`."""
    kind, device = _KINDS.get(keys.dtype), keys.get_device()
    _need(kind is not None and device >= 0 and keys.dim() == 5 and q.dim() == 5,
          "keys: bf16 or f16 [layers, batch, kv_heads, capacity, head_dim], q [layers, batch, "
          "nodes, heads, head_dim], on a CUDA device")
    layers, batch, kv_heads, capacity, d = keys.shape
    nodes, heads = q.shape[2], q.shape[3]
    length = path.shape[-1]
    steps = length if steps is None else steps
    q_strides = element_rows("q", q, (layers, batch, nodes, heads, d), keys.dtype, device)
    keys_strides = element_rows("keys", keys, keys.shape, keys.dtype, device)
    values_strides = element_rows("values", values, keys.shape, keys.dtype, device)
    if weights is not None:
        whole("lse", lse, (layers, batch, heads, nodes), torch.float32, device)
    for name, t in (("lengths", lengths), ("seen", seen), ("accepted", accepted)):
        whole(name, t, (batch,), torch.int32, device)
    whole("path", path, (batch, length) if path.dim() == 2 else (length,), torch.int32, device)
    before_at = taken_at = counts_at = 0
    if taken is not None:
        taken_at = whole("taken", taken, (batch,), torch.int32, device)
    if before is not None:
        before_at = whole("taken", before, (batch,), torch.int32, device)
    if counts is not None:
        counts_at = whole("counts", counts, (batch,), torch.int32, device)
    tables = weights if weights is not None else positions
    strides = (0, 0, 0)
    for name, t, kept in (("weights", weights, torch.float32),
                          ("positions", positions, torch.int32)):
        if t is not None:
            element_rows(name, t, (layers, batch, kv_heads, capacity), kept, device)
            _need(t.stride() == tables.stride(), "weights and positions are laid out alike")
            strides = t.stride()[:3]
    if status is not None:
        whole("status", status, (1,), torch.int32, device)
    if taken is not None and (layers == 0 or steps == 0):
        taken.zero_()
    beside = begin(device)
    try:
        if runtime.library().ppyb200_accept_part(_ACCEPT.pack(
                q.data_ptr(), lse.data_ptr(), keys.data_ptr(), values.data_ptr(),
                _address(weights), _address(positions), lengths.data_ptr(), seen.data_ptr(),
                path.data_ptr(), accepted.data_ptr(), _address(status), kind, layers, batch, nodes,
                steps, heads, kv_heads, d, capacity, *q_strides[:4], *keys_strides[:4],
                *values_strides[:4], *strides,
                1.0 / math.sqrt(d) if scale is None else scale), _PART.pack(
                    counts_at, before_at, taken_at, first, length,
                    length if path.dim() == 2 else 0)) != runtime.STATUS_OK:
            raise B200Error(runtime.last_error())
    finally:
        end(beside)


@functools.lru_cache(maxsize=4096)
def _evict_workspace(layers, batch, kv_heads, head_dim, capacity, budget) -> int:
    return runtime.library().ppyb200_evict_workspace(_EVICT.pack(
        *(0,) * 12, layers, batch, kv_heads, head_dim, capacity, budget, *(0,) * 15))


def evict(keys, values, weights, positions, lengths, seen, budget, recent=0, weights_out=None,
          positions_out=None, status=None):
    """Cut every key head's cache to `budget` entries, keys and values in place. Returns `kept`,
    int32 [layers, batch, kv_heads, budget]: the slot that each entry came from, -1 behind a
    sequence's entries.

    keys and values [layers, batch, kv_heads, capacity, head_dim]; weights f32 and positions int32
    [layers, batch, kv_heads, capacity]; lengths, seen int32 [batch]. Entries at positions
    seen[b] - recent and later stay first, then those of largest weight (NaN last; the lowest
    slot first among equals). Kept entries in slots below the budget stay where they are; those
    behind it move into the holes, both in ascending order, so slots are in no order of position
    afterwards. The kept entries' weights and positions go to weights_out and positions_out
    [layers, batch, kv_heads, at least budget], the tables themselves by default. Sequences of up
    to `budget` entries keep them all. lengths are the caller's to set to min(lengths, budget)."""
    device = keys.get_device()
    _need(keys.dtype in _KINDS and device >= 0 and keys.dim() == 5,
          "keys: bf16 or f16 [layers, batch, kv_heads, capacity, head_dim] on a CUDA device")
    layers, batch, kv_heads, capacity, d = keys.shape
    budget, recent = int(budget), int(recent)
    _need(0 < budget <= capacity and recent >= 0,
          "a budget of 1 up to the capacity, and recent not negative")
    keys_strides = element_rows("keys", keys, keys.shape, keys.dtype, device)
    values_strides = element_rows("values", values, keys.shape, keys.dtype, device)
    table = (layers, batch, kv_heads, capacity)
    weights_strides = element_rows("weights", weights, table, torch.float32, device)
    _need(element_rows("positions", positions, table, torch.int32, device) == weights_strides,
          "weights and positions are laid out alike")
    weights_out = weights if weights_out is None else weights_out
    positions_out = positions if positions_out is None else positions_out
    width = weights_out.shape[-1]
    _need(width >= budget, "weights_out: at least budget entries a head")
    table = (layers, batch, kv_heads, width)
    out_strides = element_rows("weights_out", weights_out, table, torch.float32, device)
    _need(element_rows("positions_out", positions_out, table, torch.int32, device) == out_strides,
          "weights_out and positions_out are laid out alike")
    for name, t in (("lengths", lengths), ("seen", seen)):
        whole(name, t, (batch,), torch.int32, device)
    if status is not None:
        whole("status", status, (1,), torch.int32, device)
    beside = begin(device)
    try:
        kept = lengths.new_empty((layers, batch, kv_heads, budget))
        size = _evict_workspace(layers, batch, kv_heads, d, capacity, budget)
        workspace = lengths.new_empty(max(size // 4, 4))
        if runtime.library().ppyb200_evict(_EVICT.pack(
                keys.data_ptr(), values.data_ptr(), weights.data_ptr(), positions.data_ptr(),
                weights_out.data_ptr(), positions_out.data_ptr(), kept.data_ptr(),
                lengths.data_ptr(), seen.data_ptr(), _address(status), workspace.data_ptr(),
                workspace.numel() * 4, layers, batch, kv_heads, d, capacity, budget, recent,
                *keys_strides[:4], *values_strides[:4], *weights_strides[:3],
                *out_strides[:3])) != runtime.STATUS_OK:
            raise B200Error(runtime.last_error())
    finally:
        end(beside)
    return kept


class Extension(NamedTuple):
    """What an extension leaves for `KVCache.accept`: its queries [layers, batch, nodes, query
    heads, head_dim], log-sum-exps f32 [layers, batch, query heads, nodes], and each sequence's
    real nodes, int32 [batch] (None: all)."""

    queries: object
    lse: object
    counts: object = None


class KVCache:
    """Keys and values of `batch` sequences over `layers` layers, with what decoding keeps beside
    them, as plain torch tensors:

        keys, values   [layers, batch, heads, capacity, head_dim]
        weights        f32 [layers, batch, heads, capacity], accumulated attention weights
                       (None with weights=False: nothing is accumulated or evicted)
        positions      int32, laid out as weights: the token position of each entry
        lengths, seen  int32 [batch]: entries in the cache, and tokens accepted so far

    `pending` is what the last extension left for `accept` (an `Extension`)."""

    def __init__(self, layers: int, batch: int, heads: int, head_dim: int, capacity: int,
                 dtype=torch.bfloat16, device="cuda", weights: bool = True) -> None:
        _need(dtype in _KINDS, "a cache of bf16 or f16")
        shape = (layers, batch, heads, capacity)
        self.keys = torch.zeros(*shape, head_dim, dtype=dtype, device=device)
        self.values = torch.zeros_like(self.keys)
        self.weights = torch.zeros(shape, dtype=torch.float32, device=device) if weights else None
        self.positions = torch.zeros(shape, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.pending = None
        self.buffers: dict = {}  # the activations of the largest extension so far

    @property
    def capacity(self) -> int:
        return self.keys.shape[3]

    def release(self) -> None:
        """Give back the activations, a pending extension's among them."""
        self.pending = None
        for t in self.buffers.values():  # work on them may be under way on this stream
            t.record_stream(torch.cuda.current_stream(t.device))
        self.buffers.clear()

    def reset(self) -> None:
        """Forget every sequence, and release the activations."""
        self.release()
        self.lengths.zero_()
        self.seen.zero_()
        self.status.zero_()

    def check(self) -> None:
        """Raise if an index given to a call since the last check was out of range, or a kernel
        gave up (syncs)."""
        if int(self.status.item()) != 0:
            self.status.zero_()
            raise B200Error("a length, count, parent, path, position or token id was out of range, "
                            "or a kernel gave up a wait and left NaN")

    def accept(self, path=None, accepted=None) -> None:
        """The nodes path[b, :accepted[b]] of the last extension (int32 [batch, steps] and
        [batch], as `accept_nodes`; all nodes without a path, each sequence's first accepted[b]
        of them, or as many as it has) join the cache: lengths and seen grow by the steps taken, fewer than `accepted`
        where the path is cut. Paths longer than accept_nodes takes go in pieces."""
        _need(self.pending is not None, "accept follows an extension")
        q, lse, counts = Extension(*self.pending)
        nodes, heads, device = q.shape[2], q.shape[3], self.keys.device
        if path is None:
            path = torch.arange(nodes, dtype=torch.int32, device=device)
            accepted = counts if accepted is None else accepted
        else:
            _need(path.dim() == 2, "path: int32 [batch, steps]")
            path = path.contiguous()
        steps = path.shape[-1]
        if accepted is None:
            accepted = torch.full_like(self.lengths, steps)
        group = heads // self.keys.shape[2]
        _need(group <= PATH_ROWS, "up to 512 query heads a key head")
        most, before = min(PATH_STEPS, PATH_ROWS // group), None
        for first in range(0, steps, most):
            taken = torch.empty_like(self.lengths)
            _accept(q, lse, self.keys, self.values, self.weights, self.positions, self.lengths,
                    self.seen, path, accepted, None, self.status, taken, counts, first,
                    min(most, steps - first), before)
            grown = taken if before is None else taken - before
            self.lengths += grown
            self.seen += grown
            before = taken
        self.pending = None

    def evict(self, budget: int, recent: int = 0):
        """Cut every sequence to `budget` entries (see `evict`); returns `kept`. Not while an
        extension is pending: its nodes lie behind the lengths that this changes."""
        _need(self.weights is not None, "eviction takes a cache with weights")
        _need(self.pending is None, "an extension is pending: accept it, or none of it, first")
        kept = evict(self.keys, self.values, self.weights, self.positions, self.lengths,
                     self.seen, budget, recent, status=self.status)
        self.lengths.clamp_(max=budget)
        return kept
