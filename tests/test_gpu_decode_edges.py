"""The decoding operators where their sizes, masks and orders of calls are odd. Inputs, plain forms and
tolerances are those of test_gpu_decode.py unless a test says otherwise."""

from __future__ import annotations

import math

import pytest

from test_gpu_decode import BF16, F16, Inputs, _near, bound  # noqa: F401 - the fixture

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


def _plain_accept(cache, before, path, accepted, nodes):
    """What lengths, seen, positions, keys and values are after `path` (a list per sequence) of an
    extension of `nodes` nodes: steps up to the first that is out of order or not in the cache."""
    for b, steps in enumerate(path):
        length, seen = int(before["lengths"][b]), int(before["seen"][b])
        want, last = [], -1
        for p in steps[:max(0, int(accepted[b]))]:
            if p <= last or p >= nodes or length + p >= cache.capacity:
                break
            want.append(p)
            last = p
        n = len(want)
        assert int(cache.lengths[b]) == length + n and int(cache.seen[b]) == seen + n
        old = [length + p for p in want]
        for name in ("keys", "values"):
            now = getattr(cache, name)[:, b]
            assert torch.equal(now[:, :, :length], before[name][:, b, :, :length])
            assert torch.equal(now[:, :, length:length + n], before[name][:, b][:, :, old])
            assert torch.equal(now[:, :, length + n:], before[name][:, b, :, length + n:])
        assert bool((cache.positions[:, b, :, length:length + n] == torch.arange(
            seen, seen + n, device="cuda")).all())


def _pending_cache(lengths, nodes, capacity, heads=2, kv=2, d=64, seed=3):
    """A cache with an extension of random keys, values and queries behind `lengths`."""
    from ppy_b200 import decode

    g = torch.Generator(device="cuda").manual_seed(seed)
    batch = len(lengths)
    cache = decode.KVCache(2, batch, kv, d, capacity)
    cache.keys.normal_(generator=g)
    cache.values.normal_(generator=g)
    cache.lengths.copy_(torch.tensor(lengths))
    cache.seen.copy_(torch.tensor(lengths) + 5)
    cache.pending = (torch.randn(2, batch, nodes, heads, d, device="cuda", generator=g).to(BF16),
                     5 + torch.rand(2, batch, heads, nodes, device="cuda", generator=g))
    before = {k: getattr(cache, k).clone() for k in ("keys", "values", "lengths", "seen")}
    return cache, before


@pytest.mark.parametrize("path,accepted,raises", [
    ([[0, 2, 3], [1, 4, 5]], [3, 2], False),
    ([[0, 2, 2], [4, 1, 5]], [3, 3], True),       # cut after two steps, and after one
    ([[5, 6, 7], [0, 1, 2]], [3, 3], True),       # nodes that do not exist
    ([[0, 1, 2], [-1, 0, 1]], [3, 3], True),
    ([[0, 1, 2], [0, 1, 2]], [4, -1], True),      # counts out of range: all, and none
    ([[0, 1, 2], [0, 1, 2]], [0, 0], False),
])
def test_cache_grows_by_the_steps_taken(path, accepted, raises):
    from ppy_b200.runtime import B200Error

    cache, before = _pending_cache((20, 7), 6, 64)
    cache.accept(torch.tensor(path, dtype=torch.int32, device="cuda"),
                 torch.tensor(accepted, dtype=torch.int32, device="cuda"))
    if raises:
        with pytest.raises(B200Error, match="out of range"):
            cache.check()
    cache.check()
    _plain_accept(cache, before, path, accepted, 6)


def test_cache_never_grows_past_its_capacity():
    """An extension that does not fit: the nodes that do are taken, and the cache stays usable."""
    from ppy_b200.runtime import B200Error

    cache, before = _pending_cache((60, 64, 20), 6, 64)
    cache.accept()
    with pytest.raises(B200Error, match="out of range"):
        cache.check()
    assert cache.lengths.tolist() == [64, 64, 26] and cache.seen.tolist() == [69, 69, 31]
    _plain_accept(cache, before, [list(range(6))] * 3, [6, 6, 6], 6)


@pytest.mark.parametrize("heads,kv,cut", [(2, 2, None), (2, 2, 64), (8, 1, 70), (2, 2, 130),
                                          (16, 1, 31)])
def test_long_paths_in_pieces(heads, kv, cut):
    """Paths of 150 of 200 nodes, in pieces of 64 steps (32 with 16 heads on a key head), ascending
    across the pieces; cut for one sequence by a step that repeats the one before. Weights and
    rows are those of the same steps taken one after the other."""
    from ppy_b200 import decode

    nodes, lengths = 200, (90, 0, 33)
    g = torch.Generator().manual_seed(7)
    path = torch.stack([torch.randperm(nodes, generator=g)[:150].sort().values for _ in lengths])
    if cut is not None:
        path[1, cut] = path[1, cut - 1]
    accepted = [150, 150, 97]
    cache, before = _pending_cache(lengths, nodes, 400, heads, kv)
    q, lse = cache.pending
    other, _ = _pending_cache(lengths, nodes, 400, heads, kv)
    cache.accept(path.to(torch.int32).cuda(),
                 torch.tensor(accepted, dtype=torch.int32, device="cuda"))
    assert int(cache.status) == (0 if cut is None else 2)
    _plain_accept(cache, before, path.tolist(), accepted, nodes)
    taken = [150, 150 if cut is None else cut, 97]
    # one step a call: the node's slot, counted from the length as it is now, moves down with it
    for step in range(150):
        node = path[:, step].clamp(min=0)
        on = torch.tensor([int(step < n) for n in taken], dtype=torch.int32, device="cuda")
        index = node.cuda()[None, :, None, None, None]
        here = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
        # bring the node's row to the slot at the length, where a tree of one node has it
        for b in range(3):
            if step < taken[b]:
                at, to = lengths[b] + int(node[b]), int(other.lengths[b])
                for t in (other.keys, other.values):
                    t[:, b, :, to] = t[:, b, :, at].clone()
        decode.accept_nodes(q.gather(2, index.expand(2, 3, 1, heads, 64)),
                            lse.gather(3, index[..., 0].permute(0, 1, 3, 2).expand(2, 3, heads, 1)),
                            other.keys, other.values, other.weights, other.positions,
                            other.lengths, other.seen, here, on)
        other.lengths += on
        other.seen += on
    # a score is off by at most ds on either side, f32 sums of the same terms in another order by
    # half a step a term
    ds = 66 * 2.0 ** -23 / 8 * float((q.abs().double().transpose(2, 3).reshape(2, 3, kv, -1, 64)
                                      @ before["keys"].abs().double().transpose(3, 4)).max())
    terms = 150 * heads // kv
    for b, n in enumerate(taken):
        end = lengths[b] + n
        assert torch.equal(cache.keys[:, b, :, :end], other.keys[:, b, :, :end])
        got, want = cache.weights[:, b, :, :end].double(), other.weights[:, b, :, :end].double()
        assert bool(((got - want).abs() <= (2 * ds + 2 * terms * 2.0 ** -24) * want).all())


def test_padded_extensions_are_accepted_without_their_padding():
    """Prompts of different lengths in one batch: accept() takes each sequence's own nodes, and the
    next token's logits are those of each prompt by itself. The counts may change meanwhile."""
    model, cache = _model_and_cache(3, 64)
    ids, token = _ids(3, 20), _ids(3, 1, seed=1)
    counts = torch.tensor([20, 3, 11], dtype=torch.int32, device="cuda")
    model.extend(cache, _ids(3, 20, seed=2))  # leaves other nodes behind, never accepted
    model.extend(cache, ids, counts=counts)
    counts.fill_(1)
    cache.accept()
    cache.check()
    assert cache.lengths.tolist() == [20, 3, 11] == cache.seen.tolist()
    logits = model.extend(cache, token)
    for b, n in enumerate((20, 3, 11)):
        alone = model.new_cache(1, capacity=64)
        model.extend(alone, ids[b:b + 1, :n])
        alone.accept()
        _near(cache.keys[:, b, :, :n], alone.keys[:, 0, :, :n])
        _near(logits[b], model.extend(alone, token[b:b + 1])[0])
        total = cache.weights[:, b, :, :n].sum(-1)
        assert bool(((total - n).abs() <= 1e-3 * n).all())


def test_a_path_ends_at_a_sequences_nodes():
    from ppy_b200.runtime import B200Error

    cache, before = _pending_cache((20, 7, 9), 6, 64)
    counts = torch.tensor([6, 3, 0], dtype=torch.int32, device="cuda")
    cache.pending = (*cache.pending, counts)
    path = [[0, 4, 5], [1, 2, 4], [0, 1, 2]]
    cache.accept(torch.tensor(path, dtype=torch.int32, device="cuda"))
    with pytest.raises(B200Error, match="out of range"):
        cache.check()
    assert cache.lengths.tolist() == [23, 9, 9]
    _plain_accept(cache, before, path, [3, 2, 0], 6)


# ---------------------------------------------------------------- outputs


@pytest.mark.parametrize("nodes,heads,kv,cap,tree", [
    (5, 4, 2, 200, True),        # the kernel of few rows
    (70, 8, 2, 300, False),      # the tensor-core kernel
    (12, 8, 2, 40_000, True),    # that, with copies of its rows
])
@pytest.mark.parametrize("padded", [False, True])
def test_nodes_that_do_not_fit_have_zeros(nodes, heads, kv, cap, tree, padded):
    lengths = (cap - nodes, cap - 3, cap, 10)
    counts = (nodes, nodes - 1, 4, 2) if padded else None
    x = Inputs(lengths, nodes, heads, kv, 64, tree=tree, counts=counts, spare=0)
    x.keys, x.values = x.keys[:, :, :cap], x.values[:, :, :cap]
    out = torch.full_like(x.q, 7.0, memory_format=torch.contiguous_format)
    lse = torch.full((4, heads, nodes), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x.call(out=out, lse=lse, status=status)
    assert int(status) == 2
    made, made_lse = x.call()
    for b, length in enumerate(lengths):
        n = nodes if counts is None else counts[b]
        fit = min(n, cap - length)
        assert bool(lse[b, :, :fit].ne(5.0).all()) and bool(out[b, :fit].ne(7.0).any(-1).all())
        assert not out[b, fit:n].any() and not lse[b, :, fit:n].any()
        assert bool((out[b, n:] == 7.0).all()) and bool((lse[b, :, n:] == 5.0).all())
        assert not made[b, fit:].any() and not made_lse[b, :, fit:].any()
    # what fits is right: the same nodes as counts that say so
    y = Inputs(lengths, nodes, heads, kv, 64, tree=tree, spare=0, counts=[
        min(nodes if counts is None else counts[b], cap - n) for b, n in enumerate(lengths)])
    y.keys, y.values = y.keys[:, :, :cap], y.values[:, :, :cap]
    want, want_lse = y.call()
    assert torch.equal(made, want) and torch.equal(made_lse, want_lse)


@pytest.mark.parametrize("nodes", [1, 80])
def test_a_cache_without_slots(nodes):
    """No node fits: zeros and the status, from either kernel's sizes."""
    x = Inputs((0,), nodes, 4, 2, 64, tree=False)
    x.keys, x.values = x.keys[:, :, :0], x.values[:, :, :0]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = x.call(status=status)
    assert int(status) == 2 and not out.any() and not lse.any()


def test_a_refused_extension_leaves_the_pending_one():
    from ppy_b200.runtime import B200Error

    model, cache = _model_and_cache(1, 400)
    ids = _ids(1, 300)
    model.extend(cache, ids)
    parents = torch.arange(-1, 299, dtype=torch.int32, device="cuda")
    with pytest.raises(B200Error, match="256 nodes"):
        model.extend(cache, _ids(1, 300, seed=1), parents)
    cache.accept()
    alone = model.new_cache(1, capacity=400)
    model.extend(alone, ids)
    alone.accept()
    assert torch.equal(cache.keys, alone.keys) and torch.equal(cache.weights, alone.weights)


# ---------------------------------------------------------------- memory between calls


def test_activations_do_not_pile_up():
    """Extensions of many shapes hold one set of activations, as large as the largest of them, and a
    reset gives it back; what they compute is what caches of their own get."""
    model, cache = _model_and_cache(2, 300, layers=2)
    model.extend(cache, _ids(2, 1))  # everything that is made once
    cache.reset()
    # bytes asked of the allocator: what it hands out is rounded up, by up to 1 MB a tensor
    asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # noqa: E731
    start, largest = asked(), 0
    for step, length in enumerate((200, 3, 17, 1, 64, 5, 130)):
        cache.reset() if step else None
        ids = _ids(2, length, seed=step)
        logits = model.extend(cache, ids)
        held = asked() - start - 2 * length * (8 + 4 * 50272)  # ids and padded logits
        tokens, c = 2 * length, model.config.width
        # x, h, two layers' qkv, att and f, and the log sums
        assert held == tokens * c * (4 + 2 + 2 * 6 + 2 + 8) + 2 * tokens * 12 * 4
        del logits, ids
    cache.reset()
    for length in (64, 5, 200, 1, 130):  # without a reset in between: as large as the largest
        ids = _ids(2, length, seed=length)
        got = model.extend(cache, ids)
        alone = model.new_cache(2, capacity=300)
        model.extend(cache, ids)
        assert torch.equal(got, model.extend(alone, ids))
        largest = max(largest, length)
        sizes = {name: t.numel() for name, t in cache.buffers.items()}
        assert sizes["x"] == 2 * largest * model.config.width
        cache.pending = None
        del got, alone


def test_a_captured_extension_has_its_own_activations():
    """The cache's set may be replaced by a larger one, or released, between capture and replay."""
    from ppy_b200 import runtime

    model, cache = _model_and_cache(2, 200)
    prompt, tokens = _ids(2, 90, seed=3), _ids(2, 3, seed=4)
    stream = torch.cuda.Stream()
    runtime.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            token, logits = torch.zeros(2, 1, dtype=torch.int64, device="cuda"), model.new_logits(2, 1)
            model.extend(cache, token, logits=logits)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                model.extend(cache, token, logits=logits)
                cache.accept()
            cache.reset()
            model.extend(cache, prompt)
            cache.accept()
            other = model.new_cache(2, capacity=200)
            model.extend(other, prompt)
            other.accept()
            for i in range(3):
                if i == 1:
                    cache.release()
                junk = torch.full((1 << 22,), math.nan, device="cuda")
                token.copy_(tokens[:, i:i + 1])
                graph.replay()
                want = model.extend(other, tokens[:, i:i + 1])
                other.accept()
                assert torch.equal(logits, want), i
                del junk
            assert torch.equal(cache.lengths, other.lengths)
            assert torch.equal(cache.weights, other.weights)
        stream.synchronize()
    finally:
        runtime.set_stream(torch.cuda.current_stream())


def test_padded_rows_stay_finite_after_other_extensions():
    """The activations of an extension before lie in the rows behind a sequence's nodes."""
    model, cache = _model_and_cache(2, 64)
    model.extend(cache, _ids(2, 8))
    for t in cache.buffers.values():
        t.fill_(math.nan)
    cache.pending = None
    logits = model.extend(cache, _ids(2, 8), counts=torch.tensor([8, 2], dtype=torch.int32,
                                                                 device="cuda"))
    assert bool(logits.isfinite().all())


# ---------------------------------------------------------------- scoring texts


@pytest.mark.parametrize("batch,length", [(1, 1), (2, 2), (3, 37), (2, 128), (1, 129), (1, 1000)])
def test_score_texts_of_any_length(batch, length):
    from oracle import gpt2 as oracle_gpt2

    model, _ = _model_and_cache(1, 1)
    ids = _ids(batch, length + 3, seed=length)[:, :length]  # rows of a larger tensor
    scores = model.score(ids, top=3)
    assert scores.logprobs.shape == scores.entropy.shape == (batch, length - 1)
    assert scores.top_tokens.shape == scores.top_logprobs.shape == (batch, length - 1, 3)
    room = model.new_logits(batch, (length + 127) // 128 * 128)
    again = model.score(ids, top=3, logits=room)
    assert all(torch.equal(a, b) for a, b in zip(scores, again))
    rows = room[:, :length - 1].double()
    want = torch.log_softmax(rows, -1)
    # the bound of the scores given their logits (test_gpu_scoring.py)
    picked = want.gather(-1, ids[:, 1:, None])[..., 0]
    assert bool(((scores.logprobs.double() - picked).abs() < 1e-4).all())
    assert bool((scores.top_logprobs.double() - want.topk(3, -1).values).abs().lt(1e-4).all())
    if length > 1:  # and the logits are those of the text without its padding
        _near(rows, oracle_gpt2.forward(model, ids.contiguous())[:, :-1])


def test_score_texts_that_lie_in_columns():
    model, _ = _model_and_cache(1, 1)
    for length in (100, 128):
        ids = _ids(3, length)
        columns = ids.t().contiguous().t()
        assert not columns.is_contiguous()
        got, want = model.score(columns, top=1), model.score(ids, top=1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_score_beside_torchs_stream():
    """ids made on torch's stream while the launches go to another: no wait by the caller."""
    from ppy_b200 import runtime

    model, _ = _model_and_cache(1, 1)
    ids = _ids(2, 200)
    want = model.score(ids, top=2)
    torch.cuda.synchronize()
    try:
        for stream in (None, torch.cuda.Stream()):
            runtime.set_stream(stream)
            for _ in range(5):
                held = torch.randn(4096, 4096, device="cuda")
                held = held @ held  # work before the inputs on torch's stream
                got = model.score(ids + 0, top=2)
                assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        runtime.set_stream(torch.cuda.current_stream())


def test_score_refusals():
    from ppy_b200.runtime import B200Error

    model, _ = _model_and_cache(1, 1)
    for ids in (_ids(1, 5).int(), _ids(1, 5).cpu(), _ids(1, 0), _ids(1, 1025)):
        with pytest.raises(B200Error):
            model.score(ids)
    with pytest.raises(B200Error, match="logits"):
        model.score(_ids(1, 5), logits=model.new_logits(1, 5))


# ---------------------------------------------------------------- small weights, infinities


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("length,nodes,heads,kv,cap", [
    (60_000, 1, 1, 1, 60_100),     # the kernel of few rows
    (60_000, 70, 1, 1, 60_100),    # the tensor-core kernel
    (60_000, 12, 4, 4, 300_000),   # that, with copies of its rows
])
def test_many_small_weights(length, nodes, heads, kv, cap, dtype):
    """One entry of weight 1 and value 0, the rest of weight e^-18 and value 1, nodes of weight 1 and
    value 0: the small weights add up to all there is. Scores are exact; a weight is rounded to u
    of itself, or to 2^-36 of the largest where it is subnormal, the result to u of itself; 2^-18
    for exponentials and sums."""
    u = {F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]
    x = Inputs((length,), nodes, heads, kv, 64, dtype, tree=False, spare=cap - length - nodes)
    x.q.zero_()[..., 0] = 1
    x.k_new.zero_()
    x.v_new.zero_()
    x.keys[:, :, :length] = 0
    x.keys[:, :, 1:length, 0] = -18
    x.values[:, :, :length] = 1
    x.values[:, :, 0] = 0
    out, lse = x.call(scale=1.0)
    small = (length - 1) * math.exp(-18)
    ones = torch.arange(2, nodes + 2, dtype=torch.float64, device="cuda")[:, None]
    want = small / (ones + small)
    assert bool(((out[0].double() - want[..., None]).abs()
                 <= (2 * u + 2.0 ** -18) * want[..., None] + 2.0 ** -36 * length).all())
    # up to 592 parts (four CTAs an SM) are added in f32 one after the other, each sum rounded by up to
    # 2^-24 of itself: what they add is below the sum's own last bits
    assert bool(((lse[0].double().t() - (ones + small).log()).abs()
                 <= 2.0 ** -18 + 592 * 2.0 ** -24).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,nodes,heads,kv,d,cap,tree", [
    ((70, 300), 5, 4, 2, 64, 400, True),          # the kernel of few rows
    ((300, 31), 45, 6, 2, 128, 2_000, False),     # the tensor-core kernel
    ((4000, 129), 1, 8, 2, 64, 270_000, False),   # four copies of its rows
    ((1111, 500), 12, 8, 2, 128, 60_000, True),   # two copies
])
def test_infinities_in_the_cache(lengths, nodes, heads, kv, d, cap, tree, dtype):
    """A cached value that is not finite is seen by every row of its key head: an infinity gives
    infinities, two of opposite signs or a NaN give NaN, in that column and no other."""
    x = Inputs(lengths, nodes, heads, kv, d, dtype, tree=tree, spare=cap - max(lengths) - nodes)
    clean, clean_lse = x.call()
    x.values[0, 0, 3, 1] = math.inf
    x.values[0, 0, 64, 7] = -math.inf
    x.values[0, 0, [5, 20], [9, 9]] = math.inf
    x.values[0, 0, 2, 12] = math.inf
    x.values[0, 0, 29, 12] = -math.inf
    x.values[0, 0, 6, 14] = math.nan
    x.v_new[0, 0, 0, 17] = -math.inf  # a node's, for the rows that see it
    x.values[0, 0, 30, 17] = -math.inf
    out, lse = x.call()
    assert torch.equal(lse, clean_lse)
    group = heads // kv
    rows = out[0, :, :group].float()
    for col, want in ((1, math.inf), (7, -math.inf), (9, math.inf), (17, -math.inf)):
        assert bool((rows[..., col] == want).all()), col
    assert bool(rows[..., [12, 14]].isnan().all())
    same = torch.ones_like(out, dtype=torch.bool)
    same[0, :, :group, [1, 7, 9, 12, 14, 17]] = False
    assert torch.equal(out[same], clean[same])


@pytest.mark.parametrize("lengths,nodes,heads,kv,d,cap,tree", [
    ((300, 31), 45, 6, 2, 128, 2_000, False),            # two row tiles that share their keys
    ((4000, 129), 1, 8, 2, 64, 270_000, False),          # four copies of the rows
    ((1111, 5), 12, 8, 2, 128, 60_000, True),            # two
    ((1, 640), 64, 2, 2, 64, 30_000, True),
    ((60,), 20, 8, 1, 64, 128, True),                    # one CTA, no workspace
    (tuple(range(1, 161, 8)), 40, 32, 8, 64, 300, True),  # more items than CTAs
])
def test_a_wait_given_up_leaves_no_old_memory(lengths, nodes, heads, kv, d, cap, tree):
    """Every wait gives up before it tries: the status says so, and rows without a result are NaN,
    with or without a status word. The next call is right."""
    from ppy_b200 import runtime

    counts = [max(1, nodes - 3 * b) for b in range(len(lengths))]
    x = Inputs(lengths, nodes, heads, kv, d, tree=tree, counts=counts,
               spare=cap - max(lengths) - nodes)
    lib = runtime.library()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(x.q, 7.0, memory_format=torch.contiguous_format)
    lse = torch.full((len(lengths), heads, nodes), 5.0, device="cuda")
    try:
        lib.ppyb200_tree_attention_wait_limit(0)
        x.call(out=out, lse=lse, status=status)
        made, made_lse = x.call()
    finally:
        lib.ppyb200_tree_attention_wait_limit(-1)
    assert int(status) == 2
    for b, n in enumerate(counts):
        for o, s in ((out, lse), (made, made_lse)):
            assert bool(o[b, :n].isnan().all()) and bool(s[b, :, :n].isnan().all())
        assert bool((out[b, n:] == 7.0).all()) and bool((lse[b, :, n:] == 5.0).all())
    for b, n in enumerate(lengths):
        x.keys[b, :, n:] = math.nan
        x.values[b, :, n:] = math.nan
    x.check(*x.call())


# ---------------------------------------------------------------- orders of calls, captured


def test_a_padded_step_captured_on_the_runtimes_own_stream():
    """Extension, acceptance and eviction of a padded batch in one graph, torch's stream capturing and
    the launches on the runtime's: replays are the same calls made one by one."""
    from ppy_b200 import runtime

    model, cache = _model_and_cache(3, 64)
    other = model.new_cache(3, capacity=64)
    prompt, steps = _ids(3, 20, seed=1), _ids(3, 12, seed=2)
    counts = [[4, 1, 3], [2, 4, 1], [1, 1, 4]]
    for c in (cache, other):
        model.extend(c, prompt)
        c.accept()
    ids = torch.zeros(3, 4, dtype=torch.int64, device="cuda")
    real = torch.ones(3, dtype=torch.int32, device="cuda")
    logits = model.new_logits(3, 4)
    stream = torch.cuda.Stream()
    try:
        runtime.set_stream(None)
        with torch.cuda.stream(stream):
            warm = model.new_cache(3, capacity=64)
            model.extend(warm, ids, counts=real, logits=logits)
            warm.accept()
            warm.evict(21, recent=2)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                model.extend(cache, ids, counts=real, logits=logits)
                cache.accept()
                kept = cache.evict(21, recent=2)
        for i, n in enumerate(counts):
            with torch.cuda.stream(stream):
                ids.copy_(steps[:, 4 * i:4 * i + 4])
                real.copy_(torch.tensor(n, dtype=torch.int32))
                graph.replay()
                got = logits.clone()
                want = model.extend(other, steps[:, 4 * i:4 * i + 4],
                                    counts=torch.tensor(n, dtype=torch.int32, device="cuda"))
                other.accept()
                want_kept = other.evict(21, recent=2)
                for b in range(3):
                    assert torch.equal(got[b, :n[b]], want[b, :n[b]])
                assert torch.equal(kept, want_kept)
                for name in ("lengths", "seen"):
                    assert torch.equal(getattr(cache, name), getattr(other, name))
                for b in range(3):
                    length = int(cache.lengths[b])
                    for name in ("keys", "values", "weights", "positions"):
                        assert torch.equal(getattr(cache, name)[:, b, :, :length],
                                           getattr(other, name)[:, b, :, :length]), name
        cache.check()
        other.check()
        assert cache.seen.tolist() == [27, 26, 28]
    finally:
        torch.cuda.synchronize()
        runtime.set_stream(torch.cuda.current_stream())


def test_a_cache_without_weights_decodes_the_same():
    model, cache = _model_and_cache(2, 120, layers=2)
    bare = model.new_cache(2, capacity=120, weights=False)
    prompt, tree = _ids(2, 80, seed=1), _ids(2, 4, seed=2)
    parents = torch.tensor([-1, 0, 0, 2], dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 2, 3], [0, 1, 3]], dtype=torch.int32, device="cuda")
    accepted = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    for step in range(2):
        outs = []
        for c in (cache, bare):
            model.extend(c, prompt[:, 40 * step:40 * step + 40])
            c.accept()
            outs.append(model.extend(c, tree, parents))
            c.accept(path, accepted)
            c.check()
        assert torch.equal(*outs)
    assert torch.equal(cache.keys, bare.keys) and torch.equal(cache.values, bare.values)
    assert torch.equal(cache.positions, bare.positions) and bare.weights is None
