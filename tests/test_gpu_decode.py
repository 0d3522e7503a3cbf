"""Tree attention over a cache, acceptance and eviction against plain forms in float64, and the
three as GPT-2 decodes with them.

Tolerances. With u half a step of the 16-bit type (bf16 2^-8, f16 2^-11): products of 16-bit values
are exact in f32, and a score sums head_dim of them, so it is off by at most ds = (head_dim + 2)
2^-23 scale max_j sum |q||k_j| (the tensor core may truncate: a whole f32 step a sum). A weight e^s
is then off by at most 2 ds + 2^-20 of itself (its own error and its row's normaliser's, and the
exponential's 2^-22), and it is rounded to u before it meets the values; the result is rounded
once more. Hence |out - ref| <= (u + 2 ds + 2^-20) sum p |v| + u |ref|, in f16 plus 2^-25 sum |v|,
where weights are subnormal. Accumulated weights are sums of e^{s - lse} in f32: 2 ds + 2^-18 of
themselves (up to 64 terms summed, 2^-24 each)."""

from __future__ import annotations

import math

import pytest

from oracle import gpt2 as oracle_gpt2

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def bound():
    from ppy_b200 import runtime

    if not torch.cuda.is_available():
        pytest.fail("a GPU test ran without a CUDA device")
    runtime.init(0)
    runtime.set_stream(torch.cuda.current_stream())


def _ancestors(parents, i):
    found = [i]
    while parents[found[-1]] >= 0:
        found.append(parents[found[-1]])
    return found


class Inputs:
    """Random queries, nodes and a cache whose slots behind the lengths hold NaN."""

    def __init__(self, lengths, nodes, heads, kv, d, dtype=BF16, layout="heads", tree=True,
                 counts=None, spare=5, seed=0, sharp=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        batch, cap = len(lengths), max(lengths) + nodes + spare
        self.d, self.dtype, self.parents_list = d, dtype, None
        qkv = torch.randn(batch, nodes, (heads + 2 * kv) * d, device="cuda", generator=g)
        q, k, v = qkv.to(dtype).split((heads * d, kv * d, kv * d), -1)
        self.q = q.mul_(sharp).view(batch, nodes, heads, d)
        self.k_new, self.v_new = k.view(batch, nodes, kv, d), v.view(batch, nodes, kv, d)
        shape = (batch, kv, cap, d) if layout == "heads" else (batch, cap, kv, d)
        self.keys = torch.randn(shape, device="cuda", generator=g).to(dtype)
        self.values = torch.randn(shape, device="cuda", generator=g).to(dtype)
        if layout == "tokens":
            self.keys, self.values = self.keys.transpose(1, 2), self.values.transpose(1, 2)
        for b, n in enumerate(lengths):
            self.keys[b, :, n:] = math.nan
            self.values[b, :, n:] = math.nan
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.parents = None
        if tree:
            back = 1 + torch.randint(0, 6, (batch, nodes), device="cuda", generator=g)
            index = torch.arange(nodes, device="cuda")
            self.parents = (index - back).clamp(min=-1).to(torch.int32)
        self.counts = None if counts is None else torch.tensor(counts, dtype=torch.int32,
                                                               device="cuda")

    def call(self, **more):
        from ppy_b200 import decode

        return decode.tree_attention(self.q, self.k_new, self.v_new, self.keys, self.values,
                                     self.lengths, self.parents, self.counts, **more)

    def check(self, out, lse, scale=None, heads=None):
        """The outputs against float64, and the cache's new rows bit for bit."""
        batch, nodes, count, d = self.q.shape
        group = count // self.keys.shape[1]
        scale = d ** -0.5 if scale is None else scale
        u = U[self.dtype]
        for b, length in enumerate(self.lengths.tolist()):
            n = nodes if self.counts is None else int(self.counts[b])
            if n == 0:
                continue
            parents = (list(range(-1, nodes - 1)) if self.parents is None
                       else self.parents[b].tolist())
            for h in range(count) if heads is None else heads:
                k = torch.cat((self.keys[b, h // group, :length], self.k_new[b, :n, h // group]))
                v = torch.cat((self.values[b, h // group, :length],
                               self.v_new[b, :n, h // group]))
                seen = torch.zeros(n, length + n, dtype=torch.bool)
                seen[:, :length] = True
                for i in range(n):
                    seen[i, [length + a for a in _ancestors(parents, i)]] = True
                seen = seen.cuda()
                q, k, v = self.q[b, :n, h].double(), k.double(), v.double()
                score = torch.where(seen, (q @ k.t()) * scale, -math.inf)
                ds = ((d + 2) * 2.0 ** -23 * abs(scale)
                      * float(torch.where(seen, q.abs() @ k.abs().t(), 0.0).max()))
                p = torch.softmax(score, 1)
                used = seen.any(0)
                v = torch.where(used[:, None], v, 0.0)
                ref, spread = p @ v, p @ v.abs()
                tol = (u + 2 * ds + 2.0 ** -20) * spread + u * ref.abs()
                if self.dtype == F16:
                    tol = tol + 2.0 ** -25 * v.abs().sum(0)
                off = (out[b, :n, h].double() - ref).abs()
                assert bool((off <= tol).all()), (b, h, float((off / tol).max()))
                want = torch.logsumexp(score, 1)
                got = lse[b, h, :n].double()
                assert bool(((got - want).abs() <= ds + 2.0 ** -20 * (1 + want.abs())).all())
            end = length + n
            assert torch.equal(self.keys[b, :, length:end], self.k_new[b, :n].transpose(0, 1))
            assert torch.equal(self.values[b, :, length:end], self.v_new[b, :n].transpose(0, 1))
            assert bool(self.keys[b, :, end:].isnan().all())
            assert bool(self.values[b, :, end:].isnan().all())


@pytest.mark.parametrize("lengths,nodes,heads,kv,d,dtype,layout,tree", [
    ((0,), 1, 1, 1, 64, BF16, "heads", True),          # nothing cached: a row sees itself only
    ((1, 0, 64), 1, 12, 12, 64, BF16, "heads", False),
    ((63, 64, 65, 129), 1, 4, 2, 128, F16, "tokens", False),  # around a tile's edge
    ((1000,), 1, 12, 12, 64, BF16, "heads", False),
    ((300, 17), 5, 6, 2, 64, BF16, "tokens", True),    # 15 rows
    ((200, 31), 16, 4, 4, 64, F16, "heads", True),     # 16 rows
    ((190,), 17, 3, 3, 80, BF16, "heads", True),       # 17 rows, a head size between 64 and 128
    ((77, 500), 8, 16, 4, 128, BF16, "heads", True),   # 32 rows
    ((77, 500), 33, 2, 2, 64, BF16, "tokens", True),   # 33 rows
    ((260,), 64, 5, 5, 64, F16, "heads", True),        # 64 rows, GPT-2 XL's odd head counts
    ((5, 129), 65, 4, 4, 128, BF16, "heads", True),    # 65 rows
    ((100, 3), 40, 16, 2, 128, F16, "tokens", True),   # 320 rows
    ((0, 70), 150, 8, 2, 64, BF16, "heads", False),    # a chain over many row tiles
    ((9,), 256, 2, 1, 64, BF16, "heads", True),        # the largest tree
    ((40,), 300, 1, 1, 72, BF16, "heads", False),      # a chain longer than that
    ((5000,), 3, 2, 1, 8, BF16, "heads", True),        # the smallest head size, many splits
    ((90, 33), 2, 160, 1, 64, BF16, "heads", True),    # more query heads a key head than a tile
    ((150, 0, 260), 3, 100, 1, 64, F16, "tokens", True),   # one node a tile of rows
    (tuple(range(0, 700, 10)), 1, 4, 2, 64, BF16, "heads", False),  # 70 sequences
    (tuple(range(5, 705, 10)), 40, 2, 1, 128, F16, "tokens", True),
    ((3000, 9000), 1, 64, 8, 128, BF16, "tokens", False),  # a large cache, few rows
])
def test_tree_attention(lengths, nodes, heads, kv, d, dtype, layout, tree):
    x = Inputs(lengths, nodes, heads, kv, d, dtype, layout, tree)
    x.check(*x.call())


def test_tree_attention_sharp_scores_and_scale():
    """Scores of a few hundred: the running maximum moves by large steps; another scale, a
    negative one among them."""
    for scale, sharp in ((None, 16.0), (0.5, 1.0), (-0.125, 4.0), (0.0, 1.0)):
        x = Inputs((700, 90), 6, 4, 2, 64, sharp=sharp, seed=3)
        x.check(*x.call(scale=scale), scale=scale)


def test_tree_attention_padded_batch_leaves_rows_alone():
    """Rows behind a sequence's nodes (all of them for one), of the outputs and of the cache."""
    counts = (7, 0, 3, 1)
    x = Inputs((100, 20, 0, 64), 7, 8, 4, 64, counts=counts)
    out = torch.full_like(x.q, 7.0, memory_format=torch.contiguous_format)
    lse = torch.full((4, 8, 7), 5.0, device="cuda")
    x.check(*x.call(out=out, lse=lse))
    for b, n in enumerate(counts):
        assert bool((out[b, n:] == 7.0).all()) and bool((lse[b, :, n:] == 5.0).all())
    made, made_lse = x.call()  # outputs made by the call are zeros there
    assert not made[1].any() and not made_lse[2, :, 3:].any()


def test_tree_attention_hidden_values_that_are_not_finite():
    """Nodes with infinities and NaN in their values and keys: rows that do not see them are as
    without them; rows that do are not finite where those are."""
    x = Inputs((70,), 12, 4, 2, 64, seed=5)
    x.parents = torch.tensor([-1, 0, 0, 1, 1, 2, -1, 6, 3, 4, 5, 7], dtype=torch.int32,
                             device="cuda")[None]
    clean, clean_lse = x.call()
    x.v_new[0, 2, 0, 3] = math.nan
    x.v_new[0, 2, 1, 9] = math.inf
    x.k_new[0, 4, 0, 0] = math.nan
    out, lse = x.call()
    parents = x.parents[0].tolist()
    for i in range(12):
        up = _ancestors(parents, i)
        for h in range(4):
            if h < 2 and 4 in up:
                assert bool(out[0, i, h].isnan().all()) and bool(lse[0, h, i].isnan())
                continue
            assert torch.equal(lse[0, h, i], clean_lse[0, h, i])
            hit = 2 in up
            assert bool(out[0, i, h, 3].isnan()) == (hit and h < 2)
            assert bool(out[0, i, h, 9].isinf()) == (hit and h >= 2)
            fine = torch.ones(64, dtype=torch.bool, device="cuda")
            fine[[3, 9]] = not hit
            assert torch.equal(out[0, i, h][fine], clean[0, i, h][fine])


@pytest.mark.parametrize("lengths,nodes,heads,kv,d,dtype,layout,tree,cap", [
    ((4000, 129), 1, 8, 2, 64, BF16, "heads", False, 270_000),  # 4 rows: four copies of each
    ((700, 0), 5, 6, 2, 128, F16, "heads", True, 140_000),      # 15 rows
    ((2500, 128), 10, 6, 2, 64, BF16, "tokens", True, 50_000),  # 30 rows, groups of three
    ((1111,), 12, 8, 2, 128, BF16, "heads", True, 60_000),      # 48 rows: two copies
    ((1, 640), 64, 2, 2, 64, F16, "heads", True, 30_000),       # 64 rows
    ((90, 1500), 20, 14, 2, 64, BF16, "heads", True, 2_000),    # groups of seven: 140 rows
    ((300, 31), 45, 6, 2, 128, F16, "tokens", False, 2_000),    # 135 rows in two uneven tiles
])
def test_tree_attention_few_rows_over_a_large_cache(lengths, nodes, heads, kv, d, dtype, layout,
                                                    tree, cap):
    x = Inputs(lengths, nodes, heads, kv, d, dtype, layout, tree,
               spare=cap - max(lengths) - nodes)
    x.check(*x.call())


@pytest.mark.parametrize("nodes,cap", [(12, 300_000), (30, 50_000), (64, 30_000)])
def test_tree_attention_hidden_values_over_a_large_cache(nodes, cap):
    """As above, for the kernel that large caches take: an infinity shows in the rows that see
    it, and in no other."""
    x = Inputs((70, 128), nodes, 4, 4, 64, seed=6, spare=cap - 128 - nodes)
    clean, clean_lse = x.call()
    x.v_new[1, 2, 1, 9] = math.inf
    out, lse = x.call()
    assert torch.equal(lse, clean_lse) and torch.equal(out[0], clean[0])
    parents = x.parents[1].tolist()
    for i in range(nodes):
        hit = 2 in _ancestors(parents, i)
        assert bool(out[1, i, 1, 9].isinf()) == hit
        fine = torch.ones(4, 64, dtype=torch.bool, device="cuda")
        fine[1, 9] = not hit
        assert torch.equal(out[1, i][fine], clean[1, i][fine])


def test_tree_attention_out_of_range_raises_status_and_keeps_to_the_buffers():
    x = Inputs((60, 20, 30), 4, 2, 2, 64, spare=0)  # a capacity of 64
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x.check(*x.call(status=status))
    assert int(status) == 0
    before = x.keys.clone()
    x.lengths.copy_(torch.tensor([62, -5, 1 << 30]))
    x.call(status=status)
    assert int(status) == 2
    # what fits is written, at the slots that the lengths held inside the buffer give
    assert torch.equal(x.keys[0, :, 62:], x.k_new[0, :2].transpose(0, 1))
    assert torch.equal(x.keys[1, :, :4], x.k_new[1].transpose(0, 1))
    assert torch.equal(x.keys[2].nan_to_num(9.0), before[2].nan_to_num(9.0))
    for wrong in (3, 4, 100, -2):  # its own index, a later one, none at all
        y = Inputs((10, 20), 4, 2, 2, 64)
        y.parents[1, 3] = wrong
        status.zero_()
        out, lse = y.call(status=status)
        assert int(status) == 2
        y.parents[1, 3] = -1  # what such a parent is taken for
        y.check(out, lse)


def test_tree_attention_cache_beyond_32_bit_offsets():
    """A token-major cache whose last slots lie more than 2^31 elements from its first."""
    cap, kv, d = 300_000, 64, 128
    x = Inputs((20,), 2, kv, kv, d)
    keys = torch.empty(1, cap, kv, d, dtype=BF16, device="cuda").normal_()
    values = torch.empty(1, cap, kv, d, dtype=BF16, device="cuda").normal_()
    x.keys, x.values = keys.transpose(1, 2), values.transpose(1, 2)
    x.lengths.fill_(cap - 2)
    x.check(*x.call(), heads=(0, 31, 63))


def test_tree_attention_on_another_stream():
    """Tensors made and used on torch's stream while the launches go to another: no wait in
    between by the caller."""
    from ppy_b200 import runtime

    x = Inputs((3000, 100), 6, 8, 4, 64)
    want, want_lse = x.call()
    x.keys[0, :, 3000:] = math.nan
    x.keys[1, :, 100:] = math.nan
    torch.cuda.synchronize()
    try:
        for stream in (None, torch.cuda.Stream()):  # the runtime's own, and a torch stream
            runtime.set_stream(stream)
            for _ in range(5):
                held = torch.randn(4096, 4096, device="cuda")
                held = held @ held  # work before the inputs on torch's stream
                q = x.q * 1
                x_q, x.q = x.q, q
                out, lse = x.call()
                same = torch.equal(out, want) and torch.equal(lse, want_lse)
                x.q = x_q
                assert same
    finally:
        runtime.set_stream(torch.cuda.current_stream())


def test_tree_attention_replays_as_the_cache_grows():
    """Captured once, replayed with other lengths: the lengths are read on the device. Two graphs
    with workspaces of their own replay on two streams at once."""
    xs = [Inputs((2000, 700), 1, 8, 8, 64, tree=False, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    from ppy_b200 import runtime

    stream = torch.cuda.Stream()
    runtime.set_stream(stream)
    try:
        for x in xs:
            with torch.cuda.stream(stream):
                x.call()
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(x.call())
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in xs]
        for lengths in ((2000, 700), (1, 0), (1500, 701)):
            for x in xs:
                x.lengths.copy_(torch.tensor(lengths))
                for b, n in enumerate(lengths):
                    x.keys[b, :, :n].nan_to_num_(0.5)
                    x.values[b, :, :n].nan_to_num_(0.5)
                    x.keys[b, :, n:] = math.nan
                    x.values[b, :, n:] = math.nan
            torch.cuda.synchronize()
            for _ in range(3):
                for graph, side in zip(graphs, streams):
                    with torch.cuda.stream(side):
                        graph.replay()
            torch.cuda.synchronize()
            for x, out in zip(xs, outs):
                x.check(*out)
    finally:
        runtime.set_stream(torch.cuda.current_stream())


# ---------------------------------------------------------------- acceptance


def _accept_inputs(layers, lengths, nodes, steps, heads, kv, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    batch, cap = len(lengths), max(lengths) + nodes + 3
    s = {"q": torch.randn(layers, batch, nodes, heads, d, device="cuda", generator=g).to(dtype),
         "keys": torch.randn(layers, batch, kv, cap, d, device="cuda", generator=g).to(dtype),
         "values": torch.randn(layers, batch, kv, cap, d, device="cuda", generator=g).to(dtype),
         "weights": torch.rand(layers, batch, kv, cap, device="cuda", generator=g),
         "positions": torch.randint(0, 99, (layers, batch, kv, cap), device="cuda",
                                    generator=g).to(torch.int32),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    s["lse"] = 4 + torch.rand(layers, batch, heads, nodes, device="cuda", generator=g)
    s["seen"] = s["lengths"] + 11
    path = torch.rand(batch, nodes, device="cuda", generator=g).argsort(1)[:, :steps]
    s["path"] = path.sort(1).values.to(torch.int32).contiguous()
    s["accepted"] = torch.tensor([max(0, steps - b) for b in range(batch)], dtype=torch.int32,
                                 device="cuda")
    return s


def _check_accept(s, done, scale=None):
    layers, batch, nodes, heads, d = s["q"].shape
    group = heads // s["keys"].shape[2]
    scale = d ** -0.5 if scale is None else scale
    for b in range(batch):
        length, n, seen = (int(s[k][b]) for k in ("lengths", "accepted", "seen"))
        path = s["path"][b, :n].tolist()
        slots = torch.tensor(list(range(length)) + [length + p for p in path], device="cuda",
                             dtype=torch.long)
        for name in ("keys", "values", "weights", "positions"):
            # what is not the path's (or, for weights, the prefix's) is as it was
            first = 0 if name == "weights" and n else length
            assert torch.equal(done[name][:, b, :, :first], s[name][:, b, :, :first])
            assert torch.equal(done[name][:, b, :, length + n:], s[name][:, b, :, length + n:])
        if n == 0:
            continue
        k = s["keys"][:, b].index_select(2, slots)
        assert torch.equal(done["keys"][:, b, :, length:length + n], k[:, :, length:])
        v = s["values"][:, b].index_select(2, slots)
        assert torch.equal(done["values"][:, b, :, length:length + n], v[:, :, length:])
        want = torch.arange(seen, seen + n, dtype=torch.int32, device="cuda")
        assert bool((done["positions"][:, b, :, length:length + n] == want).all())
        q = s["q"][:, b, path].double().transpose(1, 2)  # [layers, heads, n, d]
        k = k.double().repeat_interleave(group, 1)
        score = q @ k.transpose(2, 3) * scale
        ds = (d + 2) * 2.0 ** -23 * scale * float((q.abs() @ k.abs().transpose(2, 3)).max())
        p = torch.exp(score - s["lse"][:, b][:, :, path, None].double())
        later = torch.triu(torch.ones(n, length + n, dtype=torch.bool, device="cuda"),
                           diagonal=length + 1)
        p = p.masked_fill(later, 0.0).view(layers, -1, group * n, length + n).sum(2)
        old = s["weights"][:, b, :, :length].double()
        p[:, :, :length] += old
        got = done["weights"][:, b, :, :length + n].double()
        assert bool(((got - p).abs() <= (2 * ds + 2.0 ** -18) * p).all())


@pytest.mark.parametrize("layers,lengths,nodes,steps,heads,kv,d,dtype", [
    (1, (0,), 1, 1, 1, 1, 64, BF16),
    (2, (1, 513, 512), 8, 4, 12, 12, 64, BF16),
    (3, (100, 0, 30, 7), 20, 3, 8, 2, 128, F16),
    (1, (2000, 17), 64, 64, 8, 1, 80, BF16),  # 512 rows
    (1, (33,), 30, 17, 5, 5, 8, F16),
])
def test_accept(layers, lengths, nodes, steps, heads, kv, d, dtype):
    from ppy_b200 import decode

    s = _accept_inputs(layers, lengths, nodes, steps, heads, kv, d, dtype)
    done = {k: v.clone() for k, v in s.items()}
    decode.accept_nodes(**done)
    _check_accept(s, done)


def test_accept_strided_tables_and_rows_only():
    """A token-major cache and tables that are views; no weights: the rows move, nothing else."""
    from ppy_b200 import decode

    s = _accept_inputs(2, (40, 9), 12, 5, 8, 4, 64, BF16)
    for name in ("keys", "values"):
        s[name] = s[name].transpose(2, 3).contiguous().transpose(2, 3)
    wide = torch.zeros(2, 2, 4, 100, device="cuda")
    cap = s["weights"].shape[3]
    wide[..., :cap] = s["weights"]
    wide_positions = torch.zeros(2, 2, 4, 100, dtype=torch.int32, device="cuda")
    wide_positions[..., :cap] = s["positions"]
    done = {k: v.clone(memory_format=torch.preserve_format) for k, v in s.items()}
    done["weights"], done["positions"] = wide[..., :cap], wide_positions[..., :cap]
    decode.accept_nodes(**done)
    _check_accept(s, done)
    assert not wide[..., cap:].any()
    moved = {k: v.clone(memory_format=torch.preserve_format) for k, v in s.items()}
    moved["weights"] = None
    decode.accept_nodes(**moved)
    assert torch.equal(moved["keys"], done["keys"])
    assert torch.equal(moved["values"], done["values"])
    assert torch.equal(moved["positions"], done["positions"])


def test_accept_cuts_a_path_out_of_order():
    from ppy_b200 import decode

    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    s = _accept_inputs(1, (50, 50, 50), 10, 4, 2, 2, 64, BF16)
    s["path"].copy_(torch.tensor([[1, 3, 3, 5], [0, 4, 9, 10], [-1, 2, 3, 4]]))
    s["accepted"].copy_(torch.tensor([4, 4, 4]))
    done = {k: v.clone() for k, v in s.items()}
    decode.accept_nodes(**done, status=status)
    assert int(status) == 2
    s["accepted"].copy_(torch.tensor([2, 3, 0]))  # up to the first step out of order
    _check_accept(s, done)


# ---------------------------------------------------------------- eviction


def _evict_reference(weights, positions, lengths, seen, budget, recent):
    """kept [layers, batch, kv, budget], by sorting each head's entries in Python."""
    kept = torch.full((*weights.shape[:3], budget), -1, dtype=torch.int32)
    w, p = weights.cpu(), positions.cpu()
    for index in torch.cartesian_prod(*(torch.arange(n) for n in weights.shape[:3])).tolist():
        n, last = int(lengths[index[1]]), int(seen[index[1]])
        ws, ps = w[tuple(index)].tolist(), p[tuple(index)].tolist()

        def rank(j):
            if ps[j] >= last - recent:
                return (0, 0.0, j)
            return (2, 0.0, j) if math.isnan(ws[j]) else (1, -ws[j], j)

        if n <= budget:
            kept[tuple(index)][:n] = torch.arange(n)
            continue
        chosen = sorted(sorted(range(n), key=rank)[:budget])
        late = iter(j for j in chosen if j >= budget)
        early = set(j for j in chosen if j < budget)
        kept[tuple(index)] = torch.tensor([j if j in early else next(late)
                                           for j in range(budget)])
    return kept.cuda()


def _evict_inputs(layers, lengths, kv, d, cap, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    batch = len(lengths)
    weights = torch.randn(layers, batch, kv, cap, device="cuda", generator=g).exp()
    weights[weights < 0.6] = 0.0  # many equal ones
    return {"keys": torch.randn(layers, batch, kv, cap, d, device="cuda", generator=g).to(dtype),
            "values": torch.randn(layers, batch, kv, cap, d, device="cuda", generator=g).to(dtype),
            "weights": weights,
            "positions": torch.rand(layers, batch, kv, cap, device="cuda", generator=g).argsort(
                -1).to(torch.int32),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            "seen": torch.full((batch,), cap, dtype=torch.int32, device="cuda")}


def _check_evict(s, done, kept, budget, recent):
    want = _evict_reference(s["weights"], s["positions"], s["lengths"], s["seen"], budget, recent)
    assert torch.equal(kept, want)
    used = want >= 0
    at = want.clamp(min=0).long()
    for name, row in (("keys", True), ("values", True), ("weights", False),
                      ("positions", False)):
        bits = torch.int16 if row else torch.int32  # NaN and the sign of zero count
        old, new = s[name].view(bits), done[name].view(bits)
        index = at[..., None].expand(*at.shape, old.shape[-1]) if row else at
        chosen = old.gather(3, index)
        assert torch.equal(new[:, :, :, :budget][used], chosen[used])
        # slots from the budget on, and behind a short sequence, are as they were
        assert torch.equal(new[:, :, :, budget:], old[:, :, :, budget:])
        assert torch.equal(new[:, :, :, :budget][~used], old[:, :, :, :budget][~used])


@pytest.mark.parametrize("layers,lengths,kv,d,cap,budget,recent,dtype", [
    (1, (10,), 1, 64, 10, 4, 0, BF16),
    (2, (100, 60, 0, 61), 3, 64, 100, 60, 8, BF16),
    (1, (1, 2), 2, 8, 5, 1, 1, F16),
    (2, (3000, 2047), 2, 128, 3001, 1500, 100, F16),
    (1, (5000,), 1, 80, 5000, 4999, 0, BF16),     # one goes
    (1, (4097, 2049), 2, 64, 4100, 1, 0, BF16),   # one stays
    (1, (700,), 2, 64, 700, 300, 700, BF16),      # everything protected: the lowest slots stay
    (1, (40000, 39001), 1, 8, 40000, 30000, 100, BF16),  # several CTAs a head, a tie to cut
    (2, (20000,), 2, 8, 20001, 3000, 0, F16),
    (1, (150000,), 1, 8, 150000, 60000, 7, BF16),  # more entries than shared memory holds
    (300, (900, 512), 1, 8, 900, 511, 9, BF16),    # many heads
])
def test_evict(layers, lengths, kv, d, cap, budget, recent, dtype):
    from ppy_b200 import decode

    s = _evict_inputs(layers, lengths, kv, d, cap, dtype)
    done = {k: v.clone() for k, v in s.items()}
    kept = decode.evict(**done, budget=budget, recent=recent)  # in place
    _check_evict(s, done, kept, budget, recent)
    # into tables of their own, the inputs left alone
    apart = {k: v.clone() for k, v in s.items()}
    outs = {"weights": torch.zeros(layers, len(lengths), kv, budget, device="cuda"),
            "positions": torch.zeros(layers, len(lengths), kv, budget, dtype=torch.int32,
                                     device="cuda")}
    again = decode.evict(**apart, budget=budget, recent=recent, weights_out=outs["weights"],
                         positions_out=outs["positions"])
    assert torch.equal(again, kept) and torch.equal(apart["keys"], done["keys"])
    assert torch.equal(apart["weights"], s["weights"])
    used = kept >= 0
    for name, t in outs.items():
        assert torch.equal(t[used], done[name][..., :budget][used]) and not t[~used].any()


def test_evict_odd_weights():
    """NaN, infinities, both zeros, negative numbers and all-equal heads; a token-major cache."""
    from ppy_b200 import decode

    s = _evict_inputs(1, (400, 380), 3, 64, 400, BF16, seed=4)
    w = s["weights"]
    w[0, 0, 0, ::3] = math.nan
    w[0, 0, 0, 1::7] = math.inf
    w[0, 0, 1] = 0.0
    w[0, 0, 1, ::2] = -0.0
    w[0, 1, 0] = -w[0, 1, 0]
    w[0, 1, 0, 5:50] = -math.inf
    w[0, 1, 1] = math.nan
    w[0, 1, 2] = 1.0
    for name in ("keys", "values"):
        s[name] = s[name].transpose(2, 3).contiguous().transpose(2, 3)
    for budget, recent in ((200, 0), (150, 20), (399, 1)):
        done = {k: v.clone(memory_format=torch.preserve_format) for k, v in s.items()}
        kept = decode.evict(**done, budget=budget, recent=recent)
        _check_evict(s, done, kept, budget, recent)


def test_evict_length_out_of_range():
    from ppy_b200 import decode

    s = _evict_inputs(1, (50, 50), 1, 64, 50, BF16)
    s["lengths"].copy_(torch.tensor([1000, -4]))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    done = {k: v.clone() for k, v in s.items()}
    kept = decode.evict(**done, budget=20, status=status)
    assert int(status) == 2
    s["lengths"].copy_(torch.tensor([50, 0]))
    _check_evict(s, done, kept, 20, 0)


# ---------------------------------------------------------------- together, as GPT-2 decodes


def _near(out, ref, rel=2e-2):
    """The bound of the prompt forward's logits (test_gpu_gpt2.py): bf16 operands throughout."""
    out, ref = out.double(), ref.double()
    assert float((out - ref).abs().max() / ref.abs().max()) <= rel
    assert float((out - ref).norm() / ref.norm()) <= rel


def _restricted_last_logits(model, ids, allowed):
    """Logits of the last token of ids [1, length] in f32, its attention in layer l and head h
    over the positions allowed[l][h] and itself; the other tokens attend to all before them."""
    import torch.nn.functional as F

    cfg = model.config
    length, c, heads, hd = ids.shape[1], cfg.width, cfg.heads, cfg.head_dim
    x = model.wte.float()[ids[0]] + model.wpe.float()[:length]
    causal = torch.ones(length, length, dtype=torch.bool, device="cuda").tril()
    for layer, blk in enumerate(model.blocks):
        hh = F.layer_norm(x, (c,), blk["ln1_g"], blk["ln1_b"], 1e-5)
        q, k, v = F.linear(hh, blk["w_qkv"].float(), blk["b_qkv"]).view(
            length, 3, heads, hd).permute(1, 2, 0, 3)
        seen = causal.expand(heads, length, length).clone()
        seen[:, -1] = False
        for h in range(heads):
            seen[h, -1, allowed[layer][h]] = True
        seen[:, -1, -1] = True
        s = torch.where(seen, q @ k.transpose(1, 2) * hd ** -0.5, -math.inf)
        a = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(length, c)
        x = x + F.linear(a, blk["w_o"].float(), blk["b_o"])
        n = F.layer_norm(x, (c,), blk["ln2_g"], blk["ln2_b"], 1e-5)
        ff = F.gelu(F.linear(n, blk["w_fc"].float(), blk["b_fc"]), approximate="tanh")
        x = x + F.linear(ff, blk["w_proj"].float(), blk["b_proj"])
    n = F.layer_norm(x[-1], (c,), model.lnf_g, model.lnf_b, 1e-5)
    return n @ model.wte.float().t()


def test_gpt2_decodes_with_trees_and_eviction():
    """Prompts of odd lengths into the cache, a tree of drafts verified by its log probabilities,
    the path accepted, the cache cut, the next token: each step's logits against the f32 model."""
    from ppy_b200 import gpt2, scoring

    model = gpt2.GPT2(gpt2.Config(layers=2), seed=3)
    g = torch.Generator(device="cuda").manual_seed(9)
    prompts = [37, 101]
    width = max(prompts)
    ids = torch.randint(0, 50257, (2, width), device="cuda", generator=g)
    cache = model.new_cache(2, capacity=160)
    counts = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    logits = model.extend(cache, ids, counts=counts)
    for b, n in enumerate(prompts):
        _near(logits[b, :n], oracle_gpt2.forward(model, ids[b:b + 1, :n])[0])
    cache.accept(accepted=counts)
    cache.check()
    assert cache.lengths.tolist() == prompts == cache.seen.tolist()
    # every accepted token spread a weight of one over the entries it saw, in each layer and head
    for b, n in enumerate(prompts):
        total = cache.weights[:, b, :, :n].sum(-1)
        assert bool(((total - n).abs() <= 1e-3 * n).all())

    # drafts: two candidates for the next token, continuations of the first
    parents = torch.tensor([-1, -1, 0, 0, 2], dtype=torch.int32, device="cuda")
    draft = torch.randint(0, 50257, (2, 5), device="cuda", generator=g)
    logits = model.extend(cache, draft, parents)
    paths = [[0], [1], [0, 2], [0, 3], [0, 2, 4]]
    history = [ids[b, :n] for b, n in enumerate(prompts)]
    for b in range(2):
        for i, path in enumerate(paths):
            full = torch.cat((history[b], draft[b, path]))[None]
            _near(logits[b, i], oracle_gpt2.forward(model, full)[0, -1])
    scored = scoring.token_logprobs(logits, draft.roll(-1, 1), top=4)
    want = torch.log_softmax(logits.double(), -1)
    assert bool(((scored.logprobs.double()
                  - want.gather(-1, draft.roll(-1, 1)[..., None])[..., 0]).abs() < 1e-4).all())
    assert torch.equal(scored.top_tokens[..., 0], logits.argmax(-1))

    path = torch.tensor([[0, 2, 4], [1, 0, 0]], dtype=torch.int32, device="cuda")
    accepted = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    cache.accept(path, accepted)
    cache.check()
    history = [torch.cat((history[0], draft[0, [0, 2, 4]])), torch.cat((history[1], draft[1, 1:2]))]
    token = torch.randint(0, 50257, (2, 1), device="cuda", generator=g)
    logits = model.extend(cache, token)
    for b in range(2):
        full = torch.cat((history[b], token[b]))[None]
        _near(logits[b, 0], oracle_gpt2.forward(model, full)[0, -1])

    # cut the cache and decode the same token again, over what is left
    cache.pending = None
    cache.evict(32, recent=8)
    assert cache.lengths.tolist() == [32, 32]
    for b in range(2):
        n = len(history[b])
        positions = cache.positions[:, b, :, :32]
        assert bool((positions.sort(-1).values[..., -8:] == torch.arange(
            n - 8, n, device="cuda")).all())  # the recent ones are there
        assert int(positions.max()) == n - 1
    logits = model.extend(cache, token)
    for b in range(2):
        full = torch.cat((history[b], token[b]))[None]
        allowed = [[cache.positions[layer, b, h, :32].long() for h in range(12)]
                   for layer in range(2)]
        _near(logits[b, 0], _restricted_last_logits(model, full, allowed))
    cache.accept()
    cache.check()
    assert cache.lengths.tolist() == [33, 33]


def test_gpt2_extends_in_a_graph():
    """One token a step, captured once: the replays follow the cache as it grows."""
    from ppy_b200 import gpt2, runtime

    model = gpt2.GPT2(gpt2.Config(layers=1), seed=4)
    g = torch.Generator(device="cuda").manual_seed(2)
    prompt = torch.randint(0, 50257, (2, 30), device="cuda", generator=g)
    steps = torch.randint(0, 50257, (2, 4), device="cuda", generator=g)
    stream = torch.cuda.Stream()
    runtime.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            cache = model.new_cache(2, capacity=64)
            token = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
            logits = model.new_logits(2, 1)
            model.extend(cache, prompt)
            cache.accept()
            model.extend(cache, token, logits=logits)  # buffers and launch attributes
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                model.extend(cache, token, logits=logits)
                cache.accept()
            for i in range(4):
                token.copy_(steps[:, i:i + 1])
                graph.replay()
                full = torch.cat((prompt, steps[:, :i + 1]), 1)
                _near(logits[:, 0], oracle_gpt2.forward(model, full)[:, -1])
        stream.synchronize()
        assert cache.lengths.tolist() == [34, 34]
    finally:
        runtime.set_stream(torch.cuda.current_stream())


def test_calls_beside_torchs_stream_from_two_threads():
    """Two threads, each with a torch stream of its own and the library's stream of the thread,
    make and drop their tensors at once: results stay those of one call alone."""
    import threading

    from ppy_b200 import scoring

    x = [Inputs((900, 300), 8, 4, 2, 64, seed=i, spare=40) for i in range(2)]
    logits = [torch.randn(64, 5001, device="cuda",
                          generator=torch.Generator(device="cuda").manual_seed(9 + i))
              for i in range(2)]
    tokens = torch.arange(64, device="cuda")
    want = [(x[i].call(), scoring.token_logprobs(logits[i], tokens, 3)) for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    out, lse = x[i].call()
                    scores = scoring.token_logprobs(logits[i] * 1.0, tokens, 3)
                    junk = torch.full((64, 5001), math.nan, device="cuda")
                    same = (torch.equal(out, want[i][0][0]) and torch.equal(lse, want[i][0][1])
                            and all(torch.equal(a, b) for a, b in zip(scores, want[i][1])))
                    del junk
                    if not same:
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001 - reported below
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
