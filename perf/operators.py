"""The decoding operators as measured work: cases, inputs, a plain form in elementary torch
operations and the framework's own calls, side by side.

    attention   a tree of drafted tokens (a single token is a tree of one node, a prompt piece a
                chain) attends to a cache and to its own ancestors, and is appended to the cache
    accept      the verified path of a tree: its attention weights are added to the cache's
                accumulated ones, its rows move together behind the prefix
    evict       the cache entries of least accumulated weight give way until a budget is met
    logprobs    log probabilities of given tokens with entropy and top alternatives

`own` chooses what `run` does: false, the plain form; true, the calls of `ppy_b200`.
"""

from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
VOCAB, PITCH = 50257, 50272  # GPT-2's vocabulary, and its logits rows on 128-byte lines


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one sequence generates one token with GPT-2's heads and context: the latency of a step
        attention_case("token_gpt2", 1, 1, 12, 12, 64, 1024, 1000, 1000, "bf16"),
        # speculative decoding of a few sequences: trees of up to 24 drafts over ragged caches
        attention_case("tree_gpt2", 4, 24, 12, 12, 64, 1024, 960, 301, "bf16", tree=True,
                       padded=True),
        # a serving batch with shared key heads, one token a sequence, token-major cache
        attention_case("token_batch", 16, 1, 32, 8, 128, 16384, 16001, 2500, "bf16",
                       layout="tokens"),
        # wide trees over long caches with GPT-2's heads
        attention_case("tree_long", 8, 64, 12, 12, 64, 8192, 8000, 4000, "f16", tree=True),
        # a piece of a prompt of odd length behind a long prefix, eight heads on each key head
        attention_case("piece_shared", 2, 250, 16, 2, 128, 20000, 19501, 19501, "bf16"),
        # a step of twelve layers for one sequence: four of eight drafts accepted
        accept_case("accept_gpt2", 12, 1, 8, 4, 12, 12, 64, 1024, 1000, 1000, "bf16"),
        # the same over a batch with long caches
        accept_case("accept_long", 12, 8, 32, 6, 12, 12, 64, 4096, 4000, 1700, "bf16"),
        # GPT-2's cache over its layers, cut to half
        evict_case("evict_gpt2", 12, 4, 12, 64, 1024, 1000, 700, 512, 64, "bf16"),
        # long caches of few heads, cut to a quarter
        evict_case("evict_long", 4, 2, 8, 128, 65536, 65000, 40001, 16384, 1024, "f16"),
        # the logits of one decoding step, with the alternatives a server reports
        logprobs_case("logprobs_step", 4, VOCAB, PITCH, "f32", 1, 5),
        # a scored batch of prompts, rows as the LM head writes them
        logprobs_case("logprobs_prompt", 16384, VOCAB, PITCH, "f32", 1, 5),
        # 16-bit logits of another vocabulary, rows that start anywhere, several tokens asked for
        logprobs_case("logprobs_bf16", 1500, 32011, 32011, "bf16", 3, 20),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("attention", "attention", "accept", "evict", "logprobs"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 12, 25))
    group = rng.choice((1, 1, 2, 4, 8))
    head_dim = rng.choice((64, 64, 128, 80))
    if op == "attention":
        batch, length = log(1, 24), log(1, 16000)
        chain = rng.random() < 0.5
        nodes = 1 if rng.random() < 0.4 else log(2, 250 if chain else 100)
        while batch * kv_heads * length * head_dim > 1.2e8 or (
                batch * kv_heads * group * nodes * length * head_dim > 6e9):
            batch, length = (batch + 1) // 2, (length + 1) // 2
        return attention_case(None, batch, nodes, kv_heads * group, kv_heads, head_dim,
                              length + nodes + rng.randrange(200), length,
                              rng.randrange(length + 1), dtype,
                              layout=rng.choice(("heads", "tokens")),
                              tree=not chain and nodes > 1, padded=rng.random() < 0.5)
    if op == "accept":
        layers, batch, length = rng.choice((1, 2, 6, 12)), log(1, 16), log(8, 8000)
        nodes = log(1, 64)
        while layers * batch * kv_heads * length * head_dim > 1.2e8 or (
                layers * batch * kv_heads * group * nodes * length > 2e8):
            batch, length = (batch + 1) // 2, (length + 1) // 2
        return accept_case(None, layers, batch, nodes, min(nodes, rng.randrange(1, 9)),
                           kv_heads * group, kv_heads, head_dim,
                           length + nodes + rng.randrange(200), length,
                           rng.randrange(length + 1), dtype)
    if op == "evict":
        layers, batch, length = rng.choice((1, 2, 6, 12)), log(1, 16), log(32, 40000)
        while layers * batch * kv_heads * length * head_dim > 2.5e8:
            batch, length = (batch + 1) // 2, (length + 1) // 2
        budget = max(1, int(length * rng.uniform(0.1, 0.95)))
        return evict_case(None, layers, batch, kv_heads, head_dim, length + rng.randrange(100),
                          length, rng.randrange(length + 1), budget, rng.randrange(budget + 1),
                          dtype)
    vocab = rng.choice((VOCAB, log(1000, 130000)))
    kind = rng.choice(("f32", "f32", "bf16", "f16"))
    pitch = rng.choice((vocab, (vocab + 31) // 32 * 32))
    rows = log(1, min(16000, 8e8 / vocab))
    return logprobs_case(None, rows, vocab, pitch, kind, rng.choice((1, 1, 4)),
                         rng.choice((0, 1, 5, 20)))


def attention_case(name, batch, nodes, heads, kv_heads, head_dim, capacity, length, shortest,
                   dtype, layout="heads", tree=False, padded=False):
    return named(name, op="attention", batch=batch, nodes=nodes, heads=heads, kv_heads=kv_heads,
                 head_dim=head_dim, capacity=capacity, length=length, shortest=shortest,
                 dtype=dtype, layout=layout, tree=tree, padded=padded)


def accept_case(name, layers, batch, nodes, steps, heads, kv_heads, head_dim, capacity, length,
                shortest, dtype):
    return named(name, op="accept", layers=layers, batch=batch, nodes=nodes, steps=steps,
                 heads=heads, kv_heads=kv_heads, head_dim=head_dim, capacity=capacity,
                 length=length, shortest=shortest, dtype=dtype)


def evict_case(name, layers, batch, kv_heads, head_dim, capacity, length, shortest, budget,
               recent, dtype):
    return named(name, op="evict", layers=layers, batch=batch, kv_heads=kv_heads,
                 head_dim=head_dim, capacity=capacity, length=length, shortest=shortest,
                 budget=budget, recent=recent, dtype=dtype)


def logprobs_case(name, rows, vocab, pitch, dtype, given, top):
    return named(name, op="logprobs", rows=rows, vocab=vocab, pitch=pitch, dtype=dtype,
                 given=given, top=top)


def named(name, **case):
    return case if name is None else {"name": name, **case}


def spread(low, high, count):
    """`count` whole numbers evenly from low to high (high alone when there is one)."""
    return [high - (high - low) * i // max(1, count - 1) for i in range(count)]


def lengths_of(case):
    return spread(case["shortest"], case["length"], case["batch"])


def counts_of(case):
    nodes = case["nodes"]
    return spread((nodes + 1) // 2, nodes, case["batch"]) if case["padded"] else (
        [nodes] * case["batch"])


def accepted_of(case):
    """Accepted nodes of each sequence: none for the last of several, `steps` for the first."""
    return spread(0 if case["batch"] > 1 else case["steps"], case["steps"], case["batch"])


def work(case):
    op = case["op"]
    if op == "attention":
        d, heads, kv, size = case["head_dim"], case["heads"], case["kv_heads"], 2
        keys = sum(n + c for n, c in zip(lengths_of(case), counts_of(case)))
        new, counts = sum(counts_of(case)), counts_of(case)
        pairs = sum(c * n + c * (c + 1) / (2 if not case["tree"] else 8)
                    for n, c in zip(lengths_of(case), counts))
        moved = 2 * keys * kv * d * size + 2 * new * kv * d * size  # read, and appended
        return {"bytes": moved + 2 * new * heads * d * size + 4 * new * heads,
                "flops": 4 * d * heads * pairs}
    if op == "accept":
        d, heads, kv, size = case["head_dim"], case["heads"], case["kv_heads"], 2
        pairs = list(zip(lengths_of(case), accepted_of(case)))
        keys = sum(n + a for n, a in pairs if a)
        new = sum(a for _, a in pairs)
        one = keys * kv * (d * size + 8) + new * (heads * (d * size + 4) + kv * 3 * d * size)
        return {"bytes": case["layers"] * one,
                "flops": case["layers"] * 2 * d * heads * sum(n * a for n, a in pairs)}
    if op == "evict":
        heads, budget = case["kv_heads"], case["budget"]
        row = case["head_dim"] * 2
        total = 0
        for n in lengths_of(case):
            cut = n > budget
            moved = budget * (n - budget) / n if cut else 0  # survivors behind the budget
            total += heads * (n * 8 + min(n, budget) * 12 + moved * 4 * row)
        return {"bytes": case["layers"] * total, "flops": case["layers"] * sum(
            lengths_of(case)) * heads}
    size = 4 if case["dtype"] == "f32" else 2
    rows, vocab = case["rows"], case["vocab"]
    out = 4 + case["given"] * 12 + case["top"] * 12
    return {"bytes": rows * (vocab * size + out), "flops": 5 * rows * vocab}


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"attention": prepare_attention, "accept": prepare_accept, "evict": prepare_evict,
            "logprobs": prepare_logprobs}[case["op"]](case, g)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(
        dtype)


def shuffled(values, g):
    values = torch.tensor(values, dtype=torch.int32, device="cuda")
    return values[torch.randperm(len(values), generator=g, device="cuda")]


def cache_rows(g, leading, kv_heads, capacity, d, dtype, layout="heads"):
    """Keys or values [*leading, kv_heads, capacity, d], drawn a leading slice at a time."""
    shape = (kv_heads, capacity) if layout == "heads" else (capacity, kv_heads)
    rows = torch.empty(*leading, *shape, d, dtype=dtype, device="cuda")
    flat = rows.view(-1, *shape, d)
    for i in range(flat.shape[0]):
        flat[i].copy_(torch.randn(*shape, d, generator=g, device="cuda"))
    return rows if layout == "heads" else rows.transpose(-3, -2)


def tree_of(g, batch, nodes):
    """Parents of a drafted tree: each node hangs off one of the few nodes before it."""
    index = torch.arange(nodes, device="cuda")
    back = 1 + (torch.rand(batch, nodes, generator=g, device="cuda") ** 2 * 8).long()
    return (index - back).clamp_(min=-1).to(torch.int32)


def prepare_attention(case, g):
    batch, nodes, d = case["batch"], case["nodes"], case["head_dim"]
    heads, kv, dtype = case["heads"], case["kv_heads"], DTYPES[case["dtype"]]
    # as a fused projection leaves them: q, k and v side by side in each token's row
    qkv = normal(g, batch, nodes, (heads + 2 * kv) * d, dtype=dtype)
    q, k, v = qkv.split((heads * d, kv * d, kv * d), dim=-1)
    q.mul_(1.5)  # scores of a trained model: some keys matter much more than others
    layout = case["layout"]
    return {
        "case": case,
        "q": q.view(batch, nodes, heads, d), "k_new": k.view(batch, nodes, kv, d),
        "v_new": v.view(batch, nodes, kv, d),
        "keys": cache_rows(g, (batch,), kv, case["capacity"], d, dtype, layout),
        "values": cache_rows(g, (batch,), kv, case["capacity"], d, dtype, layout),
        "lengths": shuffled(lengths_of(case), g),
        "parents": tree_of(g, batch, nodes) if case["tree"] else None,
        "counts": shuffled(counts_of(case), g) if case["padded"] else None,
        "out": torch.zeros(batch, nodes, heads, d, dtype=dtype, device="cuda"),
        "lse": torch.zeros(batch, heads, nodes, device="cuda"),
    }


def prepare_accept(case, g):
    layers, batch, nodes, d = case["layers"], case["batch"], case["nodes"], case["head_dim"]
    heads, kv, cap, steps = case["heads"], case["kv_heads"], case["capacity"], case["steps"]
    dtype = DTYPES[case["dtype"]]
    lengths = shuffled(lengths_of(case), g)
    q = normal(g, layers, batch, nodes, heads, d, dtype=dtype, scale=1.5)
    keys = cache_rows(g, (layers, batch), kv, cap, d, dtype)
    # the path: `steps` nodes in ascending order, each one's parent the one before it
    path = torch.rand(batch, nodes, generator=g, device="cuda").argsort(1)[:, :steps]
    path = path.sort(1).values.to(torch.int32)
    # the log-sum-exps that the attention left: over the prefix and the node itself
    lse = torch.empty(layers, batch, heads, nodes, device="cuda")
    slot = torch.arange(cap, device="cuda")
    node = torch.arange(nodes, device="cuda")
    for layer in range(layers):
        for b in range(batch):
            s = scores_of(q[layer, b:b + 1], keys[layer, b:b + 1])[0]
            n = lengths[b]
            seen = (slot < n) | (slot == n + node.view(-1, 1))
            lse[layer, b] = s.masked_fill(~seen, -math.inf).logsumexp(-1)
    return {
        "case": case, "q": q, "lse": lse, "keys": keys,
        "values": cache_rows(g, (layers, batch), kv, cap, d, dtype),
        "weights": torch.rand(layers, batch, kv, cap, generator=g, device="cuda"),
        "positions": torch.arange(cap, dtype=torch.int32, device="cuda").expand(
            layers, batch, kv, cap).contiguous(),
        "lengths": lengths, "seen": lengths + 7,
        "path": path.contiguous(), "accepted": shuffled(accepted_of(case), g),
    }


def prepare_evict(case, g):
    layers, batch, kv, cap = case["layers"], case["batch"], case["kv_heads"], case["capacity"]
    d, dtype = case["head_dim"], DTYPES[case["dtype"]]
    # accumulated weights: a few entries gather most, many never had any to speak of (equal ones)
    weights = normal(g, layers, batch, kv, cap, scale=2.0).exp_()
    weights = torch.where(weights < 0.2, torch.zeros_like(weights), weights)
    # entries sit in the order that earlier evictions left
    positions = torch.rand(layers, batch, kv, cap, generator=g, device="cuda").argsort(-1).to(
        torch.int32)
    return {
        "case": case,
        "keys": cache_rows(g, (layers, batch), kv, cap, d, dtype),
        "values": cache_rows(g, (layers, batch), kv, cap, d, dtype),
        "weights": weights, "positions": positions, "lengths": shuffled(lengths_of(case), g),
        "seen": torch.full((batch,), cap, dtype=torch.int32, device="cuda"),
        "weights_out": torch.zeros(layers, batch, kv, case["budget"], device="cuda"),
        "positions_out": torch.zeros(layers, batch, kv, case["budget"], dtype=torch.int32,
                                     device="cuda"),
    }


def prepare_logprobs(case, g):
    rows, vocab, pitch = case["rows"], case["vocab"], case["pitch"]
    logits = torch.empty(rows, pitch, dtype=DTYPES[case["dtype"]], device="cuda")
    # rows of different sharpness, as confident and unsure predictions are
    for at in range(0, rows, 4096):
        part = logits[at:at + 4096]
        sharp = 0.5 + 3 * torch.rand(part.shape[0], 1, generator=g, device="cuda")
        part.copy_(normal(g, *part.shape).mul_(sharp))
    given = torch.randint(0, vocab, (rows, case["given"]), generator=g, device="cuda")
    return {"case": case, "logits": logits[:, :vocab],
            "tokens": given[:, 0].contiguous() if case["given"] == 1 else given}


# ---------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": own_attention, "accept": own_accept, "evict": own_evict,
                "logprobs": own_logprobs}[op](state)
    return {"attention": plain_attention, "accept": plain_accept, "evict": plain_evict,
            "logprobs": plain_logprobs}[op](state)


@functools.cache
def framework():
    """The framework's modules, its launches following torch's stream (once, as at start-up)."""
    from ppy_b200 import decode, runtime, scoring

    runtime.init(torch.cuda.current_device())
    runtime.set_stream(torch.cuda.current_stream())
    return decode, scoring


def own_attention(s):
    out, lse = framework()[0].tree_attention(
        s["q"], s["k_new"], s["v_new"], s["keys"], s["values"], s["lengths"],
        parents=s["parents"], counts=s["counts"], out=s["out"], lse=s["lse"])
    return {"out": out, "lse": lse, "keys": s["keys"], "values": s["values"]}


def own_accept(s):
    framework()[0].accept_nodes(
        s["q"], s["lse"], s["keys"], s["values"], s["weights"], s["positions"], s["lengths"],
        s["seen"], s["path"], s["accepted"])
    return {"keys": s["keys"], "values": s["values"], "weights": s["weights"],
            "positions": s["positions"]}


def own_evict(s):
    kept = framework()[0].evict(
        s["keys"], s["values"], s["weights"], s["positions"], s["lengths"], s["seen"],
        s["case"]["budget"], recent=s["case"]["recent"], weights_out=s["weights_out"],
        positions_out=s["positions_out"])
    return {"keys": s["keys"], "values": s["values"], "weights": s["weights_out"],
            "positions": s["positions_out"], "kept": kept}


def own_logprobs(s):
    return tuple(framework()[1].token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"]))


# ---------------------------------------------------------------- the plain forms


def scores_of(q, keys):
    """q . k / sqrt(d) in f32: q [batch, rows, heads, d], keys [batch, kv_heads, slots, d] to
    [batch, heads, rows, slots]; heads share key heads in order."""
    batch, rows, heads, d = q.shape
    kv = keys.shape[1]
    grouped = q.float().view(batch, rows, kv, heads // kv, d).permute(0, 2, 3, 1, 4)
    s = grouped.reshape(batch, kv, -1, d) @ keys.float().transpose(2, 3)
    return s.view(batch, heads, rows, -1) / math.sqrt(d)


def plain_attention(s):
    q, keys, values, lengths = s["q"], s["keys"], s["values"], s["lengths"].long()
    batch, nodes, heads, d = q.shape
    kv, cap = keys.shape[1], keys.shape[2]
    node = torch.arange(nodes, device="cuda")
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(lengths, nodes)
    real = node < counts[:, None]  # [batch, nodes]
    # append the real nodes behind each sequence's entries
    b, i = real.nonzero(as_tuple=True)
    keys[b, :, lengths[b] + i] = s["k_new"][b, i]
    values[b, :, lengths[b] + i] = s["v_new"][b, i]
    # ancestors, the node itself among them: (I + A)^n > 0 for the parent relation A
    if s["parents"] is None:
        below = (node[:, None] >= node).expand(batch, nodes, nodes)
    else:
        parent = (s["parents"].long()[:, :, None] == node).double()
        below = torch.linalg.matrix_power(parent + torch.eye(nodes, device="cuda"), nodes) > 0
    slot = torch.arange(cap, device="cuda")
    behind = slot - lengths[:, None]  # [batch, cap]: which node a slot holds
    own_slot = behind.clamp(0, nodes - 1)[:, None, :].expand(batch, nodes, cap)
    seen = (behind < 0)[:, None] | ((behind >= 0) & (behind < counts[:, None]))[:, None] & (
        below.gather(2, own_slot))
    seen = seen[:, None]  # [batch, 1, nodes, cap]
    score = torch.where(seen, scores_of(q, keys), -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(real[:, None, :, None], top, 0.0)
    e = torch.exp(score - top)
    z = e.sum(-1, keepdim=True)
    used = (behind < counts[:, None])[:, None, :, None]
    v = torch.where(used, values.float(), 0.0)
    p = (e / z).view(batch, kv, (heads // kv) * nodes, cap)
    out = (p @ v).view(batch, heads, nodes, d).transpose(1, 2)
    s["out"].copy_(torch.where(real[:, :, None, None], out.to(q.dtype), s["out"]))
    s["lse"].copy_(torch.where(real[:, None], (top + z.log())[..., 0], s["lse"]))
    return {"out": s["out"], "lse": s["lse"], "keys": keys, "values": values}


def plain_accept(s):
    keys, values, weights, positions = s["keys"], s["values"], s["weights"], s["positions"]
    layers, batch, nodes, heads, d = s["q"].shape
    kv, cap = keys.shape[2], keys.shape[3]
    path, accepted, lengths = s["path"].long(), s["accepted"].long(), s["lengths"].long()
    steps = path.shape[1]
    step = torch.arange(steps, device="cuda")
    real = step < accepted[:, None]  # [batch, steps]
    b = torch.arange(batch, device="cuda")[:, None]
    # the path's rows of K and V first to where they are going
    from_slot, to_slot = lengths[:, None] + path, lengths[:, None] + step
    bb, tt = real.nonzero(as_tuple=True)
    keys[:, bb, :, to_slot[bb, tt]] = keys[:, bb, :, from_slot[bb, tt]].clone()
    values[:, bb, :, to_slot[bb, tt]] = values[:, bb, :, from_slot[bb, tt]].clone()
    positions[:, bb, :, to_slot[bb, tt]] = (s["seen"][bb] + tt).to(torch.int32)[:, None, None]
    # now step u sees the prefix and the slots up to its own
    q = s["q"][:, b, path].reshape(layers * batch, steps, heads, d)
    lse = s["lse"].permute(0, 1, 3, 2)[:, b, path].permute(0, 1, 3, 2)  # [l, b, heads, steps]
    score = scores_of(q, keys.view(layers * batch, kv, cap, d)).view(
        layers, batch, heads, steps, cap)
    behind = torch.arange(cap, device="cuda") - lengths[:, None]  # [batch, cap]
    seen = (behind[:, None] <= step[:, None]) & real[:, :, None]
    p = torch.where(seen[:, None], torch.exp(score - lse[..., None]), 0.0)
    added = p.view(layers, batch, kv, -1, cap).sum(3)
    old = torch.where((behind < 0)[:, None], weights, 0.0)
    inside = (behind < accepted[:, None])[:, None]
    weights.copy_(torch.where(inside, old + added, weights))
    return {"keys": keys, "values": values, "weights": weights, "positions": positions}


def plain_evict(s):
    keys, values, weights, positions = s["keys"], s["values"], s["weights"], s["positions"]
    cap, d = keys.shape[3], keys.shape[4]
    budget, recent = s["case"]["budget"], s["case"]["recent"]
    lengths = s["lengths"].long()[:, None, None]
    slot = torch.arange(cap, device="cuda")
    inside = slot < lengths
    protected = positions >= s["seen"][:, None, None] - recent
    # rank: protected entries, then by weight, NaN behind every number, then unused slots; the
    # sorts are stable, so ties go to the lowest slot
    by_weight = torch.where(weights.isnan() | protected, 0.0, weights)
    order = by_weight.sort(dim=-1, descending=True, stable=True).indices
    kind = torch.where(protected, 0, torch.where(weights.isnan(), 2, 1))
    kind = torch.where(inside, kind, 3).gather(-1, order)
    order = order.gather(-1, kind.sort(dim=-1, stable=True).indices)
    first = torch.arange(cap, device="cuda") < torch.minimum(lengths, lengths.new_tensor(budget))
    keep = torch.zeros_like(inside.expand_as(order)).scatter(-1, order,
                                                            first.expand_as(order))
    # survivors behind the budget into the holes before it, both in ascending order
    late = (~keep[..., budget:]).to(torch.uint8).sort(dim=-1, stable=True).indices + budget
    hole = ~keep[..., :budget] & inside[..., :budget]
    rank = (hole.long().cumsum(-1) - 1).clamp_(min=0, max=max(0, cap - budget - 1))
    here = slot[:budget].expand_as(rank)
    kept = torch.where(hole, late.gather(-1, rank) if cap > budget else here, here)
    rows = kept[..., None].expand(*kept.shape, d)
    keys[..., :budget, :] = keys.gather(3, rows)
    values[..., :budget, :] = values.gather(3, rows)
    used = inside[..., :budget].expand_as(kept)
    s["weights_out"].copy_(torch.where(used, weights.gather(-1, kept), s["weights_out"]))
    s["positions_out"].copy_(torch.where(used, positions.gather(-1, kept), s["positions_out"]))
    return {"keys": keys, "values": values, "weights": s["weights_out"],
            "positions": s["positions_out"],
            "kept": torch.where(used, kept, -1).to(torch.int32)}


def plain_logprobs(s):
    x, tokens, top = s["logits"].float(), s["tokens"], s["case"]["top"]
    rows, vocab = x.shape
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    log_z = z.log()
    entropy = (log_z + (torch.where(e > 0, m - x, 0.0) * e).sum(1, keepdim=True) / z)[:, 0]
    lse = m + log_z
    logprobs = (x.gather(1, tokens.view(rows, -1)) - m - log_z).view(tokens.shape)
    # values in the order of their bits, the lowest index first among equals
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = order * (1 << 20) + (vocab - 1 - torch.arange(vocab, device="cuda"))
    chosen = vocab - 1 - (key.topk(top, 1).values & ((1 << 20) - 1))
    return logprobs, entropy, x.gather(1, chosen) - lse, chosen


# ---------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": exact_attention, "accept": exact_accept, "evict": exact_evict,
            "logprobs": exact_logprobs}[case["op"]](state)


def ancestors(parents, i):
    found = [i]
    while parents[found[-1]] >= 0:
        found.append(parents[found[-1]])
    return found


def exact_attention(s):
    q, keys, values = s["q"], s["keys"].clone(), s["values"].clone()
    batch, nodes, heads, d = q.shape
    group = heads // keys.shape[1]
    out, lse = s["out"].double(), s["lse"].double()
    parents = ([list(range(-1, nodes - 1))] * batch if s["parents"] is None
               else s["parents"].tolist())
    counts = s["counts"].tolist() if s["counts"] is not None else [nodes] * batch
    for b, length in enumerate(s["lengths"].tolist()):
        n = counts[b]
        end = length + n
        keys[b, :, length:end] = s["k_new"][b, :n].transpose(0, 1)
        values[b, :, length:end] = s["v_new"][b, :n].transpose(0, 1)
        hidden = torch.ones(n, end, dtype=torch.bool)
        hidden[:, :length] = False
        for i in range(n):
            hidden[i, [length + a for a in ancestors(parents[b], i)]] = False
        hidden = hidden.cuda()
        for h in range(heads):
            k, v = keys[b, h // group, :end].double(), values[b, h // group, :end].double()
            score = (q[b, :n, h].double() @ k.t() / d ** 0.5).masked_fill(hidden, -math.inf)
            out[b, :n, h] = torch.softmax(score, 1) @ v
            lse[b, h, :n] = torch.logsumexp(score, 1)
    return {"out": out, "lse": lse, "keys": keys, "values": values}


def exact_accept(s):
    keys, values = s["keys"].clone(), s["values"].clone()
    weights, positions = s["weights"].double(), s["positions"].clone()
    layers, batch, nodes, heads, d = s["q"].shape
    group = heads // keys.shape[2]
    for b in range(batch):
        length, n, seen = (int(s[name][b]) for name in ("lengths", "accepted", "seen"))
        path = s["path"][b, :n].tolist()
        slots = list(range(length)) + [length + p for p in path]
        at = torch.tensor(slots, device="cuda")
        for layer in range(layers):
            if not n:
                continue
            later = torch.triu(torch.ones(n, len(slots), dtype=torch.bool, device="cuda"),
                               diagonal=length + 1)
            k = s["keys"][layer, b].index_select(1, at)  # [kv, slots, d]
            qs = s["q"][layer, b, path].double().transpose(0, 1)  # [heads, n, d]
            k64 = k.double().repeat_interleave(group, 0)
            score = qs @ k64.transpose(1, 2) / d ** 0.5
            p = torch.exp(score - s["lse"][layer, b][:, path, None].double())
            p = p.masked_fill(later, 0.0).sum(1).view(-1, group, len(slots)).sum(1)
            weights[layer, b, :, :length] += p[:, :length]
            weights[layer, b, :, length:length + n] = p[:, length:]
            positions[layer, b, :, length:length + n] = torch.arange(
                seen, seen + n, dtype=torch.int32, device="cuda")
            keys[layer, b, :, length:length + n] = k[:, length:]
            values[layer, b, :, length:length + n] = s["values"][layer, b].index_select(
                1, at)[:, length:]
    return {"keys": keys, "values": values, "weights": weights, "positions": positions}


def exact_evict(s):
    keys, values = s["keys"].clone(), s["values"].clone()
    budget, recent = s["case"]["budget"], s["case"]["recent"]
    layers, batch, kv, cap = s["weights"].shape
    weights, positions = s["weights_out"].double(), s["positions_out"].clone()
    kept_all = torch.full((layers, batch, kv, budget), -1, dtype=torch.int32, device="cuda")
    lengths, seen = s["lengths"].tolist(), s["seen"].tolist()
    for layer in range(layers):
        for b in range(batch):
            n = lengths[b]
            for h in range(kv):
                w = s["weights"][layer, b, h, :n].double()
                pos = s["positions"][layer, b, h, :n]
                w = torch.where(w.isnan(), -1.0, w)  # accumulated weights are not negative
                w = torch.where(pos >= seen[b] - recent, math.inf, w)
                kept = torch.arange(min(n, budget), device="cuda")
                if n > budget:
                    chosen = w.argsort(descending=True, stable=True)[:budget].sort().values
                    early = torch.zeros(budget, dtype=torch.bool, device="cuda")
                    early[chosen[chosen < budget]] = True
                    kept[~early] = chosen[chosen >= budget]
                m = len(kept)
                kept_all[layer, b, h, :m] = kept.to(torch.int32)
                weights[layer, b, h, :m] = s["weights"][layer, b, h][kept].double()
                positions[layer, b, h, :m] = pos[kept]
                keys[layer, b, h, :m] = s["keys"][layer, b, h].index_select(0, kept)
                values[layer, b, h, :m] = s["values"][layer, b, h].index_select(0, kept)
    return {"keys": keys, "values": values, "weights": weights, "positions": positions,
            "kept": kept_all}


def exact_logprobs(s):
    logits, tokens, top = s["logits"], s["tokens"], s["case"]["top"]
    parts = []
    for at in range(0, logits.shape[0], 512):
        x = logits[at:at + 512].double()
        logp = torch.log_softmax(x, 1)
        given = logp.gather(1, tokens[at:at + 512].view(len(x), -1))
        entropy = -(logp.exp() * logp).sum(1)
        order = x.sort(dim=1, descending=True, stable=True).indices[:, :top]
        parts.append((given, entropy, logp.gather(1, order), order))
    given, entropy, alternatives, chosen = (torch.cat(p) for p in zip(*parts))
    return given.view(tokens.shape), entropy, alternatives, chosen
