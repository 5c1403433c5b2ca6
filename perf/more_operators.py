"""Operators of drafted decoding over the paged 4-bit cache, as cases that can be timed and compared.

A server drafts a few tokens for every sequence, as a chain or a tree, runs them through the model at once and
keeps those that the model agrees with.  Four kinds, each through the entry points that a program calls:

* ``append`` -- ``int4_append_rope``: keys rotated to their positions and quantised into their pages with the
  values, queries rotated beside them (and ``int4_gather``, which reads the stored values back);
* ``tree``   -- ``int4_tree_attention``: the nodes of every sequence's tree against its pages;
* ``verify`` -- ``verify_drafts``: which nodes the target model accepts, and the token behind them;
* ``keep``   -- ``int4_keep``: the accepted tokens moved together in every layer's pages.

``run`` computes them in plain torch where ``own`` is false, and calls the framework where it is true.  Shapes are the
Llama-3.1-8B layer's (32 query heads, 8 KV heads, 128 channels, 128256 tokens) unless a case says otherwise; keys have
per-channel scales with a few outlier channels, values are N(0, 1).
"""

import math
import random

import torch

own = False

D = 128
GROUP = 32  # channels that share a scale and a lowest value
MOST = 64   # nodes of a tree
DEVICE = "cuda"
SCALING = D ** -0.5
THETA = 500000.0


def listed():
    return [
        # a decode step's tokens, each in the middle of a page; latency
        {"name": "append_32x1", "kind": "append", "seqs": 32, "short": 1, "long": 1, "context": 8000, "kv": 8,
         "gqa": 4, "page": 64, "rotary": 128, "interleaved": False, "depths": False},
        # trees of drafts: positions by depth, half of the channels rotated
        {"name": "append_32x5_40_depths", "kind": "append", "seqs": 32, "short": 5, "long": 40, "context": 8000,
         "kv": 8, "gqa": 4, "page": 64, "rotary": 64, "interleaved": False, "depths": True},
        # prompts of a batch, ragged, neighbouring channels paired
        {"name": "append_16x500_8192", "kind": "append", "seqs": 16, "short": 500, "long": 8192, "context": 0,
         "kv": 8, "gqa": 4, "page": 64, "rotary": 128, "interleaved": True, "depths": False},
        # one conversation with a small tree; latency and launches
        {"name": "tree_1x1000_8", "kind": "tree", "seqs": 1, "short": 1000, "long": 1000, "least": 8, "nodes": 8,
         "kv": 8, "gqa": 4, "page": 64},
        # a full serving batch around the 8K context, trees of up to 16 nodes
        {"name": "tree_32x2000_8192_16", "kind": "tree", "seqs": 32, "short": 2000, "long": 8192, "least": 5,
         "nodes": 16, "kv": 8, "gqa": 4, "page": 64},
        # a few very different lengths and trees, eight query heads to a KV head, wide pages
        {"name": "tree_5x17_65001_1_61_gqa8", "kind": "tree", "seqs": 5, "short": 17, "long": 65001, "least": 1,
         "nodes": 61, "kv": 4, "gqa": 8, "page": 256},
        # the widest trees over a full batch: the most arithmetic
        {"name": "tree_32x8192_64", "kind": "tree", "seqs": 32, "short": 8192, "long": 8192, "least": 64,
         "nodes": 64, "kv": 8, "gqa": 4, "page": 64},
        # one conversation, children that a draft head proposed
        {"name": "verify_1x8", "kind": "verify", "seqs": 1, "least": 8, "nodes": 8, "vocab": 128256,
         "drawn": False, "temperature": 0.8},
        # chains that a draft model has drawn, with its probabilities; a smaller, odd vocabulary
        {"name": "verify_32x6_drawn", "kind": "verify", "seqs": 32, "least": 6, "nodes": 6, "vocab": 32003,
         "drawn": True, "temperature": 1.0},
        # greedy decoding with trees of all sizes
        {"name": "verify_24x1_64_greedy", "kind": "verify", "seqs": 24, "least": 1, "nodes": 64, "vocab": 128256,
         "drawn": False, "temperature": 0.0},
        # one conversation's accepted tokens, 32 layers
        {"name": "keep_1x8", "kind": "keep", "layers": 32, "seqs": 1, "least": 8, "nodes": 8, "context": 900,
         "kv": 8, "page": 64},
        # a full batch of wide trees, 32 layers
        {"name": "keep_32x10_64", "kind": "keep", "layers": 32, "seqs": 32, "least": 10, "nodes": 64, "context": 300,
         "kv": 8, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append"] * 3 + ["tree"] * 5 + ["verify"] * 4 + ["keep"])
    kv, gqa = rng.choice([1, 2, 4, 8, 8, 8]), rng.choice([1, 2, 3, 4, 4, 4, 7, 8])
    page = rng.choice([32, 64, 64, 128, 256])
    if kind == "append":
        drafts = rng.random() < 0.5
        long = _log(rng, 1, MOST) if drafts else _log(rng, 1, 8192)
        seqs = _log(rng, 1, max(1, min(32, 8 * 8192 // long)))
        return {"kind": kind, "seqs": seqs, "short": max(1, long // rng.choice([1, 10])), "long": long,
                "context": rng.randint(1, 20000) if drafts else rng.choice([0, rng.randint(1, 3000)]), "kv": kv,
                "gqa": min(gqa, 4), "page": page, "rotary": rng.choice([16, 32, 64, 96, 128, 128, 128]),
                "interleaved": rng.random() < 0.4, "depths": drafts}
    if kind == "tree":
        long = _log(rng, 20, 65536)
        seqs = _log(rng, 1, max(1, min(64, 16 * 8192 // long)))
        nodes = _log(rng, 1, MOST)
        return {"kind": kind, "seqs": seqs, "short": max(0, long // rng.choice([1, 3, 100]) - rng.randint(0, 1)),
                "long": long, "least": max(1, nodes // rng.choice([1, 2, 20])), "nodes": nodes, "kv": kv, "gqa": gqa,
                "page": page}
    nodes = _log(rng, 1, MOST)
    seqs = _log(rng, 1, max(1, min(32, 320 // nodes)))
    least = max(1, nodes // rng.choice([1, 2, 20]))
    if kind == "verify":
        return {"kind": kind, "seqs": seqs, "least": least, "nodes": nodes, "vocab": _log(rng, 1000, 128256),
                "drawn": rng.random() < 0.4, "temperature": rng.choice([0.0, 0.0, 0.6, 1.0, 1.0, 1.3])}
    return {"kind": kind, "layers": rng.choice([1, 16, 32]), "seqs": seqs, "least": least, "nodes": nodes,
            "context": rng.randint(0, 300), "kv": kv, "page": rng.choice([32, 64])}


# -- sizes and trees, on the host ----------------------------------------------------------------------

def _spread(rng, count, low, high):
    """``count`` numbers over the logarithm of the range, one of them the largest."""
    out = [_log(rng, max(low, 1), max(high, 1)) if high > 0 else 0 for _ in range(count)]
    if low == 0 and count > 1:
        out[rng.randrange(count)] = 0
    out[rng.randrange(count)] = high
    return out


def _new(case):
    """Tokens that each sequence gets: a prompt's, or the nodes of its tree."""
    low, high = ("short", "long") if case["kind"] == "append" else ("least", "nodes")
    return _spread(random.Random(f"new {case['seqs']} {case[low]} {case[high]}"), case["seqs"], case[low], case[high])


def _contexts(case):
    """Tokens that each sequence holds before them."""
    if case["kind"] == "tree":
        rng = random.Random(f"context {case['seqs']} {case['short']} {case['long']}")
        return _spread(rng, case["seqs"], case["short"], case["long"])
    c = case.get("context", 0)
    rng = random.Random(f"context {c} {case['seqs']}")
    return [rng.randint((c + 1) // 2, c) for _ in range(case["seqs"])]


def _sums(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _tree(rng, n):
    """Parents of a tree's nodes, parents first: mostly the main branch and its neighbours."""
    return [-1] + [rng.randint(max(0, i - rng.choice([1, 2, 5])), i - 1) for i in range(1, n)]


def _trees(case, seed):
    rng = random.Random(f"tree {seed}")
    if case.get("drawn"):  # a draft model's chain
        return [[i - 1 for i in range(n)] for n in _new(case)]
    return [_tree(rng, n) for n in _new(case)]


def _seen(parents):
    """The mask of every node: its ancestors and itself, node j as bit j."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else 0) | 1 << i)
    return out


def _signed(mask):
    return mask - (1 << 64) if mask >> 63 else mask


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


# -- inputs --------------------------------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, device=DEVICE, generator=gen)


def _keys_values(gen, n, kv):
    """Keys N(0, 1) with log-normal channel scales and four outlier channels per head; values N(0, 1)."""
    scale = torch.exp(_normal(gen, 1, kv, D))
    outlier = torch.rand(1, kv, D, device=DEVICE, generator=gen).argsort(-1) < 4
    scale = torch.where(outlier, scale * 10.0, scale)
    k = torch.empty(n, kv, D, device=DEVICE, dtype=torch.float16)
    v = torch.empty_like(k)
    for r0 in range(0, n, 65536):
        rows = min(n, r0 + 65536) - r0
        k[r0: r0 + rows] = (_normal(gen, rows, kv, D) * scale).half()
        v[r0: r0 + rows] = _normal(gen, rows, kv, D).half()
    return k, v


def _rows_inputs(case, gen, seed):
    """append: the fused projection of the new tokens, their positions, and the rotation's tables."""
    new, have, kv = _new(case), _contexts(case), case["kv"]
    heads = kv * case["gqa"]
    k, v = _keys_values(gen, sum(new), kv)
    q = _normal(gen, sum(new), heads, D).half()
    qkv = torch.cat([x.flatten(1) for x in (q, k, v)], dim=1)  # as the projection of a layer gives it
    rng = random.Random(f"depth {seed}")
    positions = []
    for n, c in zip(new, have):
        depth = [bin(m).count("1") - 1 for m in _seen(_tree(rng, n))] if case["depths"] else range(n)
        positions += [c + d for d in depth]
    half = case["rotary"] // 2
    inv = THETA ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
    angle = torch.arange(max(positions) + 1, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return {"new": new, "have": have, "qkv": qkv, "positions": _int32(positions), "cos": angle.cos().float(),
            "sin": angle.sin().float()}


def _split(case, qkv):
    """q, k and v of the fused projection, as views of it."""
    kv = case["kv"]
    heads = kv * case["gqa"]
    rows = qkv.view(qkv.shape[0], heads + 2 * kv, D)
    return rows[:, :heads], rows[:, heads: heads + kv], rows[:, heads + kv:]


def _verify_inputs(case, gen, seed):
    """Target logits with a few likely tokens at every node; the drafts are mostly among them."""
    new, vocab = _new(case), case["vocab"]
    parents = _trees(case, seed)
    starts, total = _sums(new), sum(new)
    likely = torch.randint(vocab, (total, 1), device=DEVICE, generator=gen)
    likely = (likely + torch.arange(8, device=DEVICE) * (vocab // 8)) % vocab  # eight different ones
    boost = math.log(vocab) + 5.0 * torch.rand(total, 8, device=DEVICE, generator=gen).sort(-1, descending=True).values
    logits = torch.empty(total, vocab, dtype=torch.float16, device=DEVICE)
    for r0 in range(0, total, 256):
        part = 2.0 * _normal(gen, min(total, r0 + 256) - r0, vocab)
        logits[r0: r0 + 256] = part.scatter(1, likely[r0: r0 + 256], boost[r0: r0 + 256]).half()
    out = {"new": new, "tree": parents, "logits": logits,
           "accept": torch.rand(total, device=DEVICE, generator=gen),
           "sample": torch.rand(case["seqs"], device=DEVICE, generator=gen)}
    above = [starts[s] + max(p, 0) for s, row in enumerate(parents) for p in row]  # the row before every node
    above = torch.tensor(above, device=DEVICE)
    if case["drawn"]:  # the draft model's logits are near the target's
        scale = 1.0 / max(case["temperature"], 0.5)
        out["draft"] = torch.empty(total, vocab, device=DEVICE)
        for r0 in range(0, total, 256):
            rows = above[r0: r0 + 256]
            near = logits[rows].float() + 0.7 * _normal(gen, rows.shape[0], vocab)
            out["draft"][r0: r0 + 256] = torch.softmax(near * scale, -1)
        out["tokens"] = torch.multinomial(out["draft"], 1, generator=gen)[:, 0]
    else:  # siblings are different tokens
        rank, count = [], {}
        for s, row in enumerate(parents):
            for p in row:
                rank.append(count.get((s, p), 0))
                count[s, p] = rank[-1] + 1
        rank = torch.tensor(rank, device=DEVICE)
        other = torch.randint(vocab, (total,), device=DEVICE, generator=gen)
        out["tokens"] = torch.where(rank < 8, likely[above, rank.clamp(max=7)], other)
    return out


def _paths(new):
    """Accepted nodes of every tree: the main branch for a while, then nodes further on (from behind where they go,
    so that a second pass over the same pages changes nothing)."""
    rng = random.Random(f"path {new}")
    out = []
    for n in new:
        count = rng.randint(1, min(n, 9))
        first = rng.randint(1, count)
        rest = min(count - first, max(n - count, 0))
        out.append(list(range(first)) + sorted(rng.sample(range(count, n), rest)) if rest else list(range(first)))
    return out


def _inputs(case, seed):
    """The tensors of a case, from the seed alone: what ``prepare`` lays out and ``exact`` starts from."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "append":
        return _rows_inputs(case, gen, seed)
    if case["kind"] == "verify":
        return _verify_inputs(case, gen, seed)
    new, have, kv = _new(case), _contexts(case), case["kv"]
    if case["kind"] == "keep":
        tokens = [-(-(a + b) // case["page"]) for a, b in zip(new, have)]
        shape = (case["layers"], sum(tokens) + 2, kv, case["page"] * 160)
        return {"new": new, "have": have, "paths": _paths(new),
                "pool": torch.randint(256, shape, dtype=torch.uint8, device=DEVICE, generator=gen)}
    k, v = _keys_values(gen, sum(new) + sum(have), kv)
    return {"new": new, "have": have, "k": k, "v": v, "q": _normal(gen, sum(new), kv * case["gqa"], D).half(),
            "seen": [m for row in _trees(case, seed) for m in _seen(row)]}


def _page_table(case, lengths, seed):
    """Pages of every sequence in no order, as a pool that has been in use hands them out; -1 behind the last."""
    page = case["page"]
    counts = [-(-n // page) for n in lengths]
    ids = list(range(sum(counts) + 2))
    random.Random(seed).shuffle(ids)
    rows, at = [], 0
    for n in counts:
        rows.append(ids[at: at + n] + [-1] * (max(counts) - n))
        at += n
    return _int32(rows), len(ids)


def _slots(table, page, starts, lengths):
    """The pool's token slot of every packed row."""
    out = []
    for b, (s, n) in enumerate(zip(starts, lengths)):
        pos = torch.arange(s, s + n, device=DEVICE)
        out.append(table[b, pos // page].long() * page + pos % page)
    return torch.cat(out)


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    kind = case["kind"]
    if kind == "verify":
        state["offsets"] = _int32(_sums(state["new"]))
        state["parents"] = _int32([p for row in state["tree"] for p in row])
        return state
    starts = state["have"]
    ends = [a + b for a, b in zip(starts, state["new"])]
    state["table"], pages = _page_table(case, ends, seed)
    state["starts"], state["offsets"] = _int32(starts), _int32(_sums(state["new"]))
    if kind == "keep":
        width = max(state["new"])
        state["path"] = _int32([row + [-1] * (width - len(row)) for row in state["paths"]])
        state["counts"] = _int32([len(row) for row in state["paths"]])
        return state
    if kind == "tree":
        state["lengths"] = _int32(ends)
        state["seen"] = torch.tensor([_signed(m) for m in state["seen"]], dtype=torch.int64, device=DEVICE)
    if own:
        from reskv_amd.int4 import empty_pages, int4_append

        state["pool"] = empty_pages(pages, case["kv"], case["page"], device=DEVICE)
        if kind == "tree":
            int4_append(state["pool"], state["table"], torch.zeros_like(state["starts"]), state["k"], state["v"],
                        _int32(_sums(ends)))
    elif kind == "tree":
        state["cache"] = [_quantise(state["k"]), _quantise(state["v"])]
    else:
        rows = (pages * case["page"], case["kv"], D // GROUP)
        state["cache"] = [(torch.zeros(*rows, GROUP, dtype=torch.uint8, device=DEVICE),
                           torch.zeros(*rows, 1, dtype=torch.float16, device=DEVICE),
                           torch.zeros(*rows, 1, dtype=torch.float16, device=DEVICE)) for _ in range(2)]
        state["slots"] = _slots(state["table"], case["page"], starts, state["new"])
    if kind == "tree":
        del state["k"], state["v"]
    return state


# -- the plain forms -----------------------------------------------------------------------------------

def _quantise(x):
    """(codes, scale, low) of rows [N, heads, 128]: 4 bits over the range of each group of 32 channels.
    In 64 bits, as a quotient next to a half decides between two codes."""
    parts = []
    for r0 in range(0, x.shape[0], 65536):
        xd = x[r0: r0 + 65536].double().unflatten(-1, (D // GROUP, GROUP))
        low = xd.amin(-1, keepdim=True)
        scale = ((xd.amax(-1, keepdim=True) - low) / 15.0).half()
        step = scale.double()
        codes = torch.where(step > 0, ((xd - low) / step).round().clamp(0, 15), torch.zeros_like(xd))
        parts.append((codes.to(torch.uint8), scale, low.half()))
    return parts[0] if len(parts) == 1 else tuple(torch.cat(part) for part in zip(*parts))


def _values(codes, scale, low):
    """fp32 rows [N, heads, 128] that the codes stand for."""
    return (codes.float() * scale.float() + low.float()).flatten(-2)


def _rotated(x, cos, sin, interleaved):
    """fp16 rows [N, heads, 128] of x with their first 2 * cos.shape[-1] channels rotated; cos and sin [N, half]."""
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    xf = x.float()
    if interleaved:
        a, b = xf[..., 0: 2 * half: 2], xf[..., 1: 2 * half: 2]
        turned = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = xf[..., :half], xf[..., half: 2 * half]
        turned = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return torch.cat((turned, xf[..., 2 * half:]), dim=-1).half()


def _run_append(state):
    case = state["case"]
    q, k, v = _split(case, state["qkv"])
    rows = state["positions"].long()
    cos, sin = state["cos"][rows], state["sin"][rows]
    at = state["slots"]
    out = [_rotated(q, cos, sin, case["interleaved"])]
    for x, cache in zip((_rotated(k, cos, sin, case["interleaved"]), v), state["cache"]):
        for part, held in zip(_quantise(x), cache):
            held[at] = part
        out.append(_values(*(held[at] for held in cache)).half())
    return tuple(out)


def _run_tree(state):
    case = state["case"]
    kv, gqa = case["kv"], case["gqa"]
    q, seen = state["q"], state["seen"]
    out = torch.empty_like(q)
    at = first = 0
    for n, have in zip(state["new"], state["have"]):
        m = have + n
        k, v = (_values(*(part[at: at + m] for part in cache)).transpose(0, 1) for cache in state["cache"])
        rows = q[first: first + n].float().view(n, kv, gqa, D).permute(1, 2, 0, 3).reshape(kv, gqa * n, D)
        score = torch.matmul(rows, k.transpose(1, 2).contiguous()).view(kv, gqa, n, m) * SCALING
        bits = seen[first: first + n, None] >> torch.arange(n, device=DEVICE) & 1
        score[..., have:].masked_fill_(bits == 0, -math.inf)
        top = score.amax(-1, keepdim=True)
        score.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
        total = score.sum(-1, keepdim=True)
        res = torch.matmul(score.view(kv, -1, m), v.contiguous()).view(kv, gqa, n, D)
        res = torch.where(total > 0, res / total, torch.zeros_like(res))
        out[first: first + n] = res.permute(2, 0, 1, 3).reshape(n, kv * gqa, D).half()
        at, first = at + m, first + n
    return out


def _run_verify(state):
    """All sequences at once, node after node: a node is looked at when its parent is the node reached so far.  In
    64 bits, as a probability next to a random number decides."""
    case = state["case"]
    seqs, most, hot = case["seqs"], max(state["new"]), case["temperature"]
    offsets = state["offsets"].long()
    first, counts = offsets[:-1], offsets.diff()
    logits = state["logits"]
    index = torch.arange(logits.shape[1], device=DEVICE)

    def target(rows):
        x = logits[rows].double()
        if hot == 0.0:  # all of it at the largest, the lowest of equals
            best = torch.where(x == x.amax(-1, keepdim=True), index, index[-1]).amin(-1, keepdim=True)
            return torch.zeros_like(x).scatter_(1, best, 1.0)
        x = x / hot
        x = (x - x.amax(-1, keepdim=True)).exp()
        return x / x.sum(-1, keepdim=True)

    here = torch.zeros(seqs, dtype=torch.int64, device=DEVICE)
    path = torch.full((seqs, MOST), -1, dtype=torch.int32, device=DEVICE)
    path[:, 0] = 0
    length = torch.ones(seqs, dtype=torch.int64, device=DEVICE)
    left = target(first)
    for i in range(1, most):
        row = first + torch.where(i < counts, i, 0)
        token = state["tokens"][row][:, None]
        asked = (i < counts) & (state["parents"][row] == here)
        total = left.sum(-1, keepdim=True)
        if case["drawn"]:
            drawn = state["draft"][row].double()
        else:
            drawn = torch.zeros_like(left).scatter_(1, token, 1.0)
        if hot == 0.0:
            took = asked & (left.gather(1, token)[:, 0] > 0)
            less = left
        else:
            chance = left.gather(1, token) / total
            took = asked & (state["accept"][row].double() * drawn.gather(1, token)[:, 0] < chance[:, 0])
            less = (left / total - drawn).clamp(min=0) if case["drawn"] else left.scatter(1, token, 0.0)
            less = torch.where(less.sum(-1, keepdim=True) > 0, less, left)
        left = torch.where(asked[:, None], less, left)
        left = torch.where(took[:, None], target(row), left)
        here = torch.where(took, i, here)
        path.scatter_(1, torch.where(took, length, 0)[:, None], torch.where(took, i, 0)[:, None].int())
        length = length + took
    if hot == 0.0:
        token = left.argmax(-1)
    else:
        run = left.cumsum(-1)
        token = (run <= state["sample"].double()[:, None] * run[:, -1:]).sum(-1).clamp(max=logits.shape[1] - 1)
    return path, length.int(), token


def _nibbles(e):
    """Byte of a dword and shift that hold the nibble of its element e."""
    bit = 4 * (e // 2 + 4 * (e % 2))
    return bit // 8, bit % 8


def _run_keep(state):
    """On the bytes of the pool, in their documented order: a block of 32 tokens of a head holds K's codes [2, 4, 16
    tokens, 16 bytes], its scalings [2, 4, 16 tokens, 4 bytes], V's codes [2, 4 times 8 tokens, 16, 4, 8 nibbles], V's
    scales and lowest values [4, 32 tokens, 2 bytes] each."""
    case, page = state["case"], state["case"]["page"]
    pool = state["pool"]
    blocks = pool.view(*pool.shape[:3], page // 32, 5120)
    keys = blocks[..., :2048].unflatten(-1, (2, 4, 16, 16))
    scales = blocks[..., 2048:2560].unflatten(-1, (2, 4, 16, 4))
    values = blocks[..., 2560:4608].unflatten(-1, (2, 4, 16, 4, 4))
    rest = blocks[..., 4608:].unflatten(-1, (8, 32, 2))
    path, counts, starts = state["path"].long(), state["counts"].long(), state["starts"].long()
    seqs, width = path.shape
    j = torch.arange(width, device=DEVICE)[None]
    kept = j < counts[:, None]
    source = starts[:, None] + torch.where(kept, path, torch.zeros_like(path))
    target = starts[:, None] + torch.where(kept, j, torch.zeros_like(j))  # the rest: the root to itself
    source = torch.where(kept, source, target)

    def place(t):
        return torch.gather(state["table"].long(), 1, t // page), t % page // 32, t % 32

    p, b, t = place(source)
    byte = torch.tensor([_nibbles(e)[0] for e in range(8)], device=DEVICE)
    shift = torch.tensor([_nibbles(e)[1] for e in range(8)], device=DEVICE, dtype=torch.uint8)
    moved = [keys[:, p, :, b, t // 16, :, t % 16], scales[:, p, :, b, t // 16, :, t % 16], rest[:, p, :, b, :, t]]
    codes = values[:, p, :, b, :, t // 8, :, :, byte[t % 8]] >> shift[t % 8][..., None, None, None, None, None] & 15
    for i in range(width):  # one token of every sequence after the other, as neighbours share bytes
        p, b, t = place(target[:, i: i + 1])
        p, b, t = p[:, 0], b[:, 0], t[:, 0]
        keys[:, p, :, b, t // 16, :, t % 16] = moved[0][:, i]
        scales[:, p, :, b, t // 16, :, t % 16] = moved[1][:, i]
        rest[:, p, :, b, :, t] = moved[2][:, i]
        by = shift[t % 8][:, None, None, None, None, None]
        old = values[:, p, :, b, :, t // 8, :, :, byte[t % 8]]
        values[:, p, :, b, :, t // 8, :, :, byte[t % 8]] = old & ~(15 << by) | codes[:, i] << by
    return pool


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"append": _run_append, "tree": _run_tree, "verify": _run_verify, "keep": _run_keep}[kind](state)
    from reskv_amd.drafts import verify_drafts
    from reskv_amd.int4 import int4_append_rope, int4_gather, int4_keep, int4_tree_attention

    if kind == "append":
        q, k, v = _split(case, state["qkv"])
        turned = int4_append_rope(state["pool"], state["table"], state["starts"], q, k, v, state["cos"], state["sin"],
                                  state["offsets"], positions=state["positions"] if case["depths"] else None,
                                  interleaved=case["interleaved"])
        return (turned, *int4_gather(state["pool"], state["table"], state["starts"], state["offsets"], q.shape[0]))
    if kind == "tree":
        return int4_tree_attention(state["q"], state["pool"], state["table"], state["lengths"], state["offsets"],
                                   state["seen"], max_nodes=case["nodes"],
                                   max_length=max(a + b for a, b in zip(state["new"], state["have"])))
    if kind == "verify":
        return verify_drafts(state["logits"], state["tokens"], state["parents"], state["offsets"], state["accept"],
                             state["sample"], draft=state.get("draft"), temperature=case["temperature"])
    int4_keep(state["pool"], state["table"], state["starts"], state["path"], state["counts"])
    return state["pool"]


def work(case):
    kind, new = case["kind"], _new(case)
    total = sum(new)
    if kind == "verify":
        # the target's logits once; of the draft's rows the one that a sequence turns down
        drawn = case["seqs"] * case["vocab"] * 4 if case["drawn"] and case["temperature"] > 0 else 0
        return {"bytes": total * case["vocab"] * 2 + drawn + total * 16, "flops": 0}
    have, kv = _contexts(case), case["kv"]
    if kind == "append":
        # rows in, queries and codes out, codes in again, rows out
        heads = kv * case["gqa"]
        return {"bytes": total * (heads * 512 + kv * (512 + 160 + 160 + 512) + case["rotary"] * 4), "flops": 0}
    if kind == "keep":
        paths = _paths(new)
        moved = sum(i != j for row in paths for j, i in enumerate(row))
        return {"bytes": 2 * 160 * case["layers"] * kv * moved + 4 * sum(len(row) + 1 for row in paths), "flops": 0}
    heads = kv * case["gqa"]
    return {"bytes": (total + sum(have)) * kv * 160 + 2 * total * heads * D * 2,
            "flops": 4 * D * heads * sum(n * h + n * (n + 1) // 2 for n, h in zip(new, have))}


# -- the definitions, in 64 bits -----------------------------------------------------------------------

def _exact_values(x):
    """What 4 bits hold of rows [N, heads, 128], in 64 bits from the definition."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    step = ((high - low) / 15).half().double()
    code = torch.round((g - low) / torch.where(step == 0, torch.ones_like(step), step)).clamp(max=15)
    return torch.where(step == 0, low, low + step * code).reshape(x.shape)


def _exact_turn(x, angles, interleaved):
    """Rows in 64 bits as complex numbers times exp(i angle), the cache's rounding to fp16 left out."""
    half = angles.shape[1]
    x = x.double()
    pair = x[..., : 2 * half].unflatten(-1, (half, 2) if interleaved else (2, half))
    if not interleaved:
        pair = pair.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(angles), angles)[:, None])
    if not interleaved:
        turned = turned.transpose(-1, -2)
    return torch.cat((turned.flatten(-2), x[..., 2 * half:]), -1)


def _exact_append(case, x):
    q, k, v = _split(case, x["qkv"])
    half = case["rotary"] // 2
    inv = torch.exp(torch.arange(half, device=DEVICE, dtype=torch.float64) * (-math.log(THETA) / half))
    angles = x["positions"].double()[:, None] * inv
    turned = _exact_turn(k, angles, case["interleaved"]).half()  # what is quantised is an fp16 row
    return _exact_turn(q, angles, case["interleaved"]), _exact_values(turned), _exact_values(v)


def _exact_tree(case, x):
    q, out = x["q"], torch.zeros(x["q"].shape, dtype=torch.float64, device=DEVICE)
    at = row = 0
    for n, have in zip(x["new"], x["have"]):
        k, v = (_exact_values(y[at: at + have + n]) for y in (x["k"], x["v"]))
        visible = torch.ones(n, have + n, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                visible[i, have + j] = x["seen"][row + i] >> j & 1 == 1
        visible = visible.to(DEVICE)
        for h in range(q.shape[1]):
            kh, vh = k[:, h // case["gqa"]], v[:, h // case["gqa"]]
            dots = (q[row: row + n, h].double() @ kh.t()) / math.sqrt(D)
            dots = torch.where(visible, dots, torch.full_like(dots, -math.inf))
            out[row: row + n, h] = torch.exp(dots - torch.logsumexp(dots, -1, keepdim=True)) @ vh
        at, row = at + have + n, row + n
    return out


def _exact_verify(case, x):
    """Sequence by sequence down the tree, over lists of children."""
    paths, lengths, tokens = [], [], []
    accept, sample, token = x["accept"].double().tolist(), x["sample"].double().tolist(), x["tokens"].tolist()
    for s, (first, tree) in enumerate(zip(_sums(x["new"]), x["tree"])):
        node, path = 0, [0]
        while True:
            logits = x["logits"][first + node].double()
            children = [i for i, p in enumerate(tree) if p == node and i > node]
            if case["temperature"] == 0.0:
                best = int((logits == logits.max()).nonzero()[0])
                reached = [i for i in children if token[first + i] == best][:1]
            else:
                r = torch.softmax(logits / case["temperature"], -1)
                reached = []
                for i in children:
                    t = token[first + i]
                    q = x["draft"][first + i].double() if case["drawn"] else None
                    if accept[first + i] * (float(q[t]) if case["drawn"] else 1.0) < float(r[t] / r.sum()):
                        reached = [i]
                        break
                    rest = torch.relu(r / r.sum() - q) if case["drawn"] else r.index_fill(0, torch.tensor([t], device=DEVICE), 0.0)
                    r = rest if float(rest.sum()) > 0 else r
            if not reached:
                break
            node = reached[0]
            path.append(node)
        if case["temperature"] > 0.0:
            run = r.cumsum(0)
            best = min(int((run <= sample[s] * run[-1]).sum()), case["vocab"] - 1)
        paths.append(path + [-1] * (MOST - len(path)))
        lengths.append(len(path))
        tokens.append(best)
    return _int32(paths), _int32(lengths), torch.tensor(tokens, dtype=torch.int64, device=DEVICE)


def exact(case, seed):
    if case["kind"] == "keep":  # bytes that move: nothing is computed
        return None
    return {"append": _exact_append, "tree": _exact_tree, "verify": _exact_verify}[case["kind"]](case, _inputs(case, seed))
