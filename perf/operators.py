"""Serving operators for sequences of different lengths, as cases that can be timed and compared.

Four kinds, each through the entry points that a program calls:

* ``packed`` -- ``packed_attention``: causal attention of packed prompts, or of prompt chunks that continue
  on keys already there;
* ``decode`` -- ``int4_attention``: one token of every sequence against a paged cache of 4-bit keys and values;
* ``store``  -- ``int4_append`` and ``int4_gather``: new tokens quantised into their pages, and the stored
  values read back as a continuing prompt needs them;
* ``fork``   -- ``copy_pages``: pages of every layer copied, as forked sequences and compaction need it.

``run`` computes them in plain torch in 32 bits where ``own`` is false, and calls the framework where it is
true.  Shapes are the Llama-3.1-8B layer's (32 query heads, 8 KV heads, 128 channels) unless a case says
otherwise; keys have per-channel scales with a few outlier channels, values are N(0, 1).
"""

import math
import random

import torch

own = False

D = 128
GROUP = 32  # channels that share a scale and a lowest value
DEVICE = "cuda"
SCALING = D ** -0.5


def listed():
    return [
        # one short prompt: a chat turn that arrives alone; latency
        {"name": "packed_1x100", "kind": "packed", "seqs": 1, "short": 100, "long": 100, "context": 0,
         "kv": 8, "gqa": 4},
        # prompts of a busy server, most of them short, packed without padding
        {"name": "packed_24x16_1500", "kind": "packed", "seqs": 24, "short": 16, "long": 1500, "context": 0,
         "kv": 8, "gqa": 4},
        # one long document
        {"name": "packed_1x16384", "kind": "packed", "seqs": 1, "short": 16384, "long": 16384, "context": 0,
         "kv": 8, "gqa": 4},
        # chunks that continue on long contexts: few rows, many keys
        {"name": "packed_3x33_200_after_20000", "kind": "packed", "seqs": 3, "short": 33, "long": 200,
         "context": 20000, "kv": 8, "gqa": 4},
        # one conversation, one token; latency and launches
        {"name": "decode_1x1000", "kind": "decode", "seqs": 1, "short": 1000, "long": 1000, "kv": 8, "gqa": 4,
         "page": 64},
        # a full serving batch around the 8K context
        {"name": "decode_32x2000_8192", "kind": "decode", "seqs": 32, "short": 2000, "long": 8192, "kv": 8,
         "gqa": 4, "page": 64},
        # a few very different lengths, eight query heads to a KV head, wide pages
        {"name": "decode_5x17_65001_gqa8", "kind": "decode", "seqs": 5, "short": 17, "long": 65001, "kv": 4,
         "gqa": 8, "page": 256},
        # a full batch at 16K, the most bytes
        {"name": "decode_32x16384", "kind": "decode", "seqs": 32, "short": 16384, "long": 16384, "kv": 8,
         "gqa": 4, "page": 64},
        # a decode step's tokens, each in the middle of a page
        {"name": "store_32x1", "kind": "store", "seqs": 32, "short": 1, "long": 1, "context": 300, "kv": 8,
         "page": 64},
        # prompts of a batch, ragged
        {"name": "store_16x500_8192", "kind": "store", "seqs": 16, "short": 500, "long": 8192, "context": 0,
         "kv": 8, "page": 64},
        # a beam's last pages, copied before they are written to: every layer, a page or two
        {"name": "fork_32x3", "kind": "fork", "layers": 32, "pages": 64, "copies": 3, "kv": 8, "page": 64},
        # compaction of a pool
        {"name": "fork_32x300", "kind": "fork", "layers": 32, "pages": 700, "copies": 300, "kv": 8, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["packed"] * 4 + ["decode"] * 5 + ["store"] * 3 + ["fork"])
    kv, gqa = rng.choice([1, 2, 4, 8, 8, 8]), rng.choice([1, 2, 3, 4, 4, 4, 7, 8])
    page = rng.choice([32, 64, 64, 128, 256])
    if kind == "packed":
        if rng.random() < 0.3:
            return {"kind": kind, "seqs": rng.randint(1, 8), "short": 1, "long": _log(rng, 1, 400),
                    "context": _log(rng, 100, 20000), "kv": kv, "gqa": gqa}
        long = _log(rng, 20, 8192)
        seqs = _log(rng, 1, max(1, min(32, 16384 * 3 // long)))
        return {"kind": kind, "seqs": seqs, "short": max(1, long // rng.choice([1, 4, 100])), "long": long,
                "context": 0, "kv": kv, "gqa": gqa}
    if kind == "decode":
        long = _log(rng, 20, 65536)
        seqs = _log(rng, 1, max(1, min(64, 32 * 16384 // long)))
        return {"kind": kind, "seqs": seqs, "short": max(1, long // rng.choice([1, 3, 100])), "long": long,
                "kv": kv, "gqa": gqa, "page": page}
    if kind == "store":
        long = _log(rng, 1, 8192)
        seqs = _log(rng, 1, max(1, min(32, 8 * 8192 // long)))
        return {"kind": kind, "seqs": seqs, "short": max(1, long // rng.choice([1, 10])), "long": long,
                "context": rng.choice([0, rng.randint(1, 3000)]), "kv": kv, "page": page}
    copies = _log(rng, 1, 250)
    return {"kind": kind, "layers": rng.choice([1, 16, 32]), "pages": 2 * copies + rng.randint(0, 100),
            "copies": copies, "kv": kv, "page": rng.choice([32, 64])}


def _lengths(case):
    """Each sequence's new tokens: spread over the logarithm of the range, one of them the longest."""
    rng = random.Random(f"{case['seqs']} {case['short']} {case['long']}")
    out = [_log(rng, case["short"], case["long"]) for _ in range(case["seqs"])]
    out[rng.randrange(len(out))] = case["long"]
    return out


def _contexts(case):
    """Tokens that each sequence holds already."""
    c = case.get("context", 0)
    rng = random.Random(f"{c} {case['seqs']}")
    return [rng.randint((c + 1) // 2, c) for _ in range(case["seqs"])]


def _sums(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


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


def _inputs(case, seed):
    """The tensors of a case, from the seed alone: what ``prepare`` lays out and ``exact`` starts from."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "fork":
        shape = (case["layers"], case["pages"], case["kv"], case["page"] * 160)
        order = list(range(case["pages"]))
        random.Random(seed).shuffle(order)
        return {"pool": torch.randint(256, shape, dtype=torch.uint8, device=DEVICE, generator=gen),
                "source": order[: case["copies"]], "target": order[case["copies"]: 2 * case["copies"]]}
    new, have = _lengths(case), _contexts(case)
    if case["kind"] == "packed":
        k, v = _keys_values(gen, sum(new) + sum(have), case["kv"])
        return {"new": new, "all": [a + b for a, b in zip(new, have)], "k": k, "v": v,
                "q": _normal(gen, sum(new), case["kv"] * case["gqa"], D).half()}
    k, v = _keys_values(gen, sum(new), case["kv"])
    out = {"new": new, "have": have, "k": k, "v": v}
    if case["kind"] == "decode":
        out["q"] = _normal(gen, case["seqs"], case["kv"] * case["gqa"], D).half()
    return out


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


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    kind = case["kind"]
    if kind == "packed":
        if own:
            state["q_offsets"] = _int32(_sums(state["new"]))
            state["k_offsets"] = state["q_offsets"] if case["context"] == 0 else _int32(_sums(state["all"]))
        return state
    if kind == "fork":
        return state
    starts = state["have"]
    ends = [a + b for a, b in zip(starts, state["new"])]
    state["table"], pages = _page_table(case, ends, seed)
    state["starts"], state["offsets"] = _int32(starts), _int32(_sums(state["new"]))
    if own:
        from reskv_amd.int4 import empty_pages, int4_append

        state["pool"] = empty_pages(pages, case["kv"], case["page"], device=DEVICE)
        if kind == "decode":
            int4_append(state["pool"], state["table"], state["starts"], state["k"], state["v"], state["offsets"])
            state["lengths"] = _int32(state["new"])
    elif kind == "decode":
        state["cache"] = [_quantise(state["k"]), _quantise(state["v"])]
    else:
        rows = (pages * case["page"], case["kv"], D // GROUP)
        state["cache"] = [(torch.zeros(*rows, GROUP, dtype=torch.uint8, device=DEVICE),
                           torch.zeros(*rows, 1, dtype=torch.float16, device=DEVICE),
                           torch.zeros(*rows, 1, dtype=torch.float16, device=DEVICE)) for _ in range(2)]
        state["slots"] = _slots(state["table"], case["page"], starts, state["new"])
    if kind == "decode":
        del state["k"], state["v"]
    return state


def _attend(q, k, v, first, out):
    """One sequence in plain form: query i sees the keys up to i + first; a query that sees none gives zeros.
    q [n, heads, 128], k and v [m, KV heads, 128] in any type, out fp16 rows."""
    n, heads, _ = q.shape
    m, kv, _ = k.shape
    kt = k.float().permute(1, 2, 0).contiguous()
    vt = v.float().transpose(0, 1).contiguous()
    column = torch.arange(m, device=q.device)
    for r0 in range(0, n, 1024):
        rows = min(n, r0 + 1024) - r0
        qf = q[r0: r0 + rows].float().view(rows, kv, heads // kv, D).permute(1, 2, 0, 3).reshape(kv, -1, D)
        score = torch.matmul(qf, kt).view(kv, heads // kv, rows, m) * SCALING
        hidden = column[None, :] > torch.arange(r0 + first, r0 + first + rows, device=q.device)[:, None]
        score.masked_fill_(hidden, -math.inf)
        top = score.amax(-1, keepdim=True)
        score.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
        total = score.sum(-1, keepdim=True)
        res = torch.matmul(score.view(kv, -1, m), vt).view(kv, heads // kv, rows, D)
        res = torch.where(total > 0, res / total, torch.zeros_like(res))
        out[r0: r0 + rows] = res.permute(2, 0, 1, 3).reshape(rows, heads, D).half()


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "fork":
        pool = state["pool"]
        pool[:, state["target"]] = pool[:, state["source"]]
        return pool
    if kind == "store":
        rows = state["slots"]
        out = []
        for x, cache in zip((state["k"], state["v"]), state["cache"]):
            for part, held in zip(_quantise(x), cache):
                held[rows] = part
            out.append(_values(*(held[rows] for held in cache)).half())
        return tuple(out)
    q = state["q"]
    out = torch.empty_like(q)
    if kind == "packed":
        qs, ks = _sums(state["new"]), _sums(state["all"])
        for b, (n, m) in enumerate(zip(state["new"], state["all"])):
            _attend(q[qs[b]: qs[b] + n], state["k"][ks[b]: ks[b] + m], state["v"][ks[b]: ks[b] + m], m - n,
                    out[qs[b]: qs[b] + n])
        return out
    ks = _sums(state["new"])
    for b, m in enumerate(state["new"]):
        k, v = (_values(*(part[ks[b]: ks[b] + m] for part in cache)) for cache in state["cache"])
        _attend(q[b: b + 1], k, v, m - 1, out[b: b + 1])
    return out


def run(state):
    if not own:
        return _run_plain(state)
    kind = state["case"]["kind"]
    if kind == "packed":
        from reskv_amd import packed_attention

        return packed_attention(state["q"], state["k"], state["v"], state["q_offsets"], state["k_offsets"],
                                max_keys=max(state["all"]))
    from reskv_amd.int4 import copy_pages, int4_append, int4_attention, int4_gather

    if kind == "fork":
        copy_pages(state["pool"], state["source"], state["target"])
        return state["pool"]
    if kind == "store":
        int4_append(state["pool"], state["table"], state["starts"], state["k"], state["v"], state["offsets"])
        return int4_gather(state["pool"], state["table"], state["starts"], state["offsets"], state["k"].shape[0])
    return int4_attention(state["q"], state["pool"], state["table"], state["lengths"],
                          max_length=max(state["new"]))


def work(case):
    kind = case["kind"]
    if kind == "fork":
        return {"bytes": 2 * case["layers"] * case["copies"] * case["kv"] * case["page"] * 160, "flops": 0}
    new, have, kv = _lengths(case), _contexts(case), case["kv"]
    if kind == "store":
        # rows in, codes with their scales and lowest values out and in again, rows out
        return {"bytes": sum(new) * kv * (512 + 160 + 160 + 512), "flops": 0}
    heads = kv * case["gqa"]
    if kind == "decode":
        return {"bytes": sum(new) * kv * 160 + 2 * case["seqs"] * heads * D * 2,
                "flops": 4 * D * heads * sum(new)}
    pairs = sum(n * h + n * (n + 1) // 2 for n, h in zip(new, have))
    return {"bytes": (sum(new) + sum(have)) * kv * 512 + 2 * sum(new) * heads * D * 2, "flops": 4 * D * heads * pairs}


def _exact_values(x):
    """What 4 bits hold of rows [N, heads, 128], in 64 bits from the definition."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    step = ((high - low) / 15).half().double()
    code = torch.round((g - low) / torch.where(step == 0, torch.ones_like(step), step)).clamp(max=15)
    return torch.where(step == 0, low, low + step * code).reshape(x.shape)


def _exact_rows(q, k, v, first):
    """Attention of one sequence in 64 bits, head by head; query i sees keys 0 .. i + first."""
    n, heads, _ = q.shape
    m, kv, _ = k.shape
    out = torch.zeros(n, heads, D, dtype=torch.float64, device=q.device)
    for h in range(heads):
        kh, vh = k[:, h * kv // heads].double(), v[:, h * kv // heads].double()
        for r0 in range(0, n, 2048):
            qh = q[r0: r0 + 2048, h].double()
            dots = (qh @ kh.t()) / math.sqrt(D)
            seen = torch.ones(qh.shape[0], m, dtype=torch.bool, device=q.device).tril(r0 + first)
            dots = torch.where(seen, dots, torch.full_like(dots, -math.inf))
            weights = torch.exp(dots - torch.logsumexp(dots, -1, keepdim=True))
            out[r0: r0 + 2048, h] = torch.nan_to_num(weights) @ vh
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "fork":
        return None
    x = _inputs(case, seed)
    if kind == "store":
        return _exact_values(x["k"]), _exact_values(x["v"])
    out = torch.empty(x["q"].shape, dtype=torch.float64, device=DEVICE)
    held = x["all"] if kind == "packed" else x["new"]
    asked = x["new"] if kind == "packed" else [1] * case["seqs"]
    i = j = 0
    for n, m in zip(asked, held):
        k, v = x["k"][j: j + m], x["v"][j: j + m]
        if kind == "decode":
            k, v = _exact_values(k), _exact_values(v)
        out[i: i + n] = _exact_rows(x["q"][i: i + n], k, v, m - n)
        i, j = i + n, j + m
    return out
