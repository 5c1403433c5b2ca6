"""The operators of drafted decoding in 64 bits, from their definitions.

Bounds count roundings: half a step is 2^-11 of a value in fp16 and 2^-24 in fp32.
"""

import numpy as np

from serving_reference import H16, H32


def rotate(x, cos, sin, positions, interleaved):
    """(rows, bound) of x [N, heads, 128] float64, their first channels turned: products and a sum rounded to fp32, the
    result to fp16."""
    half = cos.shape[1]
    c, s = cos[positions][:, None].astype(np.float64), sin[positions][:, None].astype(np.float64)
    out, terms = x.copy(), np.zeros_like(x)
    at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., at[0]], x[..., at[1]]
    out[..., at[0]], out[..., at[1]] = a * c - b * s, b * c + a * s
    terms[..., at[0]], terms[..., at[1]] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return out, H16 * np.abs(out) + 3 * H32 * terms + 2.0 ** -25


def rotated_fp16(x, cos, sin, positions, interleaved):
    """fp16 rows as the definition rounds them: numpy rounds every fp32 product and sum by itself."""
    half = cos.shape[1]
    c, s = cos[positions][:, None], sin[positions][:, None]
    assert c.dtype == s.dtype == np.float32
    out = x.astype(np.float32)
    at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = out[..., at[0]].copy(), out[..., at[1]].copy()
    out[..., at[0]], out[..., at[1]] = a * c - b * s, b * c + a * s
    return out.astype(np.float16)


def masks(parents):
    """Every node's mask of itself and its ancestors, as Python numbers; a parent that is not before its node is none."""
    out = []
    for i, p in enumerate(parents):
        out.append(1 << i | (out[p] if 0 <= p < i else 0))
    return out


def tree_attention(q, k, v, visible, scaling, spread_k, spread_v):
    """(rows, bound) of one sequence: q [n, Hq, 128], k and v [m, Hk, 128] float64, visible [n, m].

    ``spread_k`` and ``spread_v`` bound the terms that are added up to a key or value channel.  Scores: 128 products and up to 32
    additions and scalings in fp32, within 160 H32 of the sum of their terms; a weight is off by that twice (against
    the normaliser's own weights) and by 2^-20 for the exponential and the fp32 sums.  V and the weights are rounded to
    fp16 once each (a weight to 2^-25 of 2^9, a sixty-fourth of the largest at most, where it is denormal), and so is the result.
    """
    n, hq, _ = q.shape
    m, hk, _ = k.shape
    out, bound = np.zeros((n, hq, 128)), np.full((n, hq, 128), 2.0 ** -24)
    for h in range(hq):
        kv = h * hk // hq
        for i in range(n):
            see = np.flatnonzero(visible[i])
            if see.size == 0:
                continue
            s = scaling * (k[see, kv] @ q[i, h])
            mag = abs(scaling) * (spread_k[see, kv] @ np.abs(q[i, h]))
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ v[see, kv]
            delta = 160 * H32 * mag.max()
            spread = w @ spread_v[see, kv]
            lost = 2.0 ** -34 * spread_v[see, kv].sum(0) + 2.0 ** -25
            bound[i, h] += spread * (2 * H16 + 2 * delta + 2.0 ** -20) * 1.01 + lost + H16 * np.abs(out[i, h]) * 1.01
    return out, bound


def softmax(x, temperature):
    x = x.astype(np.float64) / temperature
    e = np.exp(x - x.max())
    return e / e.sum()


def verify(logits, tokens, parents, accept, sample, draft, temperature):
    """(path, token, margin) of one sequence: logits [n, V], the others by node; margin is how near the closest of the
    decisions came to its border, relative to the sums that decide it."""
    n, vocab = logits.shape
    n = min(n, 64)
    if n == 0:
        return [], -1, 1.0
    here, path, margin = 0, [0], 1.0
    if temperature == 0.0:
        best = [-1 if np.isnan(row).any() else int(np.argmax(row)) for row in logits]
        for i in range(1, n):
            if parents[i] == here and 0 <= tokens[i] < vocab and tokens[i] == best[here]:
                here = i
                path.append(i)
        return path, best[here], margin

    def fine(row):
        return not np.isnan(row).any() and not np.isposinf(row).any() and np.isfinite(row).any()

    r = softmax(logits[0], temperature) if fine(logits[0]) else None
    for i in range(1, n):
        t = int(tokens[i])
        if r is None or parents[i] != here or not 0 <= t < vocab:
            continue
        q = np.zeros(vocab) if draft is None else draft[i].astype(np.float64)
        if draft is None:
            q[t] = 1.0
        chance, asked = r[t] / r.sum(), float(accept[i]) * q[t]
        margin = min(margin, abs(chance - asked))
        if asked < chance:
            here = i
            path.append(i)
            r = softmax(logits[i], temperature) if fine(logits[i]) else None
            continue
        rest = np.maximum(r / r.sum() - q, 0.0)
        if draft is None:
            rest = r.copy()
            rest[t] = 0.0
        if rest.sum() > 0:
            r = rest
    if r is None:
        return path, -1, margin
    run = np.cumsum(r) / r.sum()
    past = np.flatnonzero(np.cumsum(r) > float(sample) * r.sum())
    margin = min(margin, np.abs(run - float(sample)).min())
    return path, int(past[0]) if past.size else int(np.flatnonzero(r > 0)[-1]), margin
