"""Packed attention and the 4-bit cache in 64 bits, from their definitions, with error bounds.

Bounds count roundings: half a step is 2^-11 of a value in fp16 and 2^-24 in fp32.
"""

import numpy as np

H16, H32 = 2.0 ** -11, 2.0 ** -24
GROUP = 32


def heads_of(x, g):
    return np.repeat(x, g, axis=1)


def sequence(q, k, v, first, scaling, spread_k=None, spread_v=None):
    """(rows, bound) of one sequence: q [n, Hq, 128], k and v [m, Hk, 128] float64; query i sees the keys up
    to i + first.  ``spread_k`` / ``spread_v`` (default |k|, |v|) bound the terms that a kernel
    adds up to a key or value channel.

    Scores: 128 products and up to 32 additions and scalings in fp32, so within 160 H32 of the sum of
    their terms; a weight is then off by that (twice: against the normaliser's own weights) and by
    2^-20 for the exponential and the fp32 sums.  Weights are rounded to fp16, and once more where a scale is
    multiplied in; the result is rounded to fp16 (2^-25 where it is denormal).
    """
    n, hq, _ = q.shape
    m, hk, _ = k.shape
    out, bound = np.zeros((n, hq, 128)), np.full((n, hq, 128), 2.0 ** -24)
    ak = np.abs(k) if spread_k is None else spread_k
    av = np.abs(v) if spread_v is None else spread_v
    rounds = H16 if spread_v is None else 2 * H16
    for h in range(hq):
        kv = h * hk // hq
        for i in range(n):
            seen = min(max(i + first + 1, 0), m)
            if seen == 0:
                continue
            s = scaling * (k[:seen, kv] @ q[i, h])
            mag = abs(scaling) * (ak[:seen, kv] @ np.abs(q[i, h]))
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ v[:seen, kv]
            delta = 160 * H32 * mag.max()
            spread = w @ av[:seen, kv]
            bound[i, h] += spread * (rounds + 2 * delta + 2.0 ** -20) * 1.01 + H16 * np.abs(out[i, h]) * 1.01
    return out, bound


def packed(q, k, v, q_off, k_off, scaling):
    """(rows, bound) of packed sequences; rows of no sequence are zero."""
    out, bound = np.zeros(q.shape), np.full(q.shape, 2.0 ** -24)
    for s in range(len(q_off) - 1):
        a, b, c, d = q_off[s], q_off[s + 1], k_off[s], k_off[s + 1]
        out[a:b], bound[a:b] = sequence(q[a:b], k[c:d], v[c:d], (d - c) - (b - a), scaling)
    return out, bound


def quantise(x):
    """(codes, scale, low) of rows [..., 128] as float64 [..., 4, 32] and [..., 4, 1]."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], 128 // GROUP, GROUP)
    low, high = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    scale = ((high - low) / 15).astype(np.float16).astype(np.float64)
    code = np.rint((g - low) / np.where(scale == 0, 1, scale))
    return np.where(scale == 0, 0, np.clip(code, 0, 15)), scale, low


def stored(x):
    """(values, sum of the absolute terms of a value) that the cache holds of rows [..., 128]."""
    code, scale, low = quantise(x)
    return (code * scale + low).reshape(x.shape), (code * scale + np.abs(low)).reshape(x.shape)
