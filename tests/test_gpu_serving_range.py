"""Attention over 4-bit pages where values, weights or queries differ by many powers of two, against 64 bits: what one
token, channel group or head is like must not take bits from the others."""

import numpy as np
import pytest
import torch

import serving_reference as ref
from reskv_amd.int4 import empty_pages, int4_append, int4_attention

pytestmark = pytest.mark.gpu

SCALING = 128 ** -0.5


def gpu(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def attend(q, k, v, scaling=SCALING):
    n, kv, _ = k.shape
    pages = -(-n // 64)
    pool, table = empty_pages(pages, kv, 64), torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    int4_append(pool, table, i32([0]), gpu(k), gpu(v), i32([0, n]))
    return int4_attention(gpu(q), pool, table, i32([n]), scaling=scaling).double().cpu().numpy()


def expected(q, k, v, scaling=SCALING):
    """Rows and bound of serving_reference, plus what fp16 loses of small products of weight and scale: half its
    smallest step, 2^-25, where the reference of a head's group is held as 2^10 and half of the codes count
    16 times, so 2^-31 of the reference per code; the reference is not above the largest product."""
    (kd, ka), (vd, va), (_, scale, _) = ref.stored(k), ref.stored(v), ref.quantise(v)
    q, n = q.astype(np.float64), len(k)
    want, bound = ref.sequence(q, kd, vd, n - 1, scaling, ka, va)
    for h in range(q.shape[1]):
        kv = h * k.shape[1] // q.shape[1]
        s = scaling * (kd[:, kv] @ q[0, h])
        w = np.exp(s - s.max())
        largest = (w[:, None] * scale[:, kv, :, 0]).max(0) / w.sum()
        bound[0, h] += 15 * n * 2.0 ** -31 * np.repeat(largest, 32)
    return want, bound


def check(q, k, v):
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    assert all(np.isfinite(x).all() for x in (q, k, v))
    want, bound = expected(q, k, v)
    got = attend(q, k, v)
    excess = np.abs(got - want) - bound
    assert excess.max() <= 0, f"off by {np.abs(got - want).max():.3e}, {(excess > 0).sum()} values past their bound"


def inputs(seed, n, gqa, v_scale=1.0):
    r = np.random.default_rng(seed)
    return r.standard_normal((1, gqa, 128)), r.standard_normal((n, 1, 128)), r.standard_normal((n, 1, 128)) * v_scale


SIZES = pytest.mark.parametrize("n,gqa", [(1, 4), (32, 4), (500, 4), (500, 8), (3000, 3), (1111, 12)])


@SIZES
@pytest.mark.parametrize("powers", [(0, 10, 14, 18), (18, 0, 9, 4), (-12, 13, 13, -12)])
def test_channel_groups_of_different_size(device, n, gqa, powers):
    q, k, v = inputs(1, n, gqa)
    check(q, k, v * np.repeat(2.0 ** (-5.0 + np.array(powers) - 3), 32))


@SIZES
@pytest.mark.parametrize("size", [300, 3000, 10000])
@pytest.mark.parametrize("place", [0, 0.4, 1])
def test_a_large_token_without_weight(device, n, gqa, size, place):
    q, k, v = inputs(2, n, gqa, 0.1)
    at = min(int(place * n), n - 1)
    v[at] = np.clip(v[at] * 10 * size, -6e4, 6e4)
    k[at] = -4 * q[0].mean(0)
    check(q, k, v)


@SIZES
def test_scales_that_fall(device, n, gqa):
    """Large values first, whose weight is negligible once the later tokens are seen."""
    q, k, v = inputs(3, n, gqa)
    part = np.arange(n)[:, None, None] / n
    check(q, k + (4 * part - 2) * q[0].mean(0), v * 2.0 ** np.round(12 - 24 * part))


@SIZES
def test_a_largest_score_that_moves_with_every_block(device, n, gqa):
    """The largest weight so far is a new one in every block, by a little or by much."""
    q, k, v = inputs(4, n, gqa)
    q[0] = q[0, 0] + 0.01 * q[0]
    for top in (3.0, 60.0):
        rise = np.linspace(0, top, n)[:, None, None] * q[0, 0] / (q[0, 0] @ q[0, 0] * SCALING)
        check(q, 0.1 * k + rise, v * np.where(np.arange(n) < 20, 4000.0, 0.5)[:, None, None])


@SIZES
def test_heads_that_look_at_different_tokens(device, n, gqa):
    """One query head has its weight on a token of large values, its neighbours on the others."""
    q, k, v = inputs(5, n, gqa, 0.02)
    v[0] *= 2e6 / 100
    k[0] = 3 * (q[0, 0] - q[0, 1:].mean(0) if gqa > 1 else q[0, 0])
    check(q, k, v)


@SIZES
def test_values_without_a_scale(device, n, gqa):
    """Rows of equal channels (scale 0) among and before others, and scales of the smallest size."""
    q, k, v = inputs(6, n, gqa)
    v[: n // 2] = 3.0
    k[: n // 4] += 2 * q[0].mean(0)
    v[n // 2:: 3] = -0.25
    v[1::5, :, :64] *= 2.0 ** -20
    check(q, k, v)


@SIZES
def test_query_heads_of_different_size(device, n, gqa):
    """Heads at both ends of fp16, each with scores of its own over large keys."""
    q, k, v = inputs(7, n, gqa)
    q *= (2.0 ** np.array([14, -14, 0, -9]))[np.arange(gqa) % 4, None]
    check(q, k * 2.0 ** 13, v)
    check(q, k * 2.0 ** -8, v)


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("gqa", [4, 8, 16])
def test_a_query_head_that_is_no_number(device, bad, gqa):
    """The other heads are as they are without it."""
    q, k, v = (x.astype(np.float16) for x in inputs(8, 400, gqa, 2.0))
    q, k = q * np.float16(2.0 ** -12), k * np.float16(2.0 ** 11)
    want, bound = expected(q, k, v)
    q[0, 2, 5] = bad
    got = attend(q, k, v)
    assert np.isnan(got[0, 2]).all()
    excess = (np.abs(got - want) - bound)[0, [h for h in range(gqa) if h != 2]]
    assert excess.max() <= 0, f"{(excess > 0).sum()} values past their bound"


@pytest.mark.parametrize("gqa", [4, 8])
def test_a_group_of_values_that_is_no_number(device, gqa):
    """It shows in its 32 channels of the heads that see it, and nowhere else."""
    q, k, v = (x.astype(np.float16) for x in inputs(9, 700, gqa, 3.0))
    want, bound = expected(q, k, v)
    v[300, 0, 70] = np.inf
    got = attend(q, k, v)
    assert np.isnan(got[:, :, 64:96]).all()
    rest = np.r_[0:64, 96:128]
    assert (np.abs(got - want) <= bound)[:, :, rest].all()
