"""Packed prompt attention and the paged 4-bit cache on the GPU, against 64-bit definitions."""

import numpy as np
import pytest
import torch

import serving_reference as ref
from reskv_amd import packed_attention
from reskv_amd.int4 import copy_pages, empty_pages, int4_append, int4_attention, int4_gather

pytestmark = pytest.mark.gpu


def rng(seed):
    return np.random.default_rng(seed)


def half(r, *shape, scale=1.0):
    return (r.standard_normal(shape) * scale).astype(np.float16)


def gpu(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def offsets(lengths, first=0):
    return [first + int(n) for n in np.concatenate(([0], np.cumsum(lengths)))]


def outlier_scale(r, heads):
    scale = np.exp(r.standard_normal((1, heads, 128)))
    for h in range(heads):
        scale[0, h, r.permutation(128)[:4]] *= 10
    return scale


def check(got, want, bound):
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    excess = np.abs(got - want) - bound
    assert excess.max() <= 0, f"off by {np.abs(got - want).max():.3e}, {(excess > 0).sum()} values past their bound"


# ---------------------------------------------------------------------------
# packed attention
# ---------------------------------------------------------------------------

def packed_inputs(seed, nq, nk, kv, gqa):
    r = rng(seed)
    return (half(r, sum(nq), kv * gqa, 128), half(r, sum(nk), kv, 128, scale=outlier_scale(r, kv)),
            half(r, sum(nk), kv, 128))


@pytest.mark.parametrize("nq,nk,kv,gqa", [
    ([1], [1], 1, 1),
    ([5, 1, 33], None, 2, 4),
    ([64, 63, 65], None, 2, 1),
    ([32, 31, 128, 129], None, 1, 4),
    ([300], None, 1, 3),
    ([70, 0, 3, 0], None, 1, 7),
    ([40, 17], None, 1, 16),
    ([1, 1, 1], [200, 1, 64], 2, 4),      # single tokens
    ([7, 20, 3], [300, 20, 0], 1, 8),     # chunks; one without keys
    ([50, 9], [20, 8], 1, 2),             # more queries than keys: the first see nothing
    ([2, 1], [1500, 1111], 1, 4),         # keys split over workgroups
    ([130], [900], 2, 5),
    ([3, 70, 1, 0], [2600, 1030, 700, 512], 3, 4),  # some split, some not
    ([20], None, 1, 64),
])
def test_packed_attention(device, nq, nk, kv, gqa):
    nk = nq if nk is None else nk
    q, k, v = packed_inputs(len(nq) + sum(nk), nq, nk, kv, gqa)
    qo, ko = offsets(nq), offsets(nk)
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), qo, ko, 128 ** -0.5)
    got = packed_attention(gpu(q), gpu(k), gpu(v), i32(qo), None if nk is nq else i32(ko))
    check(got, want, bound)


@pytest.mark.parametrize("gqa", [1, 4, 6])
def test_packed_attention_split_and_whole_agree(device, gqa):
    """max_keys only steers the split of the keys."""
    nq, nk = [3, 40], [2100, 1300]
    q, k, v = packed_inputs(9, nq, nk, 1, gqa)
    qo, ko = offsets(nq), offsets(nk)
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), qo, ko, 0.05)
    for most in (None, 2100, 512, 0):
        check(packed_attention(gpu(q), gpu(k), gpu(v), i32(qo), i32(ko), scaling=0.05, max_keys=most), want, bound)


def test_packed_attention_reads_strided_rows(device):
    """Views of a fused projection, and rows of head-major tensors, are read in place; odd ones are copied."""
    n, kv, gqa = 77, 2, 4
    r = rng(4)
    qkv = half(r, n, (gqa + 2) * kv, 128)
    q, k, v = qkv[:, : kv * gqa], qkv[:, kv * gqa: kv * gqa + kv], qkv[:, kv * gqa + kv:]
    off = i32([0, 30, 77])
    want = packed_attention(gpu(q), gpu(k), gpu(v), off)
    fused = gpu(qkv)
    assert torch.equal(packed_attention(fused[:, : kv * gqa], fused[:, kv * gqa: kv * gqa + kv],
                                        fused[:, kv * gqa + kv:], off), want)
    major = [gpu(x.transpose(1, 0, 2)).transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(packed_attention(*major, off), want)
    odd = []
    for x in (q, k, v):
        t = torch.empty(x.size + 1, dtype=torch.float16, device="cuda")[1:].view(x.shape)
        odd.append(t.copy_(gpu(x)))
    assert torch.equal(packed_attention(*odd, off), want)
    one = gpu(k)[:1].expand(n, kv, 128)  # token stride 0
    assert torch.equal(packed_attention(gpu(q), one, one, off), packed_attention(gpu(q), one.contiguous(),
                                                                                 one.contiguous(), off))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_packed_attention_what_is_not_seen_does_not_matter(device, bad):
    """NaN and infinities in other sequences, in later keys of the same one and behind the last."""
    nq = [70, 90, 5]
    q, k, v = packed_inputs(5, nq, nq, 1, 4)
    qo = offsets(nq)
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), qo, qo, 128 ** -0.5)
    k2, v2 = (np.concatenate((x, np.full((9, 1, 128), bad, np.float16))) for x in (k, v))
    k2[70 + 80:70 + 90] = bad       # the second sequence's last ten keys
    v2[70 + 80:70 + 90, :, ::3] = bad
    v2[50, 0, 5] = bad              # one channel of one key of the first
    got = packed_attention(gpu(q), gpu(k2), gpu(v2), i32(qo)).float().cpu().numpy()
    clean = np.ones(got.shape, bool)
    clean[150:160] = False
    clean[50:70, :, 5] = False
    assert np.isfinite(got[clean]).all()
    assert (np.abs(got - want) <= bound)[clean].all()
    # what is seen shows: as itself, or as NaN where its weight is 0 in fp16 (below 2^-39 of the
    # largest, as these keys' scores make many: 0 * infinity)
    shown = got[50:70, :, 5]
    assert (np.isnan(shown) | (shown == bad)).all()
    if np.isnan(bad):
        assert np.isnan(got[150:160]).all()


@pytest.mark.parametrize("n", [1, 15, 16, 17, 62, 63, 65, 100])
def test_packed_attention_reads_no_row_of_another_sequence(device, n):
    """A sequence between others of NaN keys and values, for every place where its last tile may end."""
    q, k, v = packed_inputs(40 + n, [n], [n], 2, 4)
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), [0, n], [0, n], 128 ** -0.5)
    bad = np.full((70, 2, 128), np.nan, np.float16)
    k, v = (np.concatenate((bad, x, bad)) for x in (k, v))
    q = np.concatenate((q, np.ones((1, 8, 128), np.float16)))
    got = packed_attention(gpu(q), gpu(k), gpu(v), i32([0, 0, n, n + 1]), i32([0, 70, 70 + n, 140 + n]))
    check(got[:n], want, bound)
    assert torch.isnan(got[n:].float()).all()


def test_packed_attention_rows_of_no_sequence(device):
    nq = [20, 33]
    q, k, v = packed_inputs(6, [70], [70], 2, 4)
    off = offsets(nq, first=4)
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), off, off, 128 ** -0.5)
    got = packed_attention(gpu(q), gpu(k), gpu(v), i32(off))
    check(got, want, bound)  # zeros before and behind the sequences
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    assert packed_attention(gpu(q), gpu(k), gpu(v), i32(off), out=out) is out
    assert (out[:4] == 7).all() and (out[57:] == 7).all() and torch.equal(out[4:57], got[4:57])
    # without any sequence's rows, and offsets outside the tensors
    assert (packed_attention(gpu(q), gpu(k), gpu(v), i32([0, 0])) == 0).all()
    wild = packed_attention(gpu(q), gpu(k), gpu(v), i32([-5, 70, 2000]))
    check(wild, *ref.packed(*(x.astype(np.float64) for x in (q, k, v)), [0, 70], [0, 70], 128 ** -0.5))


def test_packed_attention_without_keys_or_rows(device):
    q = torch.ones(3, 4, 128, dtype=torch.float16, device="cuda")
    none = torch.empty(0, 2, 128, dtype=torch.float16, device="cuda")
    assert (packed_attention(q, none, none, i32([0, 3]), i32([0, 0])) == 0).all()
    assert packed_attention(q[:0], none, none, i32([0, 0])).shape == (0, 4, 128)


def test_packed_attention_many_sequences(device):
    """More sequences than a wave has lanes."""
    r = rng(8)
    nq = [int(n) for n in r.integers(0, 9, 150)]
    q, k, v = packed_inputs(8, nq, nq, 1, 2)
    off = offsets(nq)
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), off, off, 128 ** -0.5)
    check(packed_attention(gpu(q), gpu(k), gpu(v), i32(off)), want, bound)


def test_packed_attention_small_weights_add_up(device):
    """One key far above many others: their weights, below fp16's smallest number together with
    the largest weight, still count."""
    n = 4096
    q = np.zeros((1, 1, 128), np.float16)
    k = np.zeros((n, 1, 128), np.float16)
    v = np.ones((n, 1, 128), np.float16)
    q[0, 0, 0], k[0, 0, 0], v[0] = 16, 18.5 * 128 ** 0.5 / 16, 0
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), [0, 1], [0, n], 128 ** -0.5)
    assert want.min() > 1e-5
    check(packed_attention(gpu(q), gpu(k), gpu(v), i32([0, 1]), i32([0, n])), want, bound)


def test_packed_attention_far_rows(device):
    """Keys, values and queries behind 2^31 elements of their tensors."""
    r = rng(50)
    n, far = 90, (1 << 31) // (2 * 128) + 1000
    q, k, v = half(r, n, 2, 128), half(r, n, 2, 128), half(r, n, 2, 128)
    qf, kf, vf = (torch.empty(far + n, 2, 128, dtype=torch.float16, device="cuda") for _ in range(3))
    for t, x in zip((qf, kf, vf), (q, k, v)):
        t[far:] = gpu(x)
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), [0, n], [0, n], 128 ** -0.5)
    for most in (n, 4096):
        got = packed_attention(qf, kf, vf, i32([far, far + n]), max_keys=most)
        check(got[far:], want, bound)
        assert (got[:5] == 0).all() and (got[far - 5: far] == 0).all()


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------

def make_table(r, counts, spare=3):
    """Page numbers in no order, -1 behind a sequence's last page, and the size of the pool."""
    ids = r.permutation(sum(counts) + spare)
    table = np.full((len(counts), max(max(counts), 1)), -1)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = ids[at: at + n]
        at += n
    return gpu(table.astype(np.int32)), sum(counts) + spare


def pages_of(lengths, page):
    return [-(-n // page) for n in lengths]


@pytest.mark.parametrize("page", [32, 64, 96, 256])
@pytest.mark.parametrize("lengths,starts", [([1], [0]), ([32, 31, 33], [0, 0, 0]), ([5, 70, 0, 200], [3, 31, 9, 64]),
                                            ([8, 16], [8, 20])])
def test_append_and_gather_are_exact(device, page, lengths, starts):
    r = rng(page + sum(lengths))
    kv = 2
    k, v = half(r, sum(lengths), kv, 128, scale=outlier_scale(r, kv)), half(r, sum(lengths), kv, 128)
    table, count = make_table(r, pages_of([a + b for a, b in zip(lengths, starts)], page))
    pool = empty_pages(count, kv, page)
    off = i32(offsets(lengths))
    int4_append(pool, table, i32(starts), gpu(k), gpu(v), off)
    got = int4_gather(pool, table, i32(starts), off, sum(lengths))
    for x, y in zip((k, v), got):
        want = ref.stored(x)[0].astype(np.float32).astype(np.float16)  # code * scale + low in fp32, then fp16
        assert np.array_equal(y.cpu().numpy(), want)


def test_append_tokens_one_by_one(device):
    """Decode steps give the same pages as one prompt, for every place in a block."""
    r = rng(2)
    n, kv, page = 70, 3, 64
    k, v = half(r, n, kv, 128), half(r, n, kv, 128)
    table, count = make_table(r, pages_of([n, n], page))
    whole, steps = empty_pages(count, kv, page), empty_pages(count, kv, page)
    both = [gpu(np.concatenate((x, x[::-1]))) for x in (k, v)]
    int4_append(whole, table, i32([0, 0]), *both, i32([0, n, 2 * n]))
    kg, vg = gpu(k), gpu(v)
    for t in range(n):
        int4_append(steps, table, i32([t, t]), torch.stack((kg[t], kg[n - 1 - t])), torch.stack((vg[t], vg[n - 1 - t])))
    assert torch.equal(whole, steps)


def test_append_leaves_other_tokens_and_pages(device):
    r = rng(3)
    kv, page = 1, 64
    pool = torch.from_numpy(r.integers(0, 255, (6, kv, page * 160), dtype=np.uint8)).cuda()
    table = i32([4, 1]).view(1, 2)
    before = pool.clone()
    rows = [gpu(half(r, 5, kv, 128)) for _ in range(2)]
    old = int4_gather(pool, table, i32([0]), i32([0, 128]), 128)
    int4_append(pool, table, i32([62]), *rows, i32([0, 5]))
    new = int4_gather(pool, table, i32([0]), i32([0, 128]), 128)
    for a, b in zip(old, new):
        keep = [i for i in range(128) if not 62 <= i < 67]
        assert torch.equal(a[keep].view(torch.int16), b[keep].view(torch.int16))
        assert torch.isfinite(b[62:67].float()).all()
    for p in (0, 2, 3, 5):
        assert torch.equal(pool[p], before[p])


def test_append_special_rows(device):
    """Equal channels, the ends of fp16, denormals, ties, and groups that are not finite."""
    r = rng(7)
    x = half(r, 12, 1, 128)
    x[0] = 0
    x[1] = -3.25
    x[2, 0, :32] = np.linspace(-65504, 65504, 32)
    x[3] = x[3] * 2.0 ** -22
    x[4, 0, :32] = np.arange(32) * 0.5  # codes on ties
    x[5, 0, :32] = np.linspace(0, 2.0 ** -24 * 31, 32)
    x[6, 0, 40] = np.nan
    x[7, 0, 100] = np.inf
    x[8, 0, 3] = -np.inf
    x[9, 0, 64:96] = 2.0 ** -24
    x[9, 0, 70] = 0
    table = i32([0]).view(1, 1)
    pool = empty_pages(1, 1, 32)
    int4_append(pool, table, i32([0]), gpu(x), gpu(x), i32([0, 12]))
    k, v = int4_gather(pool, table, i32([0]), i32([0, 12]), 12)
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    got = k.cpu().numpy()
    bad = np.zeros(x.shape, bool)
    bad[6, 0, 32:64] = bad[7, 0, 96:] = bad[8, 0, :32] = True
    assert np.isnan(got[bad]).all()
    clean = np.where(np.isfinite(x), x, 0)
    with np.errstate(over="ignore"):
        want = ref.stored(clean)[0].astype(np.float32).astype(np.float16)
    assert np.array_equal(got[~bad], want[~bad])


def test_pages_outside_the_pool_and_positions_outside_the_table(device):
    r = rng(11)
    kv, page = 2, 32
    k, v = half(r, 100, kv, 128), half(r, 100, kv, 128)
    pool = empty_pages(4, kv, page)
    table = gpu(np.array([[0, 99, 2], [-1, 3, 4]], np.int32))  # 99, -1 and 4 are no pages
    int4_append(pool, table, i32([0, 20]), gpu(k), gpu(v), i32([0, 50, 100]))
    assert (pool[1] == 0).all()
    got = int4_gather(pool, table, i32([0, 20]), i32([0, 50, 100]), 100)
    for x, y in zip((k, v), got):
        want = ref.stored(x)[0].astype(np.float32).astype(np.float16)
        want[32:50] = 0            # first sequence's second page
        want[50:62] = 0            # second sequence: tokens 20 .. 31
        want[50 + 44:] = 0         # tokens 64 .. 69
        assert np.array_equal(y.cpu().numpy(), want)
    far = int4_gather(pool, table, i32([96, -40]), i32([0, 4, 8]), 8)  # behind and before the table
    assert all((x == 0).all() for x in far)
    kept = pool.clone()
    int4_append(pool, table, i32([96, -40]), gpu(k[:8]), gpu(v[:8]), i32([0, 4, 8]))
    int4_append(pool, table, i32([96, -1]), gpu(k[:2]), gpu(v[:2]))
    assert torch.equal(pool, kept)
    # attention passes over the tokens of such pages
    q = half(r, 2, 4, 128)
    out = int4_attention(gpu(q), pool, table, i32([50, 70]))
    kd, ka = ref.stored(k)
    vd, va = ref.stored(v)
    rows = [list(range(32)), list(range(62, 94))]
    for b in range(2):
        want, bound = ref.sequence(q[b: b + 1].astype(np.float64), kd[rows[b]], vd[rows[b]], len(rows[b]) - 1,
                                   128 ** -0.5, ka[rows[b]], va[rows[b]])
        check(out[b: b + 1], want, bound)


def test_gather_rows_of_no_sequence(device):
    r = rng(12)
    pool, table = empty_pages(2, 1, 32), i32([1]).view(1, 1)
    x = half(r, 9, 1, 128)
    int4_append(pool, table, i32([0]), gpu(x), gpu(x), i32([0, 9]))
    k, v = int4_gather(pool, table, i32([0]), i32([3, 12]), 300)
    want = ref.stored(x)[0].astype(np.float32).astype(np.float16)
    for y in (k, v):
        y = y.cpu().numpy()
        assert np.array_equal(y[3:12], want) and (y[:3] == 0).all() and (y[12:] == 0).all()
    out = tuple(torch.full((20, 1, 128), 5.0, dtype=torch.float16, device="cuda") for _ in range(2))
    int4_gather(pool, table, i32([0]), i32([3, 12]), 20, out=out)
    for y in out:
        assert np.array_equal(y[3:12].cpu().numpy(), want) and (y[:3] == 5).all() and (y[12:] == 5).all()


# ---------------------------------------------------------------------------
# attention over pages
# ---------------------------------------------------------------------------

def filled(r, lengths, kv, page, k_scale=1.0, v_scale=1.0):
    k, v = half(r, sum(lengths), kv, 128, scale=k_scale), half(r, sum(lengths), kv, 128, scale=v_scale)
    table, count = make_table(r, pages_of(lengths, page))
    pool = torch.full((count, kv, page * 160), 255, dtype=torch.uint8, device="cuda")  # unused places read as NaN
    if sum(lengths):
        int4_append(pool, table, i32([0] * len(lengths)), gpu(k), gpu(v), i32(offsets(lengths)))
    return pool, table, k, v


def expected(q, k, v, lengths, scaling=128 ** -0.5):
    (kd, ka), (vd, va) = ref.stored(k), ref.stored(v)
    off = offsets(lengths)
    parts = [ref.sequence(q[b: b + 1].astype(np.float64), kd[off[b]: off[b + 1]], vd[off[b]: off[b + 1]],
                          lengths[b] - 1, scaling, ka[off[b]: off[b + 1]], va[off[b]: off[b + 1]])
             for b in range(len(lengths))]
    return tuple(np.concatenate(x) for x in zip(*parts))


@pytest.mark.parametrize("lengths,kv,gqa,page", [
    ([1], 1, 1, 32),
    ([2, 31, 32, 33], 2, 4, 32),
    ([0, 7, 128, 0], 1, 4, 64),
    ([100, 257, 64], 2, 3, 64),
    ([129, 1], 1, 8, 128),
    ([400], 1, 7, 96),
    ([90, 300], 1, 12, 64),
    ([61], 2, 16, 32),
    ([3000, 17], 1, 4, 256),  # several splits
    ([5000], 2, 8, 64),
])
def test_int4_attention(device, lengths, kv, gqa, page):
    r = rng(sum(lengths) + gqa)
    pool, table, k, v = filled(r, lengths, kv, page, k_scale=outlier_scale(r, kv))
    q = half(r, len(lengths), kv * gqa, 128)
    want, bound = expected(q, k, v, lengths)
    check(int4_attention(gpu(q), pool, table, i32(lengths)), want, bound)
    # a tighter bound on the lengths steers the split only
    check(int4_attention(gpu(q), pool, table, i32(lengths), max_length=max(lengths)), want, bound)


@pytest.mark.parametrize("scaling", [1.0, 0.01, -0.2, 0.0])
def test_int4_attention_scaling(device, scaling):
    r = rng(20)
    pool, table, k, v = filled(r, [150], 1, 64)
    q = half(r, 1, 4, 128)
    check(int4_attention(gpu(q), pool, table, i32([150]), scaling=scaling), *expected(q, k, v, [150], scaling))


@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1e-4, 1.0, 1.0), (300.0, 1e-3, 1.0), (1.0, 1.0, 1e-5),
                                                     (0.02, 1.0, 5000.0), (1e-3, 3000.0, 30.0)])
def test_int4_attention_magnitudes(device, q_scale, k_scale, v_scale):
    r = rng(21)
    lengths = [500, 77]
    pool, table, k, v = filled(r, lengths, 1, 64, k_scale, v_scale)
    q = half(r, 2, 4, 128, scale=q_scale)
    q[0, 1] *= np.float16(1e-2)  # heads of different sizes share one scaling
    want, bound = expected(q, k, v, lengths)
    check(int4_attention(gpu(q), pool, table, i32(lengths)), want, bound)


def test_int4_attention_scales_that_grow(device):
    """Values whose scale grows block by block, and one key far above the rest whose values are small."""
    r = rng(22)
    n = 700
    k, v = half(r, n, 1, 128), half(r, n, 1, 128)
    v = (v * 2.0 ** (np.arange(n) // 50 - 8)[:, None, None]).astype(np.float16)
    k[0] *= np.float16(3)
    table, count = make_table(r, pages_of([n], 64))
    pool = empty_pages(count, 1, 64)
    int4_append(pool, table, i32([0]), gpu(k), gpu(v), i32([0, n]))
    q = half(r, 1, 4, 128)
    q[0, 0] = k[0, 0]
    check(int4_attention(gpu(q), pool, table, i32([n])), *expected(q, k, v, [n]))


def test_int4_attention_nan_rows_and_unused_places(device):
    """A NaN that is seen shows in its heads only; unused places of pages never show."""
    r = rng(23)
    pool, table, k, v = filled(r, [45, 45], 2, 32)
    q = gpu(half(r, 2, 8, 128))
    clean = int4_attention(q, pool, table, i32([45, 45]))
    assert torch.isfinite(clean.float()).all()
    k[45 + 44, 1, 7] = np.nan
    int4_append(pool, table, i32([0, 0]), gpu(k), gpu(v), i32([0, 45, 90]))
    got = int4_attention(q, pool, table, i32([45, 45]))
    assert torch.isnan(got[1, 4:].float()).all()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1, :4], clean[1, :4])
    assert torch.equal(int4_attention(q, pool, table, i32([45, 44]))[0], clean[0])
    assert torch.isfinite(int4_attention(q, pool, table, i32([45, 44])).float()).all()


def test_int4_attention_lengths_are_clamped(device):
    r = rng(24)
    pool, table, k, v = filled(r, [64, 64], 1, 32)
    q = half(r, 2, 4, 128)
    want = int4_attention(gpu(q), pool, table, i32([64, 0]))
    assert torch.equal(int4_attention(gpu(q), pool, table, i32([10 ** 6, -3])), want)
    short = int4_attention(gpu(q), pool, table, i32([40, 40]))
    assert torch.equal(int4_attention(gpu(q), pool, table, i32([64, 64]), max_length=40), short)
    assert (int4_attention(gpu(q), pool, table, i32([64, 64]), max_length=0) == 0).all()


@pytest.mark.parametrize("gqa", [2, 8])
def test_int4_attention_many_sequences(device, gqa):
    """More sequences than a wave has lanes, empty ones among them."""
    r = rng(25)
    lengths = [int(n) for n in r.integers(0, 90, 150)]
    lengths[0] = lengths[70] = lengths[71] = lengths[149] = 0
    pool, table, k, v = filled(r, lengths, 1, 32)
    q = half(r, 150, gqa, 128)
    want, bound = expected(q, k, v, lengths)
    got = int4_attention(gpu(q), pool, table, i32(lengths))
    check(got, want, bound)
    assert torch.equal(int4_attention(gpu(q), pool, table, i32(lengths)), got)  # the same every time


@pytest.mark.parametrize("gqa,entries", [(4, 200001), (8, 150000)])
def test_int4_attention_long_tables(device, gqa, entries):
    """Runs of blocks over more page numbers than a wave holds at a time: a few pages that a long
    sequence uses again and again, so that a token counts as often as its page is named."""
    r = rng(26)
    pages = 40
    pool, once, k, v = filled(r, [32 * pages], 1, 32)
    order = once.cpu().numpy()[0]
    named = r.choice(pages, entries, p=(w := r.random(pages) ** 3) / w.sum())
    table = gpu(order[named].astype(np.int32)[None])
    length = 32 * entries - 11
    q = half(r, 1, gqa, 128)
    times = np.repeat(np.bincount(named, minlength=pages), 32).astype(np.float64)
    times[32 * named[-1] + 21: 32 * named[-1] + 32] -= 1  # the last page's last eleven tokens
    (kd, ka), (vd, va) = ref.stored(k), ref.stored(v)
    want, bound = np.zeros((1, gqa, 128)), np.zeros((1, gqa, 128))
    for h in range(gqa):
        s = 128 ** -0.5 * kd[:, 0] @ q[0, h].astype(np.float64)
        w = times * np.exp(s - s.max())
        w /= w.sum()
        want[0, h] = w @ vd[:, 0]
        delta = 160 * ref.H32 * 128 ** -0.5 * (ka[:, 0] @ np.abs(q[0, h].astype(np.float64))).max()
        # as in ref.sequence, with fp32 sums over 2^12 blocks of a wave, whose errors add up at most linearly
        bound[0, h] = (w @ va[:, 0]) * (2 * ref.H16 + 2 * delta + 2.0 ** -12) * 1.01 + ref.H16 * np.abs(want[0, h]) + 2.0 ** -24
    check(int4_attention(gpu(q), pool, table, i32([length])), want, bound)


def test_far_pages(device):
    """Pages behind 2^32 bytes of the pool."""
    r = rng(27)
    kv, page = 8, 64
    count = (1 << 32) // (kv * page * 160) + 200
    pool = torch.zeros(count, kv, page * 160, dtype=torch.uint8, device="cuda")
    lengths = [100, 64]
    table = i32([count - 1, 5, count - 7, count - 2]).view(2, 2)
    k, v = half(r, 164, kv, 128), half(r, 164, kv, 128)
    off = i32(offsets(lengths))
    int4_append(pool, table, i32([0, 0]), gpu(k), gpu(v), off)
    got = int4_gather(pool, table, i32([0, 0]), off, 164)
    for x, y in zip((k, v), got):
        assert np.array_equal(y.cpu().numpy(), ref.stored(x)[0].astype(np.float32).astype(np.float16))
    q = half(r, 2, 32, 128)
    check(int4_attention(gpu(q), pool, table, i32(lengths)), *expected(q, k, v, lengths))
    copy_pages(pool, [count - 1, count - 7], [count - 3, 9])
    assert torch.equal(pool[count - 1], pool[count - 3]) and torch.equal(pool[count - 7], pool[9])


# ---------------------------------------------------------------------------
# page copies, streams, graphs
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("layers,kv,page,n", [(None, 1, 32, 1), (3, 2, 64, 5), (2, 1, 32, 400), (1, 3, 96, 0)])
def test_copy_pages(device, layers, kv, page, n):
    r = rng(n + kv)
    shape = (2 * n + 2, kv, page * 160)
    pool = torch.from_numpy(r.integers(0, 255, shape if layers is None else (layers, *shape), dtype=np.uint8)).cuda()
    order = [int(p) for p in r.permutation(2 * n + 2)]
    source, target = order[:n], order[n: 2 * n]
    want = pool.clone()
    if n:
        want.movedim(-3, 0)[target] = pool.movedim(-3, 0)[source]
    copy_pages(pool, source, target)
    assert torch.equal(pool, want)
    if n:  # a source may be copied to several targets
        copy_pages(pool, [source[0], source[0]], [order[-1], order[-2]])
        assert torch.equal(pool.movedim(-3, 0)[order[-2]], want.movedim(-3, 0)[source[0]])


def test_current_stream(device):
    """The operators run on torch's current stream: behind a long copy there, not beside it."""
    r = rng(30)
    lengths = [90, 40]
    pool, table, k, v = filled(r, lengths, 2, 64)
    q = gpu(half(r, 2, 8, 128))
    off, lens = i32(offsets(lengths)), i32(lengths)
    kg, vg = gpu(k), gpu(v)
    rows = gpu(half(r, 130, 8, 128))
    want = int4_attention(q, pool, table, lens), packed_attention(rows, kg, vg, off)
    other, late_k, late_q = empty_pages(pool.shape[0], 2, 64), torch.zeros_like(kg), torch.zeros_like(q)
    big = torch.zeros(1 << 28, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(5):
            big.add_(1.0)
        late_k.copy_(kg)
        late_q.copy_(q)
        int4_append(other, table, i32([0, 0]), late_k, vg, off)
        got = int4_attention(late_q, other, table, lens), packed_attention(rows, late_k, vg, off)
        back = int4_gather(other, table, i32([0, 0]), off, 130)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert np.array_equal(back[0].cpu().numpy(), ref.stored(k)[0].astype(np.float32).astype(np.float16))


def test_decode_steps_in_a_graph(device):
    """An append and the attention captured together, replayed with eager work between: lengths,
    positions and rows come from device memory."""
    r = rng(31)
    start, steps, kv, gqa, page = [60, 2000], 40, 2, 4, 64
    ends = [n + steps for n in start]
    k, v = half(r, sum(ends), kv, 128), half(r, sum(ends), kv, 128)
    off = offsets(ends)
    table, count = make_table(r, pages_of(ends, page))
    pool = empty_pages(count, kv, page)
    first = [np.concatenate([x[off[b]: off[b] + start[b]] for b in range(2)]) for x in (k, v)]
    int4_append(pool, table, i32([0, 0]), *(gpu(x) for x in first), i32(offsets(start)))
    eager = pool.clone()
    row = [torch.zeros(2, kv, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    q = torch.zeros(2, kv * gqa, 128, dtype=torch.float16, device="cuda")
    pos, lens, out = i32(start), i32([n + 1 for n in start]), torch.zeros_like(q)

    def step(pages, out):
        int4_append(pages, table, pos, *row)
        int4_attention(q, pages, table, lens, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pool, out)
    for t in range(steps):
        for x, y in zip(row, (k, v)):
            x.copy_(gpu(np.stack([y[off[b] + start[b] + t] for b in range(2)])))
        q.copy_(gpu(half(r, 2, kv * gqa, 128)))
        graph.replay()
        want = torch.zeros_like(out)
        step(eager, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want), t
        assert torch.equal(pool, eager), t
        pos += 1
        lens += 1


def test_packed_attention_in_a_graph(device):
    """Replays read the offsets anew, with and without a split of the keys."""
    r = rng(32)
    for most in (400, 4096):
        q, k, v = (gpu(half(r, 400, h, 128)) for h in (8, 2, 2))
        off = i32([0, 100, 400])
        graph = torch.cuda.CUDAGraph()
        packed_attention(q, k, v, off, max_keys=most)
        with torch.cuda.graph(graph):
            out = packed_attention(q, k, v, off, max_keys=most)
        for mid in (100, 7, 399, 0):
            off[1] = mid
            q.copy_(gpu(half(r, 400, 8, 128)))
            graph.replay()
            assert torch.equal(out, packed_attention(q, k, v, off, max_keys=most))


def test_two_graphs_share_a_pool(device):
    """Workspaces of two captured graphs, of one memory pool, replayed in turns."""
    r = rng(34)
    lengths = [700, 45]
    pool, table, k, v = filled(r, lengths, 2, 64)
    lens, off = i32(lengths), i32([0, 2, 3])
    qa, qb = (torch.zeros(n, 8, 128, dtype=torch.float16, device="cuda") for n in (2, 3))
    kg, vg, ko = gpu(k), gpu(v), i32(offsets(lengths))
    first = lambda: int4_attention(qa, pool, table, lens)  # noqa: E731
    second = lambda: packed_attention(qb, kg, vg, off, ko, max_keys=4096)  # noqa: E731
    first(), second()
    handle, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for f in (first, second):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=handle):
            outs.append(f())
    for turn in range(6):
        for t in (qa, qb):
            t.copy_(gpu(half(r, *t.shape)))
        for i in (0, 1) if turn % 2 else (1, 0):
            graphs[i].replay()
            assert torch.equal(outs[i], (first, second)[i]())


def test_served_batch(device):
    """The operators together: prompts packed and stored, a chunk of each continued on the cached
    tokens, a page copied for a fork, and decode steps over the cache."""
    r = rng(33)
    kv, gqa, page = 2, 4, 64
    prompt, chunk, steps = [70, 5, 130], [9, 64, 1], 3
    total = [a + b + steps for a, b in zip(prompt, chunk)]
    off = offsets(total)
    q, k, v = half(r, off[-1], kv * gqa, 128), half(r, off[-1], kv, 128), half(r, off[-1], kv, 128)
    table, count = make_table(r, pages_of(total, page), spare=1)
    pool = empty_pages(count, kv, page)
    pick = lambda x, a, n: np.concatenate([x[off[b] + a[b]: off[b] + a[b] + n[b]] for b in range(3)])  # noqa: E731
    zero = [0] * 3
    int4_append(pool, table, i32(zero), gpu(pick(k, zero, prompt)), gpu(pick(v, zero, prompt)), i32(offsets(prompt)))
    int4_append(pool, table, i32(prompt), gpu(pick(k, prompt, chunk)), gpu(pick(v, prompt, chunk)), i32(offsets(chunk)))
    have = [a + b for a, b in zip(prompt, chunk)]
    kc, vc = int4_gather(pool, table, i32(zero), i32(offsets(have)), sum(have))
    got = packed_attention(gpu(pick(q, prompt, chunk)), kc, vc, i32(offsets(chunk)), i32(offsets(have)))
    want, bound = ref.packed(pick(q, prompt, chunk).astype(np.float64), kc.double().cpu().numpy(),
                             vc.double().cpu().numpy(), offsets(chunk), offsets(have), 128 ** -0.5)
    check(got, want, bound)
    last = pages_of(have, page)[0] - 1
    free = [p for p in range(count) if p not in table.cpu().numpy()][0]
    copy_pages(pool, [int(table[0, last])], [free])
    table[0, last] = free
    for t in range(steps):
        at = [n + t for n in have]
        one = [1] * 3
        int4_append(pool, table, i32(at), gpu(pick(k, at, one)), gpu(pick(v, at, one)))
        lens = [n + 1 for n in at]
        rows = pick(q, at, one)
        want, bound = expected(rows, pick(k, zero, lens), pick(v, zero, lens), lens)
        check(int4_attention(gpu(rows), pool, table, i32(lens)), want, bound)
