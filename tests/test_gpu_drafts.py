"""Operators of drafted decoding against their definitions in 64 bits (drafts_reference.py)."""

import numpy as np
import pytest
import torch

import drafts_reference as ref
from reskv_amd.drafts import draft_tree, verify_drafts
from reskv_amd.int4 import empty_pages, int4_append, int4_append_rope, int4_gather, int4_keep, int4_tree_attention
from serving_reference import stored

pytestmark = pytest.mark.gpu

D = 128


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def sums(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device="cuda")


def random_parents(rng, n):
    return [-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, n)] if n else []


def page_table(rng, lengths, page, spare=2):
    """A shuffled table for sequences of these lengths and the number of pages; -1 behind a sequence's pages."""
    need = [-(-n // page) for n in lengths]
    ids = rng.permutation(sum(need) + spare)
    table = np.full((len(lengths), max(max(need), 1)), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at: at + n]
        at += n
    return i32(table.tolist()), len(ids)


# -- append with rotation --------------------------------------------------------------------------------

def tables(positions, rotary, seed=0):
    half = rotary // 2
    inv = 10000.0 ** (-np.arange(half) / half)
    ang = np.arange(positions)[:, None] * inv[None]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


APPEND = [  # starts, new tokens, KV heads, ratio, page, rotated channels, interleaved, positions given
    ([0], [1], 1, 1, 32, 128, False, False),
    ([37, 0, 95], [1, 1, 1], 2, 4, 64, 128, False, False),
    ([5, 31, 64], [70, 0, 33], 3, 1, 32, 64, False, False),
    ([0, 40], [129, 3], 2, 3, 64, 128, True, False),
    ([17, 3, 60, 200], [5, 64, 1, 17], 1, 8, 256, 32, True, True),
    ([100, 31], [9, 33], 4, 2, 96, 16, False, True),
    ([8], [40], 8, 4, 64, 96, True, True),
]


@pytest.mark.parametrize("case", APPEND, ids=range(len(APPEND)))
@pytest.mark.parametrize("packed", [True, False])
def test_append_rope(case, packed):
    """The bits of a rotation that numpy rounds step by step, then int4_append; the queries likewise, and within their roundings
    of 64 bits."""
    starts, new, heads, ratio, page, rotary, interleaved, given = case
    if not packed:
        new = [1] * len(starts)
    rng = np.random.default_rng(rotary + sum(starts))
    n = sum(new)
    ends = [a + b for a, b in zip(starts, new)]
    table, pages = page_table(rng, ends, page)
    cos, sin = tables(max(ends) + 3, rotary)
    positions = np.concatenate([s + np.arange(c) for s, c in zip(starts, new)]).astype(np.int32)
    if given:
        positions = rng.integers(0, max(ends) + 3, n).astype(np.int32)
    rows = rng.standard_normal((n, heads * (ratio + 2), D)).astype(np.float16)
    fused = torch.from_numpy(rows.reshape(n, -1)).cuda().view(n, -1, D)
    q, k, v = fused[:, : heads * ratio], fused[:, heads * ratio: heads * (ratio + 1)], fused[:, heads * (ratio + 1):]
    pool = torch.randint(256, empty_pages(pages, heads, page).shape, dtype=torch.uint8, device="cuda",
                         generator=torch.Generator("cuda").manual_seed(1))
    other = pool.clone()
    offsets = i32(sums(new).tolist()) if packed else None
    out = int4_append_rope(pool, table, i32(starts), q, k, v, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), offsets,
                           positions=i32(positions.tolist()) if given else None, interleaved=interleaved)
    want = ref.rotated_fp16(rows[:, : heads * (ratio + 1)], cos, sin, positions, interleaved)
    assert np.array_equal(out.cpu().numpy().view(np.uint16), want[:, : heads * ratio].view(np.uint16))
    exact, bound = ref.rotate(rows[:, : heads * ratio].astype(np.float64), cos, sin, positions, interleaved)
    assert (np.abs(out.cpu().numpy() - exact) <= bound).all()
    turned = torch.from_numpy(want[:, heads * ratio:].copy()).cuda()
    int4_append(other, table, i32(starts), turned, v, offsets)
    assert torch.equal(pool, other)


def test_append_rope_leaves_out_rows_outside():
    """A position outside the tables, a page that is not there, rows of no sequence: not stored, and queries zero or left."""
    rng = np.random.default_rng(3)
    n, heads = 12, 2
    cos, sin = tables(20, 128)
    table = i32([[1, -1], [0, 2]])
    starts, offsets = i32([30, 4]), i32([2, 6, 10])  # rows 0, 1, 10, 11 are nobody's; row 4 on of sequence 0 has no page
    positions = i32([0, 0, 3, 25, 5, 6, 7, -1, 20, 19, 0, 0])
    q, k, v = (torch.from_numpy(rng.standard_normal((n, h, D)).astype(np.float16)).cuda() for h in (4, 2, 2))
    pool = torch.randint(256, (4, heads, 32 * 160), dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    before, kept = pool.clone(), torch.full_like(q, 7.0)
    c, s = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    zero = int4_append_rope(pool, table, starts, q, k, v, c, s, offsets, positions=positions)
    again = before.clone()
    int4_append_rope(again, table, starts, q, k, v, c, s, offsets, positions=positions, out=kept)
    assert torch.equal(pool, again)
    good = [2, 4, 5, 6, 9]
    want = ref.rotated_fp16(q.cpu().numpy()[good], cos, sin, positions.cpu().numpy()[good], False)
    assert np.array_equal(zero.cpu().numpy()[good], want) and np.array_equal(kept.cpu().numpy()[good], want)
    bad = [i for i in range(n) if i not in good]
    assert (zero[bad] == 0).all() and (kept[bad] == 7).all()
    # what is stored: row 2 at token 30 of sequence 0, rows 6 and 9 at tokens 4 and 7 of sequence 1
    turned = torch.from_numpy(ref.rotated_fp16(k.cpu().numpy(), cos, sin, positions.clamp(0, 19).cpu().numpy(), False)).cuda()
    for row, seq, at in ((2, 0, 30), (6, 1, 4), (9, 1, 7)):
        int4_append(before, table[seq: seq + 1].contiguous(), i32([at]), turned[row: row + 1], v[row: row + 1])
    assert torch.equal(pool, before)


def test_append_rope_without_queries_and_with_strides():
    rng = np.random.default_rng(4)
    cos, sin = tables(50, 64)
    c, s = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    k, v = (torch.from_numpy(rng.standard_normal((5, 2, D)).astype(np.float16)).cuda() for _ in range(2))
    table, starts, offsets = i32([[0, 1]]), i32([30]), i32([0, 5])
    a, b = empty_pages(2, 2, 32), empty_pages(2, 2, 32)
    assert int4_append_rope(a, table, starts, None, k, v, c, s, offsets) is None
    wide = torch.zeros(5, 2, 2 * D, dtype=torch.float16, device="cuda")
    wide[..., ::2] = k  # a channel stride that the kernel does not read: copied
    q = wide[..., ::2].transpose(0, 1).contiguous().transpose(0, 1)
    out = int4_append_rope(b, table, starts, q, wide[..., ::2], v.expand(5, 2, D), c, s, offsets)
    assert torch.equal(a, b)
    assert np.array_equal(out.cpu().numpy(), ref.rotated_fp16(k.cpu().numpy(), cos, sin, 30 + np.arange(5), False))
    odd = torch.empty(50 * 32 + 1, device="cuda")[1:].view(50, 32).copy_(c)  # tables off their alignment
    b2 = empty_pages(2, 2, 32)
    int4_append_rope(b2, table, starts, None, k, v, odd, s, offsets)
    assert torch.equal(a, b2)


def test_append_rope_of_numbers_that_are_none():
    """Infinities and NaN in a group: stored as NaN, others untouched by them."""
    cos, sin = tables(4, 128)
    k = torch.ones(2, 1, D, dtype=torch.float16, device="cuda")
    k[0, 0, 70] = float("inf")  # turned with channel 6: groups 0 and 2
    v = torch.ones_like(k)
    v[1, 0, 40] = float("nan")
    pool = empty_pages(1, 1, 32)
    int4_append_rope(pool, i32([[0]]), i32([1]), None, k, v, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), i32([0, 2]))
    ko, vo = int4_gather(pool, i32([[0]]), i32([1]), i32([0, 2]), 2)
    nan = torch.isnan(ko[0, 0]).view(4, 32)
    assert nan.all(1).tolist() == [True, False, True, False] and not nan[1].any() and not nan[3].any()
    assert not torch.isnan(ko[1]).any() and torch.isnan(vo[1, 0]).view(4, 32).all(1).tolist() == [False, True, False, False]


# -- masks -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("seed", range(4))
def test_draft_tree(seed):
    rng = np.random.default_rng(seed)
    new = [int(x) for x in rng.integers(0, 65, 7)] + [64, 1]
    trees = [random_parents(rng, n) for n in new]
    trees[-2] = [i - 1 for i in range(64)]  # the deepest
    if seed == 1:  # parents that are none: themselves, later ones, far ones
        trees[0] = [5, 0, 2, 9, -7, 1 << 30, 3][: len(trees[0])] + trees[0][7:]
    first = 3
    parents = [9] * first + [p for t in trees for p in t] + [0, 0]
    offsets = i32((sums(new) + first).tolist())
    starts = [int(x) for x in rng.integers(0, 100, len(new))]
    seen, positions = draft_tree(i32(parents), offsets, i32(starts))
    want = [m for t in trees for m in ref.masks(t)]
    assert seen[first: -2].tolist() == signed(want).tolist()
    depth = [bin(m).count("1") - 1 for m in want]
    assert positions[first: -2].tolist() == [d + s for d, s in zip(depth, np.repeat(starts, new))]
    assert seen[:first].tolist() == [0] * first and seen[-2:].tolist() == [0, 0]
    assert draft_tree(i32(parents), offsets)[1][first: -2].tolist() == depth


# -- attention ---------------------------------------------------------------------------------------------

def attention_case(seed, contexts, new, heads, ratio, page, chain=False, spread=0.5, missing=()):
    """Inputs of a call and, from the stored values in 64 bits, its rows and bounds; pages in ``missing`` (sequence,
    entry) are not there."""
    rng = np.random.default_rng(seed)
    lengths = [a + b for a, b in zip(contexts, new)]
    n, total = sum(new), sum(lengths)
    scale = np.exp(spread * rng.standard_normal((1, heads, D)))
    k = (rng.standard_normal((total, heads, D)) * scale).astype(np.float16)
    v = rng.standard_normal((total, heads, D)).astype(np.float16)
    q = rng.standard_normal((n, heads * ratio, D)).astype(np.float16)
    table, pages = page_table(rng, lengths, page)
    pool = torch.randint(256, empty_pages(pages, heads, page).shape, dtype=torch.uint8, device="cuda",
                         generator=torch.Generator("cuda").manual_seed(seed))  # what lies behind a sequence may be anything
    if total:
        int4_append(pool, table, i32([0] * len(new)), torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32(sums(lengths).tolist()))
    for s, e in missing:
        table[s, e] = -1
    trees = [random_parents(rng, m) for m in new]
    masks = [m for t in trees for m in ref.masks([i - 1 for i in range(len(t))] if chain else t)]
    (kd, ks), (vd, vs) = stored(k), stored(v)
    out, bound = np.zeros((n, heads * ratio, D)), np.full((n, heads * ratio, D), 2.0 ** -24)
    at = row = 0
    for s, (c, m) in enumerate(zip(contexts, new)):
        visible = np.ones((m, c + m), bool)
        for i in range(m):
            for j in range(m):
                visible[i, c + j] = masks[row + i] >> j & 1
        for _, e in (x for x in missing if x[0] == s):
            visible[:, e * page: (e + 1) * page] = False
        r = slice(at, at + c + m)
        out[row: row + m], bound[row: row + m] = ref.tree_attention(q[row: row + m].astype(np.float64), kd[r], vd[r], visible, D ** -0.5,
                                                                    ks[r], vs[r])
        at, row = at + c + m, row + m
    args = dict(q=torch.from_numpy(q).cuda(), pages=pool, table=table, lengths=i32(lengths), offsets=i32(sums(new).tolist()),
                seen=None if chain else signed(masks))
    return args, out, bound


def within(got, out, bound):
    bad = np.abs(got.float().cpu().numpy() - out) - bound
    assert (bad <= 0).all(), f"{(bad > 0).sum()} of {bad.size} past their bounds, by up to {bad.max()}"


CASES = [  # contexts, nodes, KV heads, ratio, page
    ([0], [1], 1, 1, 32),
    ([0, 5], [7, 0], 1, 2, 32),
    ([31, 32, 33], [1, 1, 1], 2, 4, 64),
    ([60], [8], 2, 4, 64),
    ([1000], [4], 2, 4, 32),
    ([300, 0, 17], [16, 64, 5], 2, 1, 64),
    ([97, 640], [64, 33], 1, 4, 128),
    ([1, 2, 3, 4, 5], [3, 40, 2, 1, 21], 3, 3, 32),
    ([500, 90], [11, 29], 1, 8, 256),
    ([70], [64], 1, 7, 64),
    ([2000], [2], 8, 1, 64),
]


@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
@pytest.mark.parametrize("chain", [False, True])
def test_tree_attention(case, chain):
    args, out, bound = attention_case(sum(case[0]) + case[3], *case, chain=chain)
    within(int4_tree_attention(**args), out, bound)
    nodes, most = max(case[1]), max(a + b for a, b in zip(case[0], case[1]))
    within(int4_tree_attention(**args, max_nodes=nodes, max_length=most), out, bound)


def test_tree_attention_of_many_sequences():
    rng = np.random.default_rng(7)
    contexts, new = [int(x) for x in rng.integers(0, 150, 70)], [int(x) for x in rng.integers(0, 6, 70)]
    args, out, bound = attention_case(11, contexts, new, 2, 2, 64)
    within(int4_tree_attention(**args), out, bound)


def test_tree_attention_reads_no_page_that_is_not_there():
    args, out, bound = attention_case(5, [130, 40], [6, 3], 2, 2, 32, missing=[(0, 1), (0, 4), (1, 0), (1, 1)])
    within(int4_tree_attention(**args), out, bound)
    args["table"][0, 0] = 1 << 30
    args["table"][0, 2:] = -5
    assert (int4_tree_attention(**args) == 0).all()


def test_tree_attention_is_that_of_single_tokens():
    """A root alone is a decode step: int4_attention's result up to the roundings of V and the weights."""
    from reskv_amd.int4 import int4_attention

    args, out, bound = attention_case(9, [700, 33, 64], [1, 1, 1], 2, 4, 64)
    got = int4_tree_attention(**args)
    single = int4_attention(args["q"], args["pages"], args["table"], args["lengths"])
    within(got, out, bound)
    within(single, out, 2 * bound)


def test_masks_hide_and_rows_may_be_empty():
    """Masks need be no tree: nothing at all, not even itself; bits behind the last node are nobody's."""
    args, _, _ = attention_case(3, [0, 64], [5, 3], 1, 2, 64)
    args["seen"] = signed([0, 0b10000, 0b1, 0, (1 << 64) - 1, 0, 0b100, 0b1000])
    got = int4_tree_attention(**args)
    assert (got[[0, 3]] == 0).all() and (got[[1, 2, 4]] != 0).any(-1).all()
    # row 4 sees the five nodes, row 7 only its context (bit 3 is behind the last node)
    args["seen"][4] = 0b11111
    args["seen"][7] = 0
    assert torch.equal(got, int4_tree_attention(**args))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("of", ["k", "v"])
def test_what_a_node_does_not_see_does_not_matter(bad, of):
    """Nodes 2 and 5 hold no numbers: only the rows that see them show it, and V's only in the group's channels."""
    rng = np.random.default_rng(1)
    parents = [-1, 0, 1, 0, 3, 2, 4]
    k, v = (torch.from_numpy(rng.standard_normal((47, 2, D)).astype(np.float16)).cuda() for _ in range(2))
    clean, dirty = empty_pages(2, 2, 32), empty_pages(2, 2, 32)
    q = torch.from_numpy(rng.standard_normal((7, 4, D)).astype(np.float16)).cuda()
    table = i32([[1, 0]])
    args = dict(table=table, lengths=i32([47]), offsets=i32([0, 7]), seen=draft_tree(i32(parents), i32([0, 7]))[0])
    int4_append(clean, table, i32([0]), k, v, i32([0, 47]))
    (k if of == "k" else v)[[42, 45], :, 37] = bad
    int4_append(dirty, table, i32([0]), k, v, i32([0, 47]))
    a, b = int4_tree_attention(q, clean, **args), int4_tree_attention(q, dirty, **args)
    sees = [2, 5]
    rest = [i for i in range(7) if i not in sees]
    assert torch.equal(a[rest], b[rest])
    wrong = torch.isnan(b[sees]).view(2, 4, 4, 32)
    if of == "k":
        assert wrong.all()
    else:
        assert wrong[:, :, 1].all() and torch.equal(b[sees].view(2, 4, 4, 32)[:, :, [0, 2, 3]], a[sees].view(2, 4, 4, 32)[:, :, [0, 2, 3]])


def test_values_at_the_ends_of_fp16():
    """A group's largest value may come out past fp16's by the rounding of its scale: it stays a number, also for rows
    that barely see it."""
    v = torch.zeros(40, 1, D, dtype=torch.float16, device="cuda")
    v[:, :, ::2], v[:, :, 1::2] = -65504.0, 65504.0
    k = torch.zeros_like(v)
    k[3] = 1.0
    pool, table = empty_pages(2, 1, 32), i32([[0, 1]])
    int4_append(pool, table, i32([0]), k, v, i32([0, 40]))
    q = torch.ones(2, 1, D, dtype=torch.float16, device="cuda")
    got = int4_tree_attention(q, pool, table, i32([40]), i32([0, 2]))
    assert torch.isfinite(got).all() and (got[..., 1::2] >= 65400).all() and (got[..., ::2] <= -65400).all()


def test_rows_of_no_sequence_and_nodes_past_the_last():
    args, out, bound = attention_case(4, [50, 20], [6, 4], 1, 2, 32)
    q = torch.cat([args["q"][:1], args["q"], args["q"][:2]])
    seen = torch.cat([args["seen"][:1], args["seen"], args["seen"][:2]])
    more = dict(args, q=q, seen=seen, offsets=args["offsets"] + 1)
    got = int4_tree_attention(**more)
    within(got[1:-2], out, bound)
    assert (got[0] == 0).all() and (got[-2:] == 0).all()
    kept = torch.full_like(q, 3.0)
    assert int4_tree_attention(**more, out=kept) is kept
    assert (kept[0] == 3).all() and (kept[-2:] == 3).all() and torch.equal(kept[1:-2], got[1:-2])
    few = int4_tree_attention(**more, max_nodes=4)  # six rows of the first sequence, of which four are worked on
    assert (few[5:7] == 0).all() and torch.equal(few[1:5], got[1:5]) and torch.equal(few[7:], got[7:])
    # lengths that are nothing, or more than the table holds
    none = int4_tree_attention(**dict(more, lengths=i32([-3, 24])))
    assert (none[:7] == 0).all() and torch.equal(none[7:-2], got[7:-2])
    cut = int4_tree_attention(**dict(more, lengths=i32([1 << 30, 24])), max_length=56)
    assert torch.equal(cut, got)


@pytest.mark.parametrize("offsets", [[0, -5, 10], [0, 99, 10], [7, 3, 10], [-9, 4, 99]])
def test_offsets_are_clamped(offsets):
    """Whatever the offsets hold, nothing outside the tensors is read or written."""
    args, _, _ = attention_case(4, [50, 20], [6, 4], 1, 2, 32)
    guard = torch.full((12, 2, D), 5.0, dtype=torch.float16, device="cuda")
    int4_tree_attention(**dict(args, offsets=i32(offsets)), out=guard[1:-1])
    assert (guard[0] == 5).all() and (guard[-1] == 5).all()


@pytest.mark.parametrize("power", [-20, -8, 6])
def test_queries_and_keys_of_other_sizes(power):
    """Heads whose queries are many powers of two apart; keys far from one."""
    args, _, _ = attention_case(8, [90], [6], 2, 2, 32)
    rng = np.random.default_rng(2)
    k = (rng.standard_normal((96, 2, D)) * 2.0 ** (power / 2)).astype(np.float16)
    v = (rng.standard_normal((96, 2, D)) * 2.0 ** np.arange(-8, 8).repeat(6)[:, None, None]).astype(np.float16)
    q = (rng.standard_normal((6, 4, D)) * 2.0 ** np.array([power, 0, -power, 3])[:, None]).clip(-60000, 60000).astype(np.float16)
    int4_append(args["pages"], args["table"], i32([0]), torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32([0, 96]))
    (kd, ks), (vd, vs) = stored(k), stored(v)
    visible = np.tri(6, 96, 90, dtype=bool)
    out, bound = ref.tree_attention(q.astype(np.float64), kd, vd, visible, 0.01, ks, vs)
    got = int4_tree_attention(torch.from_numpy(q).cuda(), args["pages"], args["table"], i32([96]), i32([0, 6]), scaling=0.01)
    within(got, out, bound)


@pytest.mark.parametrize("nodes", [2, 40])
@pytest.mark.parametrize("power", [-9, 0, 15])
def test_scores_of_keys_whose_groups_are_level(nodes, power):
    """Every key's channels of a group are equal, so that scores are sums of q times lowest values alone, and two groups' sums of q cancel
    but for a 2^-15 of them.

    In fp32 a sum of q takes up to ten roundings (four elements that are not zero, the lanes' shares), the products of two groups
    in three parts six, the scaling and the exponent two; a third part is off by 2^-25 of q's largest element and the lowest value: fewer
    than 32 half steps of 2^-24 of the terms' sum, which a weight is off by twice.  The rest as in drafts_reference.tree_attention."""
    rng = np.random.default_rng(100 + nodes + power)
    m, heads = 40 + nodes, 4
    sign = rng.choice([-1.0, 1.0], (m, 1, 1))
    k = np.zeros((m, 1, D))
    k[..., :64] = sign * 2.0 ** power * (1 + rng.integers(0, 900, (m, 1, 1)) / 1024)
    v = (sign * (1 + 0.1 * rng.standard_normal((m, 1, D)))).astype(np.float16)
    q = np.zeros((nodes, heads, D))
    q[..., 0], q[..., 32] = 1.0, -1.0
    for at in (1, 33):
        q[..., at: at + 3] = rng.uniform(-1, 1, (nodes, heads, 3)) * 2.0 ** -15
    q, k = (q * 2.0 ** min(15, 15 - power)).astype(np.float16), k.astype(np.float16)
    pool, table = empty_pages(4, 1, 32), i32([[2, 0, 1, 3]])
    int4_append(pool, table, i32([0]), torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32([0, m]))
    (kd, ks), (vd, vs) = stored(k), stored(v)
    assert np.array_equal(kd, k)
    visible = np.tri(nodes, m, 40, dtype=bool)
    out, _ = ref.tree_attention(q.astype(np.float64), kd, vd, visible, D ** -0.5, ks, vs)
    spread, _ = ref.tree_attention(q.astype(np.float64), kd, np.abs(vs), visible, D ** -0.5, ks, vs)
    delta = 32 * 2.0 ** -24 * D ** -0.5 * np.abs(q.astype(np.float64)).sum(-1).max() * np.abs(kd).max()
    bound = spread * (2 * 2.0 ** -11 + 2 * delta + 2.0 ** -20) * 1.01 + 2.0 ** -34 * vs.sum(0) + 2.0 ** -24 + 2.0 ** -11 * np.abs(out) * 1.01
    within(int4_tree_attention(torch.from_numpy(q).cuda(), pool, table, i32([m]), i32([0, nodes])), out, bound)


def test_long_context():
    """More blocks than waves, with a tree that is split over many of them; 64 bits on the GPU."""
    gen = torch.Generator("cuda").manual_seed(1)
    m, n = 70000, 9
    k, v = (torch.randn(m, 1, D, device="cuda", generator=gen).half() for _ in range(2))
    q = torch.randn(n, 4, D, device="cuda", generator=gen).half()
    pool = empty_pages(-(-m // 64), 1, 64)
    table = torch.randperm(pool.shape[0], device="cuda", generator=gen).int()[None]
    int4_append(pool, table, i32([0]), k, v, i32([0, m]))
    parents = [-1, 0, 0, 1, 1, 2, 3, 3, 5]
    got = int4_tree_attention(q, pool, table, i32([m]), i32([0, n]), signed(ref.masks(parents)))
    kd, vd = (torch.from_numpy(stored(x.cpu().numpy())[0]).cuda()[:, 0] for x in (k, v))
    s = torch.einsum("nhd,md->nhm", q.double(), kd) * D ** -0.5
    see = torch.ones(n, m, dtype=torch.bool, device="cuda")
    for i, mask in enumerate(ref.masks(parents)):
        for j in range(n):
            see[i, m - n + j] = bool(mask >> j & 1)
    w = torch.softmax(s.masked_fill(~see[:, None], -float("inf")), -1)
    # 70000 weights of about 1 / 70000: rounding errors of V and weights average out to well below fp16's step of the result
    assert (got.double() - w @ vd).abs().max() <= 2.0 ** -11 * (w @ vd).abs().max() + 2.0 ** -11 * (w @ vd.abs()).max()


# -- verification --------------------------------------------------------------------------------------------

def verify_case(seed, new, vocab, temperature, drawn, fp32=False, ties=False, padding=0):
    rng = np.random.default_rng(seed)
    n = sum(new)
    logits = (3 * rng.standard_normal((n, vocab))).astype(np.float32 if fp32 else np.float16)
    if ties:
        logits = np.rint(logits).clip(-3, 3).astype(logits.dtype)
    hidden = rng.random((n, vocab)) < 0.1
    hidden[np.arange(n), rng.integers(0, vocab, n)] = False
    logits[hidden] = -np.inf
    trees = [random_parents(rng, m) for m in new]
    parents = np.array([p for t in trees for p in t], np.int32)
    above = np.concatenate([f + np.maximum(t, 0) for f, t in zip(sums(new), trees)]).astype(int) if n else np.zeros(0, int)
    q = None
    tokens = np.zeros(n, np.int64)
    for i in range(n):
        near = ref.softmax(logits[above[i]].astype(np.float64), max(temperature, 0.5) * 1.3)
        if drawn:
            if q is None:
                q = np.zeros((n, vocab), np.float32)
            near = near * np.exp(0.5 * rng.standard_normal(vocab))
            q[i] = near / near.sum()
            near = q[i].astype(np.float64) / q[i].astype(np.float64).sum()
        tokens[i] = rng.choice(vocab, p=near)
        if temperature == 0.0 and rng.random() < 0.6:
            tokens[i] = np.argmax(logits[above[i]])
    accept, sample = rng.random(n, np.float32), rng.random(len(new), np.float32)
    full = torch.zeros(n, vocab + padding, dtype=torch.float32 if fp32 else torch.float16, device="cuda")
    full[:, :vocab] = torch.from_numpy(logits).cuda()
    args = dict(logits=full[:, :vocab], tokens=torch.from_numpy(tokens).cuda(), parents=i32(parents.tolist()),
                offsets=i32(sums(new).tolist()), accept=torch.from_numpy(accept).cuda(), sample=torch.from_numpy(sample).cuda(),
                draft=None if q is None else torch.from_numpy(q).cuda(), temperature=temperature)
    return args, (logits, tokens, parents, accept, sample, q)


def check_verify(args, host, new, close=1e-9):
    """Equal to the walk in 64 bits but where a decision comes so near to its border that roundings may decide it."""
    path, counts, token = (x.cpu().numpy() for x in verify_drafts(**args))
    logits, tokens, parents, accept, sample, q = host
    lengths = []
    for s, (f, m) in enumerate(zip(sums(new), new)):
        r = slice(f, f + m)
        want, last, margin = ref.verify(logits[r].astype(np.float64), tokens[r], parents[r], accept[r], sample[s], None if q is None else q[r],
                                        args["temperature"])
        if margin < close:
            continue
        assert counts[s] == len(want) and path[s].tolist() == want + [-1] * (64 - len(want)), s
        assert token[s] == last, s
        lengths.append(len(want))
    return lengths


VERIFY = [  # nodes, vocabulary
    ([1], 1),
    ([5], 7),
    ([1, 64, 0, 9], 100),
    ([20, 3, 40], 1000),
    ([6] * 10, 2049),
    ([12, 12], 8191),
    ([8], 50001),
]


@pytest.mark.parametrize("case", VERIFY, ids=range(len(VERIFY)))
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0, 2.5])
@pytest.mark.parametrize("fp32", [False, True])
def test_verify(case, drawn, temperature, fp32):
    new, vocab = case
    args, host = verify_case(sum(new) + vocab, new, vocab, temperature, drawn, fp32)
    check_verify(args, host, new)


@pytest.mark.parametrize("seed", range(6))
def test_verify_of_many_trees(seed):
    """Small vocabularies: siblings with the same token, rows where little is left, long paths."""
    rng = np.random.default_rng(seed)
    new = [int(x) for x in rng.integers(0, 40, 60)]
    vocab = [2, 3, 5, 17, 300, 2500][seed]
    for temperature, drawn in ((1.0, False), (1.0, True), (0.3, True), (0.0, False)):
        args, host = verify_case(seed, new, vocab, temperature, drawn, ties=True, padding=seed)
        lengths = check_verify(args, host, new)
        assert max(lengths) >= (3 if vocab <= 17 else 1)  # one-hot drafts of wide vocabularies are mostly turned down


def test_verify_takes_the_lowest_of_equals():
    logits = torch.zeros(1, 9000, dtype=torch.float16, device="cuda")
    for at in ([8999, 4, 5000], [8191, 8192], [0, 8999], [2047, 2048, 2049]):
        row = logits.clone()
        row[0, at] = 2.0
        assert verify_drafts(row, torch.zeros(1, dtype=torch.int64, device="cuda"), i32([-1]), i32([0, 1]), temperature=0)[2].tolist() == [min(at)]


def test_verify_where_nothing_is_left():
    """A draft that is certain to the target is accepted; all siblings turned down leave the others' probability; the last token
    with any probability is the end of a walk that samples past it."""
    logits = torch.full((4, 3000), -float("inf"), dtype=torch.float16, device="cuda")
    logits[0, [5, 2500]] = 0.0
    logits[1:, 7] = 1.0
    tokens = torch.tensor([0, 5, 2500, 7], device="cuda")
    args = dict(parents=i32([-1, 0, 0, 2]), offsets=i32([0, 4]), sample=torch.tensor([0.999], device="cuda"))
    path, counts, token = verify_drafts(logits, tokens, accept=torch.tensor([0.0, 0.6, 0.99, 0.999], device="cuda"), **args)
    assert path[0, :4].tolist() == [0, 2, 3, -1] and counts.tolist() == [3] and token.tolist() == [7]
    # 2500 is turned down by a number that no generator gives: nothing would be left, so that it stays
    path, counts, token = verify_drafts(logits, tokens, accept=torch.tensor([0.0, 0.6, 1.5, 0.9], device="cuda"), **args)
    assert counts.tolist() == [1] and token.tolist() == [2500]
    # a draft of which 2^-40 is left
    wide = torch.zeros(2, 40, dtype=torch.float32, device="cuda")
    wide[0, 3] = 40 * 0.6931472 + 3.7
    u = torch.tensor([0.0, 1.0], device="cuda")
    for sample, want in ((0.0, 0), (0.5 / 39, 0), (1.5 / 39, 1), (2.9 / 39, 2), (3.1 / 39, 4), (38.5 / 39, 39)):
        got = verify_drafts(wide, torch.tensor([0, 3], device="cuda"), i32([-1, 0]), i32([0, 2]), u, torch.tensor([sample], device="cuda"))
        assert got[1].tolist() == [1] and got[2].tolist() == [want]


@pytest.mark.parametrize("fp32", [False, True])
def test_verify_where_all_of_a_segment_is_turned_down(fp32):
    """The siblings that were turned down are all that the row has among its first tokens: what rounding leaves of their sum is no
    token, and a walk that samples at 0 ends with the first of the others."""
    rng = np.random.default_rng(3)
    count, vocab = 60, 9001
    logits = np.full((4 * count, vocab), -np.inf, np.float32 if fp32 else np.float16)
    logits[0::4, 8000] = logits[0::4, 8999] = 0.0
    for at in (3, 70, 900):
        logits[0::4, at] = rng.uniform(-4, 1, count)
    logits[:, 8000] = 0.0
    tokens = torch.tensor([0, 3, 70, 900] * count, device="cuda")
    accept = torch.tensor([0.0, 0.999, 0.9995, 0.9999] * count, device="cuda")
    path, counts, token = verify_drafts(torch.from_numpy(logits).cuda(), tokens, i32([-1, 0, 0, 0] * count), i32(list(range(0, 4 * count + 1, 4))),
                                        accept, torch.zeros(count, device="cuda"))
    assert (counts == 1).all() and (token == 8000).all()


def test_verify_rows_without_a_distribution():
    rng = np.random.default_rng(0)
    good = rng.standard_normal((6, 4000)).astype(np.float16)
    bad = good.copy()
    bad[1, 77] = np.nan
    bad[2, :] = -np.inf
    bad[3, 3999] = np.inf
    logits = torch.from_numpy(bad).cuda()
    tokens, parents = torch.zeros(6, dtype=torch.int64, device="cuda"), i32([-1] * 6)
    offsets, u = i32([0, 1, 2, 3, 4, 4, 5, 6]), torch.full((7,), 0.5, device="cuda")
    path, counts, token = verify_drafts(logits, tokens, parents, offsets, u[:6], u)
    assert (token >= 0).tolist() == [True, False, False, False, False, True, True]
    assert counts.tolist() == [1, 1, 1, 1, 0, 1, 1] and (path[4] == -1).all()
    greedy = verify_drafts(logits, tokens, parents, offsets, temperature=0)[2].tolist()
    assert greedy == [int(np.argmax(good[0])), -1, 0, 3999, -1, int(np.argmax(good[4])), int(np.argmax(good[5]))]


def test_verify_passes_over_what_is_no_token_or_no_parent():
    logits = torch.zeros(7, 10, dtype=torch.float16, device="cuda")
    logits[:, 4] = 5.0
    tokens = torch.tensor([4, 10, -1, 4, 4, 1 << 40, 4], device="cuda")
    parents = i32([-1, 0, 0, 3, 5, 0, 0])  # node 3 is its own parent, node 4 has a later one
    path, counts, token = verify_drafts(logits, tokens, parents, i32([0, 7]), temperature=0)
    assert path[0, :3].tolist() == [0, 6, -1] and counts.tolist() == [2] and token.tolist() == [4]
    u = torch.zeros(7, device="cuda")
    path, counts, token = verify_drafts(logits, tokens, parents, i32([0, 7]), u, u[:1] + 0.5)
    assert path[0, :3].tolist() == [0, 6, -1] and token.tolist() == [4]


def test_verified_tokens_are_distributed_as_the_targets():
    """The token behind the root, accepted or sampled, over 40000 sequences of two siblings: every frequency within five
    standard deviations of the target's probability, for both ways of drafting."""
    count, vocab = 40000, 5
    gen = torch.Generator("cuda").manual_seed(0)
    p = torch.tensor([0.4, 0.05, 0.25, 0.2, 0.1], device="cuda")
    q = torch.tensor([0.1, 0.3, 0.3, 0.05, 0.25], device="cuda")
    logits = p.log().expand(3 * count, vocab).contiguous()
    parents, offsets = i32([-1, 0, 0] * count), torch.arange(0, 3 * count + 1, 3, dtype=torch.int32, device="cuda")
    for drawn in (False, True):
        tokens = torch.multinomial(q.expand(3 * count, vocab), 1, generator=gen)[:, 0]
        if not drawn:
            tokens = torch.randint(vocab, (3 * count,), device="cuda", generator=gen)
        path, counts, token = verify_drafts(logits, tokens, parents, offsets, torch.rand(3 * count, device="cuda", generator=gen),
                                            torch.rand(count, device="cuda", generator=gen),
                                            draft=q.expand(3 * count, vocab).contiguous() if drawn else None)
        first = torch.where(counts > 1, tokens.view(count, 3).gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token)
        share = torch.bincount(first, minlength=vocab) / count
        assert ((share - p).abs() <= 5 * (p * (1 - p) / count).sqrt()).all(), share


# -- keep ------------------------------------------------------------------------------------------------------

def kept_reference(pool, table, page, starts, path, counts):
    """The pool's stored numbers after the move, from the documented layout: token by token, out of a copy."""
    layers, _, heads, _ = pool.shape
    old, new = pool.reshape(*pool.shape[:3], page // 32, 5120), pool.reshape(*pool.shape[:3], page // 32, 5120).copy()
    byte = [(4 * (e // 2 + 4 * (e % 2))) // 8 for e in range(8)]
    shift = [(4 * (e // 2 + 4 * (e % 2))) % 8 for e in range(8)]

    def token(blocks, s, t):
        if t < 0 or t // page >= table.shape[1] or not 0 <= table[s, t // page] < pool.shape[1]:
            return None
        b = blocks[:, table[s, t // page], :, t % page // 32]
        t %= 32
        keys, scales = b[..., :2048].reshape(layers, heads, 2, 4, 16, 16), b[..., 2048:2560].reshape(layers, heads, 2, 4, 16, 4)
        values, rest = b[..., 2560:4608].reshape(layers, heads, 2, 4, 16, 4, 4), b[..., 4608:].reshape(layers, heads, 8, 32, 2)
        return (keys[:, :, t // 16, :, t % 16], scales[:, :, t // 16, :, t % 16], rest[:, :, :, t],
                values[:, :, :, t // 8, :, :, byte[t % 8]], shift[t % 8])

    def put(s, t, data):
        blocks = new
        p, b, u = table[s, t // page], t % page // 32, t % 32
        view = blocks[:, p, :, b]
        view[..., :2048].reshape(layers, heads, 2, 4, 16, 16)  # (a copy: written through indices below)
        k = view[..., :2048].reshape(layers, heads, 2, 4, 16, 16).copy()
        k[:, :, u // 16, :, u % 16] = data[0]
        c = view[..., 2048:2560].reshape(layers, heads, 2, 4, 16, 4).copy()
        c[:, :, u // 16, :, u % 16] = data[1]
        v = view[..., 2560:4608].reshape(layers, heads, 2, 4, 16, 4, 4).copy()
        r = view[..., 4608:].reshape(layers, heads, 8, 32, 2).copy()
        r[:, :, :, u] = data[2]
        at = v[:, :, :, u // 8, :, :, byte[u % 8]]
        v[:, :, :, u // 8, :, :, byte[u % 8]] = at & ~np.uint8(15 << shift[u % 8]) | ((data[3] >> data[4] & 15) << shift[u % 8])
        blocks[:, p, :, b] = np.concatenate([x.reshape(layers, heads, -1) for x in (k, c, v, r)], -1)

    for s, (start, count) in enumerate(zip(starts, counts)):
        for j in range(min(count, path.shape[1])):
            if not 0 <= path[s, j] < 64 or path[s, j] == j:
                continue
            data = token(old, s, start + path[s, j])
            if data is not None and token(new, s, start + j) is not None:
                put(s, start + j, data)
    return new.reshape(pool.shape)


@pytest.mark.parametrize("seed", range(8))
def test_keep(seed):
    rng = np.random.default_rng(seed)
    page, heads, layers = [32, 64, 96, 256][seed % 4], [1, 2, 3][seed % 3], [1, 3][seed % 2]
    starts = [int(x) for x in rng.integers(0, 150, 5)]
    new = [int(x) for x in rng.integers(1, 65, 5)]
    width = max(new)
    path, counts = np.full((5, width), -1, np.int32), []
    for s, n in enumerate(new):
        c = int(rng.integers(0, n + 1))
        row = rng.permutation(n)[:c] if seed % 2 else np.sort(rng.permutation(n)[:c])  # any order will do
        path[s, :c] = row
        counts.append(c)
    table, pages = page_table(rng, [a + b for a, b in zip(starts, new)], page)
    if seed == 5:
        path[0, 0], path[1, :1], counts[2] = 64, -9, width + 7
        path[3, :counts[3]] = path[3, 0]  # one node several times
        table[4, 0] = -1
    pool = torch.randint(256, (layers, pages, heads, page * 160), dtype=torch.uint8, device="cuda",
                         generator=torch.Generator("cuda").manual_seed(seed))
    want = kept_reference(pool.cpu().numpy(), table.cpu().numpy(), page, starts, path, counts)
    int4_keep(pool if layers > 1 else pool[0], table, i32(starts), torch.from_numpy(path).cuda(), i32(counts))
    assert np.array_equal(pool.cpu().numpy(), want)


def test_kept_values_read_back():
    """Through the other operators: what a gather gives of the kept tokens is what it gave of them before."""
    rng = np.random.default_rng(2)
    k, v = (torch.from_numpy(rng.standard_normal((90, 2, D)).astype(np.float16)).cuda() for _ in range(2))
    pool, table = empty_pages(3, 2, 32), i32([[2, 0, 1]])
    int4_append(pool, table, i32([0]), k, v, i32([0, 90]))
    before = int4_gather(pool, table, i32([0]), i32([0, 90]), 90)
    path = [0, 3, 4, 17, 40, 59]
    int4_keep(pool, table, i32([30]), i32([path]), i32([6]))
    after = int4_gather(pool, table, i32([0]), i32([0, 90]), 90)
    order = list(range(30)) + [30 + p for p in path] + list(range(36, 90))
    for a, b in zip(after, before):
        assert torch.equal(a, b[order])


# -- graphs, streams, devices ------------------------------------------------------------------------------------

def test_a_step_in_a_graph():
    """All operators captured, replayed with other inputs between eager work, and two graphs that share a pool."""
    rng = np.random.default_rng(0)
    new, contexts, heads, vocab = [6, 6], [70, 33], 2, 3001
    table, pages = page_table(rng, [c + 6 for c in contexts], 32)
    pool = empty_pages(pages, heads, 32)
    starts, lengths, offsets = i32(contexts), i32([c + 6 for c in contexts]), i32(sums(new).tolist())
    old = [torch.from_numpy(rng.standard_normal((103, heads, D)).astype(np.float16)).cuda() for _ in range(2)]
    int4_append(pool, table, i32([0, 0]), *old, i32([0, 70, 103]))
    cos, sin = (torch.from_numpy(x).cuda() for x in tables(80, 128))
    q, k, v = (torch.empty(12, h, D, dtype=torch.float16, device="cuda") for h in (8, heads, heads))
    logits = torch.empty(12, vocab, dtype=torch.float16, device="cuda")
    tokens, parents = torch.empty(12, dtype=torch.int64, device="cuda"), i32([-1, 0, 0, 1, 2, 3] * 2)
    accept, sample = torch.empty(12, device="cuda"), torch.empty(2, device="cuda")

    def fill(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        for t in (q, k, v, logits):
            t.normal_(generator=g)
        tokens.random_(0, vocab, generator=g)
        tokens[1] = logits[0].argmax()
        accept.uniform_(generator=g)
        accept[1] = 0.0
        sample.uniform_(generator=g)

    def step():
        seen, positions = draft_tree(parents, offsets, starts)
        turned = int4_append_rope(pool, table, starts, q, k, v, cos, sin, offsets, positions=positions)
        out = int4_tree_attention(turned, pool, table, lengths, offsets, seen)
        path, counts, token = verify_drafts(logits, tokens, parents, offsets, accept, sample)
        greedy = verify_drafts(logits, tokens, parents, offsets, temperature=0)
        int4_keep(pool, table, starts, path, counts)
        return [turned, out, path, counts, token, *greedy, pool.clone()]

    base = pool.clone()
    fill(0)
    step()
    side, memory = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, pool=memory, stream=side):
            outs = step()
        graphs.append((g, outs))
    for seed in (1, 2, 3, 4):
        fill(seed)
        pool.copy_(base)
        want = [x.clone() for x in step()]
        g, outs = graphs[seed % 2]
        pool.copy_(base)
        torch.cuda.synchronize()
        g.replay()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        assert want[3][0] >= 2


def test_another_stream():
    args, out, bound = attention_case(6, [400], [9], 2, 4, 64)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1000000)
        q = args["q"] * 1.0
        got = int4_tree_attention(**dict(args, q=q))
    side.synchronize()
    within(got, out, bound)


def test_append_rope_has_the_bits_of_the_decoder_steps():
    """A decode step both ways: fused_qkv_rope and int4_append, int4_append_rope."""
    from reskv_amd.llama import fused_qkv_rope

    b, hq, hk, pos = 5, 8, 2, 45
    qkv = torch.randn(b, (hq + 2 * hk) * D, device="cuda", generator=torch.Generator("cuda").manual_seed(9)).half()
    cos, sin = (torch.from_numpy(x).cuda() for x in tables(64, 128))
    q, qr = (torch.empty(b, hq, D, dtype=torch.float16, device="cuda") for _ in range(2))
    k, kr, v = (torch.empty(b, hk, D, dtype=torch.float16, device="cuda") for _ in range(3))
    fused_qkv_rope(qkv, cos, sin, torch.tensor([pos], device="cuda"), q, qr, k, kr, v)
    starts, table = i32([pos] * b), torch.arange(2 * b, dtype=torch.int32, device="cuda").view(b, 2)
    one, two = empty_pages(2 * b, hk, 32), empty_pages(2 * b, hk, 32)
    int4_append(one, table, starts, kr, v)
    rows = qkv.view(b, -1, D)
    out = int4_append_rope(two, table, starts, rows[:, :hq], rows[:, hq: hq + hk], rows[:, hq + hk:], cos, sin)
    assert torch.equal(out, qr) and torch.equal(one, two)


@pytest.mark.parametrize("nodes", [2, 40])
def test_values_past_the_ends_of_fp16_mix(nodes):
    """Tokens at both ends of fp16 in one block with ordinary ones, few rows and many: a row's result is their average."""
    rng = np.random.default_rng(nodes)
    m = 70 + nodes
    v = rng.standard_normal((m, 1, D)).astype(np.float16)
    v[40, :, ::2], v[40, :, 1::2] = 65504.0, -65504.0
    v[41] = -v[40]
    k = rng.standard_normal((m, 1, D)).astype(np.float16)
    q = rng.standard_normal((nodes, 8, D)).astype(np.float16)
    pool, table = empty_pages(4, 1, 32), i32([[2, 0, 1, 3]])
    int4_append(pool, table, i32([0]), torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32([0, m]))
    (kd, ks), (vd, vs) = stored(k), stored(v)
    out, bound = ref.tree_attention(q.astype(np.float64), kd, vd, np.tri(nodes, m, 70, dtype=bool), D ** -0.5, ks, vs)
    within(int4_tree_attention(torch.from_numpy(q).cuda(), pool, table, i32([m]), i32([0, nodes])), out, bound)


@pytest.mark.parametrize("nodes,heads", [(1, 1), (2, 4), (9, 4), (24, 4), (40, 4)])
def test_values_past_the_ends_of_fp16_do_not_depend_on_the_rows(nodes, heads):
    """A step of 8736 (131008 / 15 in fp16) takes the largest code to 65536: two tokens of one weight at opposite ends have the average
    16 in every channel, with every sum exact, however many rows there are; blocks before and behind have no such tokens."""
    v = torch.full((110 + nodes, 1, D), 65504.0, dtype=torch.float16, device="cuda")
    v[:, :, ::2] = -65504.0
    v[33] = -v[33]
    k = torch.zeros_like(v)
    k[:32] = k[34:110] = -1.0
    v[:32] = v[64:110] = 0.0
    held = stored(v[32:34].cpu().numpy())[0]
    assert (held.max(axis=-1) == 65536.0).all() and (held.mean(axis=0) == 16.0).all()
    pool, table = empty_pages(5, 1, 32), i32([[2, 0, 1, 3, 4]])
    int4_append(pool, table, i32([0]), k, v, i32([0, 110 + nodes]))
    q = torch.full((nodes, heads, D), 8.0, dtype=torch.float16, device="cuda")  # the other tokens' weights are exp(-90): nothing
    hidden = torch.zeros(nodes, dtype=torch.int64, device="cuda")
    got = int4_tree_attention(q, pool, table, i32([110 + nodes]), i32([0, nodes]), hidden)
    assert (got == 16.0).all()


def test_pages_past_32_bits_of_bytes():
    """A pool of more than 4 GB, its last pages in use: appended, attended, read back and moved where they are."""
    heads, page, count = 8, 64, 56000
    pool = torch.zeros(count, heads, page * 160, dtype=torch.uint8, device="cuda")
    assert pool.numel() > 1 << 32
    table, small = i32([[count - 1, count - 3], [count - 2, 5]]), i32([[0, 1], [2, 3]])
    other = empty_pages(4, heads, page)
    rng = np.random.default_rng(6)
    n, starts, offsets = 70, i32([10, 40]), i32([0, 60, 70])
    q, k, v = (torch.from_numpy(rng.standard_normal((n, h, D)).astype(np.float16)).cuda() for h in (16, heads, heads))
    cos, sin = (torch.from_numpy(x).cuda() for x in tables(200, 128))
    got = []
    for p, t in ((pool, table), (other, small)):
        turned = int4_append_rope(p, t, starts, q, k, v, cos, sin, offsets)
        out = int4_tree_attention(turned, p, t, i32([70, 50]), offsets)
        int4_keep(p, t, starts, i32([[0, 3, 59], [2, 9, -1]]), i32([3, 2]))
        got.append([turned, out, *int4_gather(p, t, starts, offsets, n)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert not pool[6: count - 3].any()


def test_logits_past_32_bits_of_elements():
    n, vocab = 17000, 128256
    logits = torch.full((n, vocab), -5.0, dtype=torch.float16, device="cuda")
    assert logits.numel() > 1 << 31
    logits[n - 2, 77], logits[n - 1, vocab - 1] = 9.0, 8.0
    tokens = torch.zeros(n, dtype=torch.int64, device="cuda")
    tokens[n - 1] = 77
    parents, offsets = i32([-1] * (n - 1) + [0]), i32([0, n - 2, n])
    u = torch.zeros(n, device="cuda")
    for args in (dict(temperature=0), dict(accept=u, sample=torch.tensor([0.5, 0.9999999], device="cuda"))):
        path, counts, token = verify_drafts(logits, tokens, parents, offsets, **args)
        assert path[1, :3].tolist() == [0, 1, -1] and counts[1] == 2 and token[1] == vocab - 1


@pytest.mark.parametrize("vocab", [2041, 2048, 2049, 16383, 131058, 131064, 131071, 131072, 262143])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("fp32", [False, True])
def test_verify_at_the_ends_of_segments(vocab, drawn, fp32):
    """The probability lies on a row's first and last tokens and on both sides of multiples of 2048, in rows at every place relative
    to 16 bytes; siblings are turned down there.  Every token at the end of a row may be the largest."""
    for padding in (0, 1):
        rng = np.random.default_rng(1000 * padding + 2 * drawn + fp32)
        new = [4, 5]
        args, (logits, tokens, parents, accept, sample, q) = verify_case(vocab + padding, new, vocab, 1.0, drawn, fp32, padding=padding)
        at = 2048 * rng.integers(1, vocab // 2048 + 2, 4)[:, None] + np.arange(-8, 3)
        at = np.unique(np.concatenate([at.reshape(-1), np.arange(4), vocab - 1 - np.arange(9)]))
        at = at[(at >= 0) & (at < vocab)]
        logits[:, at] = (np.log(vocab) + 6 + rng.standard_normal((sum(new), at.size))).astype(logits.dtype)
        share = np.mean([ref.softmax(row, 1.0)[at].sum() for row in logits])
        assert share > 0.5
        tokens[:] = rng.choice(at, sum(new))
        if drawn:  # half of each draft's distribution on these tokens, the other as it was
            q *= 0.5
            q[:, at] += (0.5 * rng.dirichlet(np.ones(at.size), sum(new))).astype(np.float32)
            args["draft"].copy_(torch.from_numpy(q))
        args["logits"].copy_(torch.from_numpy(logits))
        args["tokens"].copy_(torch.from_numpy(tokens))
        check_verify(args, (logits, tokens, parents, accept, sample, q), new)
        logits[np.arange(sum(new)), vocab - 1 - np.arange(sum(new)) % 9] = 100.0
        args["logits"].copy_(torch.from_numpy(logits))
        tokens[:] = np.argmax(logits, axis=1)[np.maximum(parents, 0) + np.repeat(sums(new)[:-1], new)]
        args["tokens"].copy_(torch.from_numpy(tokens))
        check_verify({**args, "temperature": 0.0}, (logits, tokens, parents, accept, sample, q), new)


def test_calls_on_two_streams_at_once():
    """Calls that overlap share nothing: each stream's results are those of a call alone."""
    cases = [attention_case(s, [900, 333], [40, 7], 2, 4, 64)[0] for s in (1, 2)]
    new = [12, 12, 12]
    checks = [verify_case(s, new, 20011, 1.0, True)[0] for s in (3, 4)]
    alone = [(int4_tree_attention(**a), verify_drafts(**c)) for a, c in zip(cases, checks)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                both[i].append((int4_tree_attention(**cases[i]), verify_drafts(**checks[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for out, found in both[i]:
            assert torch.equal(out, alone[i][0]) and all(torch.equal(a, b) for a, b in zip(found, alone[i][1]))


def test_results_do_not_change_from_run_to_run():
    args, _, _ = attention_case(12, [3000, 100, 7], [33, 64, 2], 2, 4, 64)
    check = verify_case(5, [30, 30], 9001, 1.0, True)[0]
    first, found = int4_tree_attention(**args), verify_drafts(**check)
    for _ in range(5):
        assert torch.equal(first, int4_tree_attention(**args))
        assert all(torch.equal(a, b) for a, b in zip(found, verify_drafts(**check)))


def test_rows_past_the_last_node():
    """A sequence of more than 64 rows: its first 64 are nodes, the rest get zeros, and the tokens keep their places."""
    contexts, n = 40, 70
    args, _, _ = attention_case(13, [contexts], [64], 1, 2, 32, chain=True)
    q = torch.cat([args["q"], args["q"][:6]])
    table, pages = i32([[3, 0, 2, 1]]), empty_pages(4, 1, 32)
    rng = np.random.default_rng(1)
    k, v = (torch.from_numpy(rng.standard_normal((contexts + n, 1, D)).astype(np.float16)).cuda() for _ in range(2))
    int4_append(pages, table, i32([0]), k, v, i32([0, contexts + n]))
    got = int4_tree_attention(q, pages, table, i32([contexts + n]), i32([0, n]))
    want = int4_tree_attention(q[:64], pages, table, i32([contexts + 64]), i32([0, 64]))
    assert torch.equal(got[:64], want) and (got[64:] == 0).all()
    parents = [-1] + list(range(n - 1))
    seen, positions = draft_tree(i32(parents), i32([0, n]))
    assert seen[:64].tolist() == signed(ref.masks(parents[:64])).tolist() and (seen[64:] == 0).all() and (positions[64:] == 0).all()
    logits = torch.zeros(n, 33, dtype=torch.float16, device="cuda")
    logits[:, 5] = 1.0
    tokens = torch.full((n,), 5, dtype=torch.int64, device="cuda")
    path, counts, token = verify_drafts(logits, tokens, i32(parents), i32([0, n]), temperature=0)
    assert path[0].tolist() == list(range(64)) and counts.tolist() == [64] and token.tolist() == [5]
    u = torch.zeros(n, device="cuda")
    path, counts, token = verify_drafts(logits, tokens, i32(parents), i32([0, n]), u, u[:1])
    assert path[0].tolist() == list(range(64)) and counts.tolist() == [64] and token.tolist() == [0]


def test_nothing_but_rows_without_tokens():
    """Lengths that the nodes themselves pass: node i is token length - n + i, and what lies before token 0 is not there."""
    args, _, _ = attention_case(2, [0], [9], 1, 4, 32, chain=True)
    got = int4_tree_attention(**dict(args, lengths=i32([4])))  # nodes 5 .. 8 are tokens 0 .. 3
    few = int4_tree_attention(**dict(args, q=args["q"][5:].contiguous(), lengths=i32([4]), offsets=i32([0, 4])))
    assert (got[:5] == 0).all() and torch.equal(got[5:], few)
