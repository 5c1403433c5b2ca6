"""Int4Cache's bookkeeping on the CPU: pages, sharing, copies before a write, release and compaction, with
the page copies done by torch and the content of a page a tag per token."""

import random

import pytest
import torch

from reskv_amd import Int4Cache
from reskv_amd import int4
from reskv_amd.llama import GreedyDecoder, LlamaShape, RandomLlama


@pytest.fixture
def copies(monkeypatch):
    done = []

    def copy(pool, source, target):
        assert not set(source) & set(target) and len(set(target)) == len(target)
        done.extend(zip(source, target))
        if source:
            pool[:, target] = pool[:, source]

    monkeypatch.setattr(int4, "copy_pages", copy)
    return done


def cache(sequences=3, max_length=100, pages=None, **kw):
    return Int4Cache(1, 1, sequences, max_length, page_tokens=32, pages=pages, device="cpu", **kw)


def write(c, tags):
    """The reserved tokens' places get their tags (what the appends would do)."""
    for s in range(c.sequences):
        for i, t in enumerate(range(int(c.starts[s]), int(c.lengths[s]))):
            page = int(c.table[s, t // 32])
            assert c._users[page] == 1
            c.pool[0, page, 0, t % 32] = tags[s][i]


def read(c, s):
    return [int(c.pool[0, int(c.table[s, t // 32]), 0, t % 32]) for t in range(c.get_seq_length(s))]


def consistent(c):
    users = [0] * c.pool.shape[1]
    for s in range(c.sequences):
        n = -(-c.get_seq_length(s) // 32)
        row = c.table[s].tolist()
        assert all(p >= 0 for p in row[:n]) and row[n:] == [-1] * (len(row) - n)
        assert int(c.lengths[s]) == c.get_seq_length(s)
        for p in row[:n]:
            users[p] += 1
    assert users == c._users
    assert sorted(c._free) == [p for p, n in enumerate(users) if n == 0] and c.free_pages == len(c._free)


def test_reserve_gives_pages_in_order():
    c = cache()
    c.reserve([40, 0, 32])
    assert c.table.tolist() == [[0, 1, -1, -1], [-1] * 4, [2, -1, -1, -1]]
    assert c.starts.tolist() == [0, 0, 0] and c.lengths.tolist() == [40, 0, 32]
    c.reserve(1)
    assert c.starts.tolist() == [40, 0, 32] and c.lengths.tolist() == [41, 1, 33]
    assert c.table.tolist() == [[0, 1, -1, -1], [3, -1, -1, -1], [2, 4, -1, -1]]
    consistent(c)


def test_a_page_that_is_shared_is_copied_before_a_write(copies):
    c = cache(4)
    c.reserve([40, 3, 0, 0])
    write(c, [range(40), [90, 91, 92], [], []])
    c.fork(0, 2)
    c.fork(0, 3)
    assert c.table[2].tolist() == c.table[0].tolist() and not copies
    c.reserve([1, 0, 1, 2])
    assert len(copies) == 2  # the last of the three keeps the page
    write(c, [[200], [], [201], [202, 203]])
    assert read(c, 0) == [*range(40), 200] and read(c, 2) == [*range(40), 201]
    assert read(c, 3) == [*range(40), 202, 203] and read(c, 1) == [90, 91, 92]
    consistent(c)


def test_whole_pages_stay_shared(copies):
    c = cache(2)
    c.reserve([64, 0])
    write(c, [range(64), []])
    c.fork(0, 1)
    c.reserve([1, 1])
    assert not copies and c.free_pages == 8 - 4
    consistent(c)


def test_refusals_change_nothing(copies):
    c = cache(2, 64, pages=3)
    c.reserve([40, 20])
    for counts, match in (([0, 13], "0 are free"), (40, "pass 64 tokens"), ([1], "a count of tokens for every"),
                          ([-1, 0], "a count of tokens for every")):
        before = c.table.tolist(), c.lengths.tolist(), c.free_pages
        with pytest.raises(RuntimeError, match=match):
            c.reserve(counts)
        assert before == (c.table.tolist(), c.lengths.tolist(), c.free_pages)
    c.release(1)
    c.fork(0, 1)
    with pytest.raises(RuntimeError, match="are needed"):
        cache(2, 64, pages=1).reserve([1, 1])
    with pytest.raises(RuntimeError, match="not in 0 .. 1"):
        c.fork(0, 2)
    with pytest.raises(RuntimeError, match="not in 0 .. 1"):
        c.release(-1)
    with pytest.raises(RuntimeError, match="a row for every sequence"):
        c.reorder([0])
    consistent(c)


def test_no_append_between_a_fork_and_the_next_reservation(copies):
    """Rows that share the page of reserved tokens would write to one place."""
    c, kv = cache(2, 64), torch.zeros(2, 1, 128, dtype=torch.float16)
    c.reserve(1)
    for forked in (lambda: c.fork(0, 1), lambda: c.reorder([1, 1])):
        forked()
        with pytest.raises(RuntimeError, match="reserve tokens before"):
            c.append(0, kv, kv)
        c.reserve([0, 1])
        c.reorder([1, 0])
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            c.append(0, kv, kv)


@pytest.mark.parametrize("kw", [dict(layers=0), dict(sequences=0), dict(max_length=0), dict(page_tokens=48),
                                dict(kv_heads=0), dict(pages=0)])
def test_constructor_refusals(kw):
    with pytest.raises(RuntimeError):
        Int4Cache(**{**dict(layers=1, kv_heads=1, sequences=1, max_length=10, device="cpu"), **kw})


@pytest.mark.parametrize("seed", range(6))
def test_random_use_keeps_every_sequence(copies, seed):
    rnd = random.Random(seed)
    c = cache(5, 150, pages=21)
    want, tag = [[] for _ in range(5)], 0
    for _ in range(120):
        what = rnd.random()
        if what < 0.6:
            counts = [rnd.choice([0, 0, 1, 1, 2, rnd.randint(0, 40)]) for _ in range(5)]
            try:
                c.reserve(counts)
            except RuntimeError:
                c.release(rnd.randrange(5)) if rnd.random() < 0.5 else None
                for s in range(5):
                    want[s] = want[s][: c.get_seq_length(s)]
                continue
            tags = []
            for s, n in enumerate(counts):
                tags.append([(tag + i) % 251 for i in range(n)])
                want[s] = want[s] + tags[s]
                tag += n
            write(c, tags)
        elif what < 0.75:
            a, b = rnd.randrange(5), rnd.randrange(5)
            c.fork(a, b)
            want[b] = list(want[a])
        elif what < 0.85:
            index = [rnd.randrange(5) for _ in range(5)]
            c.reorder(torch.tensor(index))
            want = [list(want[s]) for s in index]
        elif what < 0.92:
            s = rnd.randrange(5)
            c.release(s)
            want[s] = []
        else:
            used = c.pool.shape[1] - c.free_pages
            c.compact()
            assert all(p < used for row in c._pages for p in row)
        consistent(c)
        assert [read(c, s) for s in range(5)] == want


def test_prefill_packed_on_the_cpu_is_each_prompt_alone():
    """Torch formulas (no GPU): keys and values of all prompts in one row, next tokens as alone."""
    shape = LlamaShape(layers=2, hidden=256, heads=2, kv_heads=1, ffn=64, vocab=50)
    model = RandomLlama(shape, "cpu", seed=3)
    lengths, got = [5, 1, 9], {}
    ids = torch.randint(50, (15,), generator=torch.Generator().manual_seed(1))
    tokens = model.prefill_packed(ids, lengths, lambda li, *kv: got.__setitem__(li, kv))
    at = 0
    for s, n in enumerate(lengths):
        alone = {}
        assert model.prefill(ids[None, at: at + n], lambda li, *kv: alone.__setitem__(li, kv)).item() == tokens[s].item()
        for li in range(2):
            for a, b in zip(alone[li], got[li]):
                assert torch.equal(a, b[:, :, at: at + n])
        at += n
    for bad in ([5, 10, 0], [5, 9], []):
        with pytest.raises(ValueError, match="lengths"):
            model.prefill_packed(ids, bad, lambda *a: None)


def test_decoder_mode_is_checked():
    model = RandomLlama(LlamaShape(layers=1, hidden=256, heads=2, kv_heads=1, ffn=64, vocab=50), "cpu")
    with pytest.raises(ValueError, match="'int4'"):
        GreedyDecoder(model, 1, 4, 4, "int8")
