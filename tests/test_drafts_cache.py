"""Int4Cache.keep and GreedyDecoder.step_drafts on the host: lengths, pages and refusals, with the launches left out."""

import contextlib

import pytest
import torch

from reskv_amd import int4, llama
from reskv_amd.int4 import Int4Cache
from reskv_amd.llama import GreedyDecoder, LlamaShape, RandomLlama

i32 = dict(dtype=torch.int32)


@pytest.fixture
def moved(monkeypatch):
    calls = []
    monkeypatch.setattr(int4, "int4_keep", lambda pages, table, starts, path, counts: calls.append((starts.tolist(), counts.tolist())))
    monkeypatch.setattr(int4, "copy_pages", lambda *a: None)
    return calls


def path(rows):
    return torch.zeros(rows, 64, **i32)


def test_keep_cuts_rows_and_frees_their_pages(moved):
    cache = Int4Cache(2, 1, 3, 400, page_tokens=32, pages=20, device="cpu")
    cache.reserve([30, 64, 0])
    free = cache.free_pages
    cache.reserve([40, 2, 33])
    assert cache.free_pages == free - 2 - 1 - 2
    assert cache.keep(path(3), torch.tensor([3, 2, 0], **i32)) == [3, 2, 0]
    assert moved == [([30, 64, 0], [3, 2, 0])]
    assert [cache.get_seq_length(s) for s in range(3)] == [33, 66, 0]
    assert cache.lengths.tolist() == [33, 66, 0] and cache.starts.tolist() == [30, 64, 0]
    assert cache.free_pages == 20 - 2 - 3 - 0 and (cache.table[0, 2:] == -1).all() and (cache.table[2] == -1).all()
    assert len(set(cache.table[cache.table >= 0].tolist())) == 5
    cache.reserve(1)  # goes on behind what was kept
    assert cache.starts.tolist() == [33, 66, 0] and cache.lengths.tolist() == [34, 67, 1]


def test_keep_of_everything_and_nothing(moved):
    cache = Int4Cache(1, 1, 2, 200, page_tokens=32, device="cpu")
    cache.reserve([31, 5])
    cache.reserve(2)
    cache.keep(path(2), torch.tensor([2, 2], **i32))
    assert cache.lengths.tolist() == [33, 7]
    cache.reserve(3)
    cache.keep(path(2), torch.tensor([0, 0], **i32))
    assert cache.lengths.tolist() == [33, 7] and cache.starts.tolist() == [33, 7]


@pytest.mark.parametrize("counts", [[4, 0], [-1, 0], [0, 2]])
def test_more_than_was_reserved_is_refused(moved, counts):
    cache = Int4Cache(1, 1, 2, 200, device="cpu")
    cache.reserve([10, 10])
    cache.reserve([3, 1])
    with pytest.raises(RuntimeError, match="between none and all of the tokens reserved last"):
        cache.keep(path(2), torch.tensor(counts, **i32))
    assert not moved and cache.lengths.tolist() == [13, 11]


def test_a_path_shorter_than_what_is_kept_is_refused(moved):
    cache = Int4Cache(1, 1, 2, 200, device="cpu")
    cache.reserve(5)
    for bad in (torch.zeros(2, 3, **i32), torch.zeros(128, **i32)):
        with pytest.raises(RuntimeError, match="path must list every token that is kept"):
            cache.keep(bad, torch.tensor([4, 1], **i32))
    assert not moved and cache.lengths.tolist() == [5, 5]


def test_forked_rows_are_refused(moved):
    cache = Int4Cache(1, 1, 2, 200, device="cpu")
    cache.reserve([10, 10])
    cache.fork(0, 1)
    with pytest.raises(RuntimeError, match="cannot be kept apart"):
        cache.keep(path(2), torch.tensor([1, 1], **i32))
    with pytest.raises(RuntimeError, match="reserve tokens before the next append"):
        cache.append_rope(0, None, torch.zeros(2, 1, 128), torch.zeros(2, 1, 128), None, None)
    assert not moved


def test_pages_shared_with_a_fork_stay_with_it(moved):
    """Drafts of a forked row lie in its own pages: keeping none of them gives back those alone."""
    cache = Int4Cache(1, 1, 2, 200, page_tokens=32, pages=8, device="cpu")
    cache.reserve([40, 0])
    cache.fork(0, 1)
    cache.reserve([30, 30])
    cache.keep(path(2), torch.tensor([0, 5], **i32))
    assert cache.lengths.tolist() == [40, 45]
    assert cache.table[0, 0] == cache.table[1, 0] and cache.table[0, 1] != cache.table[1, 1]
    cache.release(0)
    assert cache.free_pages == 8 - 2


SHAPE = LlamaShape(layers=1, hidden=256, heads=2, kv_heads=1, ffn=64, vocab=50)


@pytest.fixture
def decoder():
    return GreedyDecoder(RandomLlama(SHAPE, "cpu", seed=3), 2, 6, 40, "int4")


@pytest.mark.parametrize("kw,match", [
    (dict(drafts=torch.zeros(2, 3)), "an int64 matrix with a row for each of the 2 sequences"),
    (dict(drafts=torch.zeros(3, 3, dtype=torch.int64)), "a row for each of the 2 sequences"),
    (dict(drafts=torch.zeros(2, 64, dtype=torch.int64)), "up to 64 nodes"),
    (dict(parents=[0, 1]), "a node before it for every draft"),
    (dict(parents=[0, 2, 1]), "a node before it for every draft"),
    (dict(parents=[-1, 0, 0]), "a node before it for every draft"),
    (dict(temperature=1.0), "sampling needs random numbers"),
    (dict(temperature=1.0, accept=torch.zeros(2, 3), sample=torch.zeros(2)), r"accept must be fp32 \[2, 4\]"),
    (dict(temperature=1.0, accept=torch.zeros(2, 4, dtype=torch.float64), sample=torch.zeros(2)), r"accept must be fp32 \[2, 4\]"),
    (dict(temperature=-1.0, accept=torch.zeros(2, 4), sample=torch.zeros(2)), "temperature must be 0, or"),
    (dict(temperature=float("nan"), accept=torch.zeros(2, 4), sample=torch.zeros(2)), "temperature must be 0, or"),
    (dict(temperature=1.0, accept=torch.zeros(2, 4), sample=torch.zeros(4)), r"sample must be fp32 \[2\]"),
    (dict(temperature=1.0, accept=torch.zeros(2, 4), sample=torch.zeros(2), draft=torch.zeros(2, 4, 49)), r"draft must be fp32 \[2, 4, 50\]"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_step_drafts_checks(decoder, kw, match):
    with pytest.raises(ValueError, match=match):
        decoder.step_drafts(**{"drafts": torch.zeros(2, 3, dtype=torch.int64), **kw})
    assert decoder.pages.lengths.tolist() == [0, 0]


def test_drafts_need_the_paged_cache():
    dec = GreedyDecoder(RandomLlama(SHAPE, "cpu", seed=3), 2, 6, 4, "dense")
    with pytest.raises(ValueError, match="drafts need the 4-bit cache"):
        dec.step_drafts(torch.zeros(2, 3, dtype=torch.int64))


@pytest.mark.parametrize("fails", ["draft_tree", "fused_rmsnorm", "verify_drafts"])
def test_a_failed_step_leaves_nothing_reserved(monkeypatch, fails):
    """Whatever raises between the reservation and the accepted tokens, rows and pages are what they were."""
    def stop(*args, **kw):
        raise MemoryError("no room")

    nodes = 4 * 2  # what stands in for the GPU's operators returns tensors of their shapes
    monkeypatch.setattr(llama, "_on_gpu", lambda *t: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(llama, "draft_tree", lambda *a: (torch.zeros(nodes, dtype=torch.int64), torch.zeros(nodes, dtype=torch.int32)))
    monkeypatch.setattr(llama, "fused_rmsnorm", lambda x, *a: x)
    monkeypatch.setattr(llama, "fused_silu_mul", lambda x, out: out.zero_())
    monkeypatch.setattr(Int4Cache, "append_rope", lambda self, li, q, *a, **kw: q)
    monkeypatch.setattr(Int4Cache, "attend_tree", lambda self, li, q, *a, **kw: q.contiguous())
    monkeypatch.setattr(llama, fails, stop)
    decoder = GreedyDecoder(RandomLlama(SHAPE, "cpu", seed=3), 2, 6, 140, "int4")
    pages = decoder.pages
    pages.reserve([5, 62])  # the second row's nodes need another page
    free, state = pages.free_pages, (pages.lengths.tolist(), pages.table.tolist(), decoder.tok.tolist(), decoder.pos)
    for _ in range(2):
        with pytest.raises(MemoryError, match="no room"):
            decoder.step_drafts(torch.zeros(2, 3, dtype=torch.int64))
        assert (pages.lengths.tolist(), pages.table.tolist(), decoder.tok.tolist(), decoder.pos) == state
        assert pages.free_pages == free and pages.starts.tolist() == [5, 62] and [pages.get_seq_length(s) for s in range(2)] == [5, 62]
