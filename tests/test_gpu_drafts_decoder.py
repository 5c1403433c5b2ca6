"""GreedyDecoder.step_drafts: drafted decoding gives what decoding token by token gives."""

import pytest
import torch

from reskv_amd import llama
from reskv_amd.llama import GreedyDecoder, LlamaShape, RandomLlama

pytestmark = pytest.mark.gpu

TINY = LlamaShape(layers=2, hidden=512, heads=4, kv_heads=1, ffn=1024, vocab=1000)


@pytest.fixture(scope="module")
def setting():
    # wide embeddings and head: the argmax is far ahead of the next logit, so that roundings of other launch shapes do not turn it
    model = RandomLlama(TINY, "cuda", seed=4)
    model.lm_head *= 20
    ids = torch.randint(TINY.vocab, (3, 41), generator=torch.Generator().manual_seed(3)).cuda()
    return model, ids


def start(setting, new=60):
    model, ids = setting
    dec = GreedyDecoder(model, 3, 41, new, "int4")
    dec.start(model.prefill(ids, dec.absorb))
    return dec


@pytest.fixture(scope="module")
def plain(setting):
    dec = start(setting)
    return torch.stack([dec.tok.clone()] + [dec.step().clone() for _ in range(24)], dim=1)


def test_right_drafts_are_all_accepted(setting, plain):
    dec = start(setting)
    assert torch.equal(dec.tok, plain[:, 0])
    tokens, counts = dec.step_drafts(plain[:, 1:6])
    assert counts == [6, 6, 6] and torch.equal(tokens, plain[:, 1:7]) and dec.pos == 47
    assert torch.equal(dec.step(), plain[:, 7])  # rows of one length again: the captured step
    tokens, counts = dec.step_drafts(plain[:, 8:8])
    assert counts == [1, 1, 1] and torch.equal(tokens, plain[:, 8:9])


def test_wrong_drafts_change_nothing(setting, plain):
    """Rows that keep different numbers of drafts, chains and trees in turn, plain steps between them."""
    dec = start(setting)
    have = [1, 1, 1]
    gen = torch.Generator("cuda").manual_seed(5)
    trees = [None, [0, 0, 1, 1, 2, 3], [0, 1, 2, 0, 4, 5]]
    while max(have) < 17:
        parents = trees[sum(have) % 3]
        drafts = torch.randint(TINY.vocab, (3, 6), device="cuda", generator=gen)
        for s in range(3):  # row s: a branch of s + 1 right tokens, then wrong ones, among nodes of the tree
            node, above = 0, parents or list(range(6))
            for d in range(s + 1):
                child = max(i + 1 for i, p in enumerate(above) if p == node) if node in above else 0
                if child == 0:
                    break
                drafts[s, child - 1] = plain[s, have[s] + d]
                node = child
        tokens, counts = dec.step_drafts(drafts, parents)
        for s, c in enumerate(counts):
            assert tokens[s, :c].tolist() == plain[s, have[s]: have[s] + c].tolist()
            assert (tokens[s, c:] == -1).all()
            have[s] += c
        assert dec.pages.lengths.tolist() == [41 + h - 1 for h in have]
        if len(set(have)) > 1:
            events = []
            step = dec.step(events)
            assert len(events) == TINY.layers
            for s in range(3):
                assert step[s] == plain[s, have[s]]
                have[s] += 1
    assert have[2] > have[0]


def test_drafts_outside_the_vocabulary_are_passed_over(setting, plain):
    dec = start(setting)
    drafts = torch.full((3, 2), 1 << 40, device="cuda")
    drafts[1] = -1
    tokens, counts = dec.step_drafts(drafts)
    assert counts == [1, 1, 1] and torch.equal(tokens[:, :1], plain[:, 1:2]) and (tokens[:, 1:] == -1).all()


def test_sampling_with_one_temperature_is_reproducible(setting):
    """The same random numbers give the same tokens; drafts of the target's likeliest tokens with accept = 0 are taken."""
    runs = []
    for _ in range(2):
        dec = start(setting)
        gen = torch.Generator("cuda").manual_seed(1)
        out = []
        for _ in range(4):
            drafts = torch.randint(TINY.vocab, (3, 3), device="cuda", generator=gen)
            tokens, counts = dec.step_drafts(drafts, temperature=5.0, accept=torch.rand(3, 4, device="cuda", generator=gen),
                                             sample=torch.rand(3, device="cuda", generator=gen))
            assert all(1 <= c <= 4 for c in counts) and (tokens.gather(1, torch.tensor(counts, device="cuda")[:, None] - 1) >= 0).all()
            out.append(tokens)
        runs.append(torch.cat(out, 1))
    assert torch.equal(*runs)
    dec = start(setting)
    zero = torch.zeros(3, 4, device="cuda")
    _, counts = dec.step_drafts(torch.randint(TINY.vocab, (3, 3), device="cuda"), temperature=5.0, accept=zero, sample=zero[:, 0].contiguous())
    assert counts == [4, 4, 4]


def test_capacity(setting, plain):
    dec = start(setting, new=8)
    dec.step_drafts(plain[:, 1:4])
    with pytest.raises(RuntimeError, match="capacity exhausted"):
        dec.step_drafts(plain[:, 5:10])
    assert dec.pages.lengths.tolist() == [45, 45, 45]
    tokens, counts = dec.step_drafts(plain[:, 5:8])
    assert counts == [4, 4, 4] and dec.pos == 49
    with pytest.raises(RuntimeError, match="capacity exhausted"):
        dec.step()


def test_a_failed_step_changes_nothing(setting, plain, monkeypatch):
    """Drafts that a failed step has appended are not there for the next one, captured (rows of one length) or not."""
    dec = start(setting)
    for uneven in (False, True):
        if uneven:
            drafts = plain[:, 2:5].clone()
            drafts[1] = -1
            assert dec.step_drafts(drafts)[1] == [4, 1, 4]
        have = [n - 41 + 1 for n in dec.pages.lengths.tolist()]
        with monkeypatch.context() as m:
            m.setattr(llama, "verify_drafts", lambda *a, **kw: 1 / 0)
            with pytest.raises(ZeroDivisionError):
                dec.step_drafts(torch.zeros(3, 5, dtype=torch.int64, device="cuda"))
        assert [n - 41 + 1 for n in dec.pages.lengths.tolist()] == have and dec.pages.starts.tolist() == dec.pages.lengths.tolist()
        step = dec.step()
        assert [int(step[s]) for s in range(3)] == [int(plain[s, h]) for s, h in enumerate(have)]


def test_random_numbers_and_distributions_of_any_strides(setting):
    """accept, sample and draft as views: the results are those of contiguous tensors."""
    gen = torch.Generator("cuda").manual_seed(2)
    accept, sample = torch.rand(3, 4, 2, device="cuda", generator=gen), torch.rand(3, 2, device="cuda", generator=gen)
    q = torch.softmax(torch.randn(3, 4, TINY.vocab, 2, device="cuda", generator=gen), dim=2)
    one = torch.softmax(torch.randn(TINY.vocab, device="cuda", generator=gen), dim=0)
    wide = torch.zeros(3, 4, TINY.vocab + 5, device="cuda")
    wide[..., :TINY.vocab] = q[..., 0]
    drafts = torch.randint(TINY.vocab, (3, 3), device="cuda", generator=gen)
    for draft in (q[..., 0], one.expand(3, 4, TINY.vocab), wide[..., :TINY.vocab], q[..., 1].transpose(0, 1).contiguous().transpose(0, 1), None):
        runs = []
        for same in (lambda t: t, lambda t: t.contiguous()):
            dec = start(setting)
            for _ in range(2):
                runs.append(dec.step_drafts(drafts, temperature=5.0, accept=same(accept[..., 0]), sample=same(sample[:, 0]),
                                            draft=None if draft is None else same(draft)))
        assert all(torch.equal(a[0], b[0]) and a[1] == b[1] for a, b in zip(runs[:2], runs[2:]))
