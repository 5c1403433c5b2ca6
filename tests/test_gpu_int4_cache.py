"""Int4Cache on the GPU, and the decoder paths that use the packed and paged operators."""

import numpy as np
import pytest
import torch

import serving_reference as ref
from reskv_amd import Int4Cache, packed_attention
from reskv_amd.llama import GreedyDecoder, LlamaShape, RandomLlama

pytestmark = pytest.mark.gpu

TINY = LlamaShape(layers=2, hidden=512, heads=4, kv_heads=1, ffn=1024, vocab=1000)


def rows(g, n, heads):
    return torch.randn(n, heads, 128, generator=g).half().cuda()


def reference(q, history, scaling=128 ** -0.5):
    """(rows, bound) of one token per sequence over its rows (k, v) so far."""
    parts = []
    for b, pairs in enumerate(history):
        k, v = (np.concatenate([p[i] for p in pairs]) for i in range(2))
        (kd, ka), (vd, va) = ref.stored(k), ref.stored(v)
        parts.append(ref.sequence(q[b: b + 1].double().cpu().numpy(), kd, vd, len(k) - 1, scaling, ka, va))
    return tuple(np.concatenate(x) for x in zip(*parts))


def test_cache_through_prompt_forks_beams_and_compaction(device):
    """What every sequence attends to is what it was given, whatever became of its pages."""
    g = torch.Generator().manual_seed(1)
    layers, kv, gqa, n = 2, 2, 4, 4
    cache = Int4Cache(layers, kv, n, 300, page_tokens=32, pages=24)
    held = [[[] for _ in range(n)] for _ in range(layers)]

    def feed(counts):
        cache.reserve(counts)
        counts = [counts] * n if isinstance(counts, int) else counts
        ends = [0, *np.cumsum(counts)]
        one = counts == [1] * n
        offsets = None if one else torch.tensor(ends, dtype=torch.int32, device="cuda")
        for layer in range(layers):
            k, v = rows(g, ends[-1], kv), rows(g, ends[-1], kv)
            cache.append(layer, k, v, offsets)
            for s in range(n):
                held[layer][s] = held[layer][s] + [tuple(x[ends[s]: ends[s + 1]].cpu().numpy() for x in (k, v))]

    def check():
        for layer in range(layers):
            q = rows(g, n, kv * gqa)
            want, bound = reference(q, held[layer])
            got = cache.attend(layer, q).double().cpu().numpy()
            assert (np.abs(got - want) <= bound).all()

    def reorder(index):
        cache.reorder(index)
        for layer in range(layers):
            held[layer] = [held[layer][s] for s in index]

    feed([70, 33, 5, 64])
    check()
    feed(1)
    cache.fork(0, 2)
    for layer in range(layers):
        held[layer][2] = held[layer][0]
    feed(1)
    check()
    reorder([1, 1, 3, 0])
    feed(1)
    feed([0, 40, 1, 0])
    check()
    cache.release(3)
    for layer in range(layers):
        held[layer][3] = []
    feed([0, 0, 0, 7])
    cache.compact()
    check()
    k, v, offsets = cache.gather(1)
    assert offsets.tolist() == [0, *np.cumsum([cache.get_seq_length(s) for s in range(n)])]
    for i, got in enumerate((k, v)):
        want = np.concatenate([p[i] for s in range(n) for p in held[1][s]])
        assert np.array_equal(got.cpu().numpy(), ref.stored(want)[0].astype(np.float32).astype(np.float16))


def test_captured_steps_over_the_cache(device):
    """One captured append and attention, replayed while the cache grows (across pages, after a
    fork), equals the eager calls on a cache of its own."""
    g = torch.Generator().manual_seed(3)
    own, other = (Int4Cache(1, 2, 3, 300, page_tokens=32) for _ in range(2))
    first, at = [rows(g, 46, 2) for _ in range(2)], torch.tensor([0, 5, 14, 46], dtype=torch.int32, device="cuda")
    for c in (own, other):
        c.reserve([5, 9, 32])
        c.append(0, *first, at)
    q, k, v = rows(g, 3, 8), rows(g, 3, 2), rows(g, 3, 2)
    own.attend(0, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        own.append(0, k, v)
        out = own.attend(0, q)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            own.reserve(1)
    for step in range(150):
        for x in (q, k, v):
            x.copy_(rows(g, *x.shape[:2]))
        for c in (own, other):
            if step == 70:
                c.fork(2, 0)
            c.reserve(1)
        graph.replay()
        other.append(0, k, v)
        assert torch.equal(out, other.attend(0, q)), step
    assert own.get_seq_length(0) == 32 + 150 and own.get_seq_length(1) == 9 + 150


def test_a_prompt_in_chunks_attends_what_it_stored(device):
    """Chunked prompt: gather the cached tokens, put the chunk's own keys behind them, attend packed."""
    g = torch.Generator().manual_seed(2)
    cache = Int4Cache(1, 2, 2, 200)
    first, chunk = [50, 90], [30, 8]
    off = [0, *np.cumsum(first)]
    cache.reserve(first)
    cache.append(0, rows(g, 140, 2), rows(g, 140, 2), torch.tensor(off, dtype=torch.int32, device="cuda"))
    cache.reserve(chunk)
    at = torch.tensor([0, *np.cumsum(chunk)], dtype=torch.int32, device="cuda")
    cache.append(0, rows(g, 38, 2), rows(g, 38, 2), at)
    k, v, ends = cache.gather(0)
    q = rows(g, 38, 8)
    got = packed_attention(q, k, v, at, ends)
    want, bound = ref.packed(*(x.double().cpu().numpy() for x in (q, k, v)), at.tolist(), ends.tolist(), 128 ** -0.5)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("lengths", [[96], [1, 64, 33, 200], [5, 5]])
def test_prefill_packed_equals_each_prompt_alone(device, lengths):
    """Packed prompts give the keys, values and logits of each prompt's own pass (up to the roundings
    of attention and of GEMMs with other row counts)."""
    model = RandomLlama(TINY, "cuda", seed=5)
    ids = torch.randint(TINY.vocab, (sum(lengths),), generator=torch.Generator().manual_seed(7)).cuda()
    got = {}
    logits = model.prefill_packed(ids, lengths, lambda li, *kv: got.__setitem__(li, kv), logits=True).float()
    at = 0
    for s, n in enumerate(lengths):
        alone = {}
        want = model.prefill(ids[None, at: at + n], lambda li, *kv: alone.__setitem__(li, kv), logits=True).float()
        assert (logits[s] - want[0]).abs().max() <= 2e-2 * want.abs().max()
        for li in range(TINY.layers):
            for a, b in zip(alone[li], got[li]):
                b = b[:, :, at: at + n].float()
                assert (a.float() - b).abs().max() <= 2e-2 * a.float().abs().max()
        at += n


def test_greedy_decoder_over_the_4_bit_cache(device):
    """The harness over Int4Cache: each layer's attention is that of the keys and values the cache was
    given, for prompt tokens and decoded ones, across pages."""
    model = RandomLlama(TINY, "cuda", seed=4)
    ids = torch.randint(128, TINY.vocab, (2, 60), generator=torch.Generator().manual_seed(3)).cuda()
    dec = GreedyDecoder(model, 2, 60, 10, "int4")
    held = [[[], []] for _ in range(TINY.layers)]

    def sink(layer, raw_k, rot_k, v):
        dec.absorb(layer, raw_k, rot_k, v)
        for b in range(2):
            held[layer][b].append(tuple(x[b].transpose(0, 1).cpu().numpy() for x in (rot_k, v)))

    dec.start(model.prefill(ids, sink))
    attend, checked = dec._attend, []

    def watched(li):
        attend(li)
        for b in range(2):
            held[li][b].append(tuple(x[b: b + 1].cpu().numpy() for x in (dec.kr, dec.v)))
        want, bound = reference(dec.qr, held[li], model.scaling)
        assert (np.abs(dec.attn.double().cpu().numpy() - want) <= bound).all()
        checked.append(li)

    dec._attend = watched
    tokens = torch.stack([dec.step().clone() for _ in range(8)])
    assert checked == [0, 1] * 8 and dec.pages.get_seq_length() == 68
    assert 0 <= int(tokens.min()) and int(tokens.max()) < TINY.vocab and torch.isfinite(dec.x.float()).all()
    model.prefill(ids, dec.absorb)  # a new prompt takes the place of the old one
    assert dec.pages.get_seq_length() == 60
    ended = GreedyDecoder(model, 2, 4, 0, "int4")
    with pytest.raises(RuntimeError, match="capacity exhausted"):
        ended.step()
