"""GreedyDecoder over the 4-bit cache on the CPU: which tokens and positions it takes from a prompt, with the append
replaced by a record."""

import pytest
import torch

from reskv_amd import int4
from reskv_amd.llama import GreedyDecoder, LlamaShape, RandomLlama

SHAPE = LlamaShape(layers=2, hidden=256, heads=2, kv_heads=1, ffn=64, vocab=50)


@pytest.fixture
def appended(monkeypatch):
    calls = []
    monkeypatch.setattr(int4, "int4_append",
                        lambda pages, table, starts, k, v, offsets=None: calls.append((starts.tolist(), k, v, offsets.tolist())))
    return calls


def prompt(model, batch, tokens, sink):
    return model.prefill(torch.randint(50, (batch, tokens), generator=torch.Generator().manual_seed(tokens)), sink)


@pytest.mark.parametrize("first,second", [(6, 6), (6, 3), (4, 9)])
def test_decoding_goes_on_behind_the_last_prompt(appended, first, second):
    model = RandomLlama(SHAPE, "cpu", seed=3)
    dec = GreedyDecoder(model, 2, 6, 4, "int4")
    prompt(model, 2, first, dec.absorb)
    assert dec.pos == first and dec.pages.get_seq_length(1) == first
    dec.pages.reserve(1)
    dec.pos += 1
    prompt(model, 2, second, dec.absorb)
    assert dec.pos == second and dec.pages.get_seq_length(0) == dec.pages.get_seq_length(1) == second
    assert [c[0] for c in appended] == [[0, 0]] * 4 and appended[-1][3] == [0, second, 2 * second]


def test_a_prompt_past_the_capacity_changes_nothing(appended):
    model = RandomLlama(SHAPE, "cpu", seed=3)
    dec = GreedyDecoder(model, 2, 6, 4, "int4")
    prompt(model, 2, 5, dec.absorb)
    with pytest.raises(RuntimeError, match="a prompt of 11 tokens passes the decoder's capacity of 10"):
        prompt(model, 2, 11, dec.absorb)
    assert dec.pos == 5 and dec.pages.get_seq_length(0) == dec.pages.get_seq_length(1) == 5 and len(appended) == 2
    prompt(model, 2, 10, dec.absorb)
    with pytest.raises(RuntimeError, match="capacity exhausted"):
        dec.step()


def test_packed_prompts_are_refused(appended):
    """``prefill_packed`` hands all prompts on in one row: not one prompt per row of the decoder."""
    model = RandomLlama(SHAPE, "cpu", seed=3)
    dec = GreedyDecoder(model, 2, 6, 4, "int4")
    prompt(model, 2, 5, dec.absorb)
    ids = torch.arange(9)
    with pytest.raises(RuntimeError, match="takes 2 prompts of one length, not 1"):
        model.prefill_packed(ids, [6, 3], dec.absorb)
    with pytest.raises(RuntimeError, match="takes 2 prompts of one length, not 3"):
        prompt(model, 3, 4, dec.absorb)
    assert dec.pos == 5 and dec.pages.get_seq_length(0) == dec.pages.get_seq_length(1) == 5 and len(appended) == 2
