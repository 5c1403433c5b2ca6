"""GreedyDecoder over the 4-bit cache: a decoder that takes another prompt decodes as one that is new."""

import pytest
import torch

from reskv_amd.llama import GreedyDecoder, LlamaShape, RandomLlama

pytestmark = pytest.mark.gpu

TINY = LlamaShape(layers=2, hidden=512, heads=4, kv_heads=1, ffn=1024, vocab=1000)


@pytest.mark.parametrize("second", [60, 31, 64])
def test_a_second_prompt_decodes_as_in_a_new_decoder(device, second):
    """Same tokens in, so the same rotated keys, pages and attention (up to the roundings of GEMMs), step by step."""
    model = RandomLlama(TINY, "cuda", seed=4)
    g = torch.Generator().manual_seed(3)
    ids = [torch.randint(128, TINY.vocab, (2, n), generator=g).cuda() for n in (60, second)]
    used, new = GreedyDecoder(model, 2, 60, 10, "int4"), GreedyDecoder(model, 2, second, 70 - second, "int4")
    used.start(model.prefill(ids[0], used.absorb))
    for _ in range(4):
        used.step()
    seen = []
    for dec in (used, new):
        dec.start(model.prefill(ids[1], dec.absorb))
        assert dec.pos == second
        seen.append([])
        for t in range(6):
            dec.start(torch.tensor([t + 1, 2 * t + 200], device="cuda"))
            dec.step()
            assert dec.pages.get_seq_length(1) == dec.pos == second + t + 1
            seen[-1].append([x.float().clone() for x in (dec.kr, dec.qr, dec.attn, dec.x)])
    for a, b in zip(*seen):
        for x, y in zip(a, b):
            assert (x - y).abs().max() <= 1e-2 * y.abs().max()
