"""Prompts that continue on an ``Int4Cache``: the chunk's own fp16 rows behind what the cache held before."""

import numpy as np
import pytest
import torch

import serving_reference as ref
from reskv_amd import Int4Cache, packed_attention

pytestmark = pytest.mark.gpu


def rows(g, n, heads):
    return torch.randn(n, heads, 128, generator=g).half().cuda()


def i32(lengths):
    return torch.tensor([0, *np.cumsum(lengths)], dtype=torch.int32, device="cuda")


def behind(held, ends, new, at):
    """Each sequence's rows of ``new`` behind its rows of ``held``."""
    return torch.cat([torch.cat((held[ends[s]: ends[s + 1]], new[at[s]: at[s + 1]])) for s in range(len(at) - 1)])


@pytest.mark.parametrize("first,chunk", [([50, 90, 0], [30, 8, 5]), ([64, 1, 33], [1, 64, 0])])
def test_a_chunk_attends_its_own_rows_behind_the_cached_ones(device, first, chunk):
    """In the order of a step: reserve, then per layer gather, attend and append.  The pages that the chunk gets
    held NaN rows before."""
    g = torch.Generator().manual_seed(sum(first))
    n, kv = len(first), 2
    cache = Int4Cache(1, kv, n, 130, page_tokens=32)
    cache.pool.fill_(255)  # places of no token read as NaN
    cache.reserve(first)
    held = rows(g, sum(first), kv), rows(g, sum(first), kv)
    cache.append(0, *held, i32(first))
    cache.reserve(chunk)
    new, q = (rows(g, sum(chunk), kv), rows(g, sum(chunk), kv)), rows(g, sum(chunk), 4 * kv)
    k, v, ends = cache.gather(0, reserved=False)
    assert ends.tolist() == i32(first).tolist()
    at = i32(chunk).tolist()
    k, v = (behind(x, ends.tolist(), y, at) for x, y in zip((k, v), new))
    both = i32([a + b for a, b in zip(first, chunk)])
    got = packed_attention(q, k, v, i32(chunk), both).double().cpu().numpy()
    cache.append(0, *new, i32(chunk))
    stored = [ref.stored(x.cpu().numpy())[0].astype(np.float32).astype(np.float16) for x in held]
    want = [behind(torch.from_numpy(x), ends.tolist(), y.cpu(), at).double().numpy() for x, y in zip(stored, new)]
    want, bound = ref.packed(q.double().cpu().numpy(), *want, at, both.tolist(), 128 ** -0.5)
    assert (np.abs(got - want) <= bound).all()
    assert torch.isfinite(cache.gather(0)[0].float()).all()
