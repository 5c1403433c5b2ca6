"""Workspace of packed attention with split keys: no more than the rows that there can be, and no byte behind it."""

import ctypes

import numpy as np
import pytest
import torch

import serving_reference as ref
from reskv_amd import _lib


def size(sequences, queries, heads, kv_heads, most):
    return _lib.lib().reskv_packed_workspace_bytes(sequences, queries, heads, kv_heads, most)


@pytest.mark.parametrize("sequences,queries,heads,kv_heads", [(1, 1, 4, 1), (1, 1, 32, 8), (3, 5, 16, 2), (2, 64, 4, 1),
                                                              (2, 65, 4, 1), (1, 2000, 8, 8)])
def test_workspace_follows_the_rows(sequences, queries, heads, kv_heads):
    """128 weighted values, a reference and a sum of 4 bytes for every row of at most 256 that a workgroup can
    have, 256 workgroups, and the length of a part."""
    rows = min(256, queries * heads // kv_heads)
    assert size(sequences, queries, heads, kv_heads, 20000) in (0, 256 // kv_heads * kv_heads * rows * 130 * 4 + 16)
    assert size(1, 1, 32, 8, 20000) <= 600 * 1024


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk,kv,gqa", [([1], [3000], 1, 1), ([1, 1], [2000, 1500], 2, 4), ([9, 7], [1500, 4000], 3, 16),
                                          ([63], [2100], 1, 4), ([40, 25], [2100, 3000], 2, 4), ([5, 0, 300], [3000, 9, 4000], 1, 3)])
def test_no_byte_behind_the_workspace_is_written(device, nq, nk, kv, gqa):
    r = np.random.default_rng(sum(nq))
    q, k, v = (r.standard_normal((sum(n), h, 128)).astype(np.float16) for n, h in ((nq, kv * gqa), (nk, kv), (nk, kv)))
    at, kat = ([0, *np.cumsum(n)] for n in (nq, nk))
    nbytes = size(len(nq), sum(nq), kv * gqa, kv, max(nk))
    assert nbytes > 0
    work = torch.full((nbytes + 4096,), 77, dtype=torch.uint8, device="cuda")
    tensors = [torch.from_numpy(x).cuda() for x in (q, k, v)]
    out = torch.zeros_like(tensors[0])
    offsets = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (at, kat)]
    strides = (ctypes.c_int64 * 6)(*(n for t in tensors for n in t.stride()[:2]))
    assert _lib.lib().reskv_packed_attention(*(t.data_ptr() for t in (*tensors, out, *offsets)), len(nq), sum(nq), sum(nk),
                                             kv * gqa, kv, strides, 128 ** -0.5, max(nk), 1, work.data_ptr(), nbytes,
                                             torch.cuda.current_stream().cuda_stream) == 0
    assert (work[nbytes:] == 77).all()
    want, bound = ref.packed(*(x.astype(np.float64) for x in (q, k, v)), at, kat, 128 ** -0.5)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
