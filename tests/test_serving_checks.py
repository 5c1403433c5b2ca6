"""Argument checks of packed attention and the paged 4-bit cache, on the CPU: every mismatch is refused
before a pointer reaches a kernel (shape, dtype and layout first, then the device)."""

import ctypes

import pytest
import torch

from reskv_amd import _lib, packed_attention
from reskv_amd.int4 import copy_pages, empty_pages, int4_append, int4_attention, int4_gather

f16 = dict(dtype=torch.float16)
i32 = dict(dtype=torch.int32)


def _packed(**changes):
    kw = dict(q=torch.zeros(6, 4, 128, **f16), k=torch.zeros(6, 2, 128, **f16), v=torch.zeros(6, 2, 128, **f16),
              q_offsets=torch.tensor([0, 2, 6], **i32))
    kw.update(changes)
    return packed_attention(**kw)


@pytest.mark.parametrize("changes,match", [
    (dict(q=torch.zeros(6, 4, 128)), r"q must be fp16 \[rows, heads, 128\]"),
    (dict(q=torch.zeros(6, 4, 64, **f16)), r"q must be fp16"),
    (dict(q=torch.zeros(1, 6, 4, 128, **f16)), r"q must be fp16"),
    (dict(k=torch.zeros(6, 2, 128, dtype=torch.bfloat16)), r"k must be fp16"),
    (dict(v=torch.zeros(6, 1, 128, **f16)), "v has 1 heads, expected 2"),
    (dict(v=torch.zeros(5, 2, 128, **f16)), "same number of rows"),
    (dict(q=torch.zeros(6, 3, 128, **f16)), "multiple of the KV heads"),
    (dict(k=torch.zeros(6, 0, 128, **f16), v=torch.zeros(6, 0, 128, **f16)), "multiple of the KV heads"),
    (dict(q_offsets=torch.tensor([0, 2, 6])), "q_offsets must be a contiguous int32 vector"),
    (dict(q_offsets=torch.tensor([[0, 2, 6]], **i32)), "q_offsets must be a contiguous int32 vector"),
    (dict(q_offsets=torch.tensor([0, 9, 2, 9, 6], **i32)[::2]), "q_offsets must be a contiguous int32 vector"),
    (dict(q_offsets=torch.tensor([0], **i32)), "at least one sequence"),
    (dict(k_offsets=torch.tensor([0, 6], **i32)), "k_offsets has 2 entries, expected 3"),
    (dict(k_offsets=torch.tensor([0, 1, 6])), "k_offsets must be a contiguous int32 vector"),
    (dict(scaling=0.0), "scaling must be positive"),
    (dict(scaling=-1.0), "scaling must be positive"),
    (dict(scaling=float("nan")), "scaling must be positive"),
    (dict(scaling=float("inf")), "scaling must be positive"),
    (dict(max_keys=-1), "max_keys must not be negative"),
    (dict(out=torch.zeros(5, 4, 128, **f16)), "a row for every query"),
    (dict(out=torch.zeros(6, 2, 128, **f16)), "out has 2 heads, expected 4"),
    (dict(out=torch.zeros(6, 4, 128)), "out must be fp16"),
    (dict(out=torch.zeros(4, 6, 128, **f16).transpose(0, 1)), "out must be contiguous"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_packed_attention_checks(changes, match):
    with pytest.raises(RuntimeError, match=match):
        _packed(**changes)


def _pages(**changes):
    kw = dict(pages=empty_pages(3, 2, 64, device="cpu"), table=torch.tensor([[0, 1], [2, -1]], **i32),
              starts=torch.tensor([0, 5], **i32), k=torch.zeros(2, 2, 128, **f16), v=torch.zeros(2, 2, 128, **f16))
    kw.update(changes)
    return kw


POOL = [
    (dict(pages=torch.zeros(3, 2, 64 * 160)), "pages must be a contiguous uint8 tensor"),
    (dict(pages=torch.zeros(2, 3, 2, 64 * 160, dtype=torch.uint8)), "pages must be a contiguous uint8 tensor"),
    (dict(pages=torch.zeros(2, 3, 64 * 160, dtype=torch.uint8).transpose(0, 1)), "pages must be a contiguous uint8"),
    (dict(pages=torch.zeros(3, 2, 60 * 160, dtype=torch.uint8)), "positive multiple of 32 tokens"),
    (dict(pages=torch.zeros(3, 2, 0, dtype=torch.uint8)), "positive multiple of 32 tokens"),
    (dict(pages=torch.zeros(0, 2, 64 * 160, dtype=torch.uint8)), "positive multiple of 32 tokens"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int64)), "table must be a contiguous int32 matrix"),
    (dict(table=torch.zeros(2, 0, **i32)), "table must be a contiguous int32 matrix"),
    (dict(table=torch.zeros(2, 2, **i32).t()), "table must be a contiguous int32 matrix"),
    (dict(table=torch.zeros(4, **i32)), "table must be a contiguous int32 matrix"),
]


@pytest.mark.parametrize("changes,match", POOL + [
    (dict(starts=torch.tensor([0, 5])), "starts must be a contiguous int32 vector"),
    (dict(starts=torch.tensor([0, 5, 7], **i32)), "starts has 3 entries, expected 2"),
    (dict(k=torch.zeros(2, 3, 128, **f16)), "k has 3 heads, expected 2"),
    (dict(v=torch.zeros(2, 2, 128)), "v must be fp16"),
    (dict(v=torch.zeros(1, 2, 128, **f16)), "same number of rows"),
    (dict(k=torch.zeros(3, 2, 128, **f16), v=torch.zeros(3, 2, 128, **f16)), "one row for every sequence"),
    (dict(offsets=torch.tensor([0, 2], **i32)), "offsets has 2 entries, expected 3"),
    (dict(offsets=torch.tensor([0, 1, 2])), "offsets must be a contiguous int32 vector"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_append_checks(changes, match):
    with pytest.raises(RuntimeError, match=match):
        int4_append(**_pages(**changes))


@pytest.mark.parametrize("changes,match", POOL + [
    (dict(starts=torch.tensor([0], **i32)), "starts has 1 entries, expected 2"),
    (dict(offsets=torch.tensor([0, 1], **i32)), "offsets has 2 entries, expected 3"),
    (dict(rows=-1), "rows must not be negative"),
    (dict(out=(torch.zeros(2, 2, 128, **f16), torch.zeros(3, 2, 128, **f16))), "out v must be contiguous and have 2 rows"),
    (dict(out=(torch.zeros(2, 1, 128, **f16), torch.zeros(2, 2, 128, **f16))), "out k has 1 heads, expected 2"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_gather_checks(changes, match):
    kw = _pages(offsets=torch.tensor([0, 1, 2], **i32), rows=2)
    del kw["k"], kw["v"]
    kw.update(changes)
    with pytest.raises(RuntimeError, match=match):
        int4_gather(**kw)


@pytest.mark.parametrize("changes,match", POOL + [
    (dict(lengths=torch.tensor([1, 2])), "lengths must be a contiguous int32 vector"),
    (dict(lengths=torch.tensor([1], **i32)), "lengths has 1 entries, expected 2"),
    (dict(q=torch.zeros(2, 4, 128)), "q must be fp16"),
    (dict(q=torch.zeros(3, 4, 128, **f16)), "one row for every sequence"),
    (dict(q=torch.zeros(2, 5, 128, **f16)), "multiple of the KV heads"),
    (dict(q=torch.zeros(2, 0, 128, **f16)), "multiple of the KV heads"),
    (dict(scaling=float("inf")), "scaling must be finite"),
    (dict(scaling=float("nan")), "scaling must be finite"),
    (dict(max_length=-1), "max_length must not be negative"),
    (dict(out=torch.zeros(2, 2, 128, **f16)), "out has 2 heads, expected 4"),
    (dict(out=torch.zeros(4, 2, 128, **f16).transpose(0, 1)), "out must be contiguous and shaped like q"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_attention_checks(changes, match):
    kw = _pages(q=torch.zeros(2, 4, 128, **f16), lengths=torch.tensor([3, 64], **i32))
    del kw["k"], kw["v"], kw["starts"]
    kw.update(changes)
    with pytest.raises(RuntimeError, match=match):
        int4_attention(**kw)


@pytest.mark.parametrize("source,target,match", [
    ([0], [1, 2], "every source page needs a target page"),
    ([0, 4], [1, 2], r"page numbers must be in 0 \.\. 3"),
    ([0], [-1], r"page numbers must be in 0 \.\. 3"),
    ([0, 1], [2, 2], "neither a source nor named twice"),
    ([0, 1], [1, 2], "neither a source nor named twice"),
    ([0], [0], "neither a source nor named twice"),
    ([0], [1], "every tensor must be a CUDA tensor"),
])
def test_copy_checks(source, target, match):
    with pytest.raises(RuntimeError, match=match):
        copy_pages(empty_pages(4, 1, 32, layers=2, device="cpu"), source, target)
    with pytest.raises(RuntimeError, match=match):
        copy_pages(empty_pages(4, 1, 32, device="cpu"), source, target)


def test_copy_checks_of_the_pool():
    for bad in (torch.zeros(4, 160, dtype=torch.uint8), torch.zeros(4, 1, 5120), torch.zeros(4, 1, 5120, 2, dtype=torch.uint8)[..., 0],
                torch.zeros(4, 1, 0, dtype=torch.uint8), torch.zeros(4, 3, 10, dtype=torch.uint8)):
        with pytest.raises(RuntimeError, match="uint8 tensor|multiple of 16 bytes"):
            copy_pages(bad, [0], [1])


@pytest.mark.parametrize("args", [(0, 1, 64), (1, 0, 64), (1, 1, 0), (1, 1, 33), (1, 1, -32)])
def test_empty_pages_checks(args):
    with pytest.raises(RuntimeError, match="page"):
        empty_pages(*args, device="cpu")


def _err(status):
    assert status != 0
    return _lib.lib().reskv_last_error().decode()


def test_entry_points_refuse_bad_arguments_without_a_gpu():
    lib = _lib.lib()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(24)  # never dereferenced: validation fails first
    six = (ctypes.c_int64 * 6)(512, 128, 256, 128, 256, 128)

    def packed(q=p, out=p, S=1, Nq=4, Nk=4, Hq=4, Hk=2, strides=six, scaling=1.0, most=4, work=None, nbytes=0):
        return lib.reskv_packed_attention(q, p, p, out, p, p, S, Nq, Nk, Hq, Hk, strides, scaling, most, 0, work, nbytes, None)

    assert "null" in _err(packed(q=None))
    for scaling in (0.0, 1e300, float("nan")):  # 1e300 is infinite in 32 bits
        assert "scaling must be positive" in _err(packed(scaling=scaling))
    assert "bad sizes" in _err(packed(S=0)) and "bad sizes" in _err(packed(Hq=5)) and "bad sizes" in _err(packed(Nk=0))
    assert "aligned" in _err(packed(out=odd)) and "aligned" in _err(packed(work=odd))
    assert "aligned" in _err(packed(strides=(ctypes.c_int64 * 6)(512, 128, 256, 100, 256, 128)))
    assert "2^23" in _err(packed(strides=(ctypes.c_int64 * 6)(512, 128, 1 << 23, 128, 256, 128)))
    assert "scaling" in _err(packed(scaling=0.0)) and "scaling" in _err(packed(scaling=float("nan")))
    assert "too many rows" in _err(packed(Nq=1 << 30))
    assert lib.reskv_packed_workspace_bytes(1, 4, 4, 2, 1 << 20) > 0
    assert "workspace" in _err(packed(most=1 << 20))
    assert "workspace" in _err(packed(most=1 << 20, work=p, nbytes=64))
    assert lib.reskv_packed_workspace_bytes(0, 4, 4, 2, 1 << 20) == 0

    four = (ctypes.c_int64 * 4)(256, 128, 256, 128)

    def append(pages=p, count=4, tokens=64, Hk=2, width=2, S=1, offsets=p, N=4, strides=four):
        return lib.reskv_int4_append(pages, count, tokens, Hk, p, width, S, p, offsets, p, p, N, strides, None)

    assert "null" in _err(append(pages=None))
    assert "pool sizes" in _err(append(count=0)) and "pool sizes" in _err(append(width=0))
    assert "multiple of 32" in _err(append(tokens=40)) and "multiple of 32" in _err(append(tokens=1 << 30, width=2))
    assert "aligned" in _err(append(pages=odd))
    assert "bad sizes" in _err(append(offsets=None, N=4)) and "bad sizes" in _err(append(S=0))
    assert "aligned" in _err(append(strides=(ctypes.c_int64 * 4)(256, 128, 4, 128)))
    assert "null" in _err(lib.reskv_int4_gather(p, 4, 64, 2, p, 2, 1, p, p, None, p, 4, 1, None))
    assert "aligned" in _err(lib.reskv_int4_gather(p, 4, 64, 2, p, 2, 1, p, p, odd, p, 4, 1, None))

    def attend(q=p, B=1, Hq=4, Hk=2, most=64, out=p, work=None, nbytes=0, width=1 << 15):
        return lib.reskv_int4_attention(q, p, 4, 64, p, width, p, B, Hq, Hk, 1.0, most, out, work, nbytes, None)

    assert "null" in _err(attend(q=None))
    assert "bad sizes" in _err(attend(Hq=5)) and "bad sizes" in _err(attend(B=0))
    assert "negative" in _err(attend(most=-1))
    assert "aligned" in _err(attend(out=odd))
    assert lib.reskv_int4_workspace_bytes(1, 4, 2, 1 << 20) > 0
    assert "workspace" in _err(attend(most=1 << 20))

    pair = (ctypes.c_int32 * 1)(5)
    assert "null" in _err(lib.reskv_copy_pages(p, 1, 4, 32, None, pair, 1, None))
    assert "outside the pool" in _err(lib.reskv_copy_pages(p, 1, 4, 32, pair, pair, 1, None))
    assert "pool sizes" in _err(lib.reskv_copy_pages(p, 1, 8, 24, pair, pair, 1, None))
