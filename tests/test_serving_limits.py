"""Sizes past what one launch can count are refused by name before anything is launched (no GPU needed)."""

import ctypes

from reskv_amd import _lib


def refused(status):
    assert status != 0
    return _lib.lib().reskv_last_error().decode()


def test_launches_of_more_than_2_to_the_32_threads_are_refused():
    lib, p = _lib.lib(), ctypes.c_void_p(16)  # never dereferenced: validation fails first
    four = (ctypes.c_int64 * 4)(0, 0, 0, 0)
    for sequences, rows in ((1, (1 << 30) - 1), (1 << 21, 1 << 21)):
        assert "too many rows or sequences" in refused(
            lib.reskv_int4_append(p, 4, 64, 8, p, 2, sequences, p, p, p, p, rows, four, None))
        assert "too many rows or sequences" in refused(
            lib.reskv_int4_gather(p, 4, 64, 8, p, 2, sequences, p, p, p, p, rows, 1, None))
    heads, batch = 64, 1 << 18
    nbytes = lib.reskv_int4_workspace_bytes(batch, heads, 8, 32)
    assert nbytes > 0 and "too many tokens" in refused(
        lib.reskv_int4_attention(p, p, 4, 32, p, 1, p, batch, heads, 8, 1.0, 32, p, p, nbytes, None))
    six = (ctypes.c_int64 * 6)(512, 128, 256, 128, 256, 128)
    assert "too many rows or sequences" in refused(
        lib.reskv_packed_attention(p, p, p, p, p, p, 1 << 20, 1 << 20, 1 << 20, 8, 8, six, 1.0, 4, 0, None, 0, None))
    pair = (ctypes.c_int32 * 1)(1)
    assert "pages are too large" in refused(lib.reskv_copy_pages(p, 1, 4, 1 << 38, pair, pair, 1, None))
