"""Which tokens ``Int4Cache.gather`` asks for, on the CPU with the gather replaced by a record."""

import pytest
import torch

from reskv_amd import Int4Cache, int4


@pytest.fixture
def asked(monkeypatch):
    calls = []

    def gather(pages, table, starts, offsets, rows):
        calls.append((starts.tolist(), offsets.tolist(), rows))
        return torch.zeros(rows, 1, 128), torch.zeros(rows, 1, 128)

    monkeypatch.setattr(int4, "int4_gather", gather)
    monkeypatch.setattr(int4, "copy_pages", lambda *a: None)
    return calls


def test_reserved_tokens_can_be_left_out(asked):
    c = Int4Cache(2, 1, 3, 100, page_tokens=32, device="cpu")
    for counts, whole, before in (([40, 0, 7], [0, 40, 40, 47], [0, 0, 0, 0]),
                                  ([5, 60, 0], [0, 45, 105, 112], [0, 40, 40, 47]),
                                  (1, [0, 46, 107, 115], [0, 45, 105, 112])):
        c.reserve(counts)
        for kw, want in ((dict(), whole), (dict(reserved=True), whole), (dict(reserved=False), before)):
            k, v, offsets = c.gather(1, **kw)
            assert offsets.tolist() == want and offsets.dtype is torch.int32 and k.shape[0] == v.shape[0] == want[-1]
            assert asked[-1] == ([0, 0, 0], want, want[-1])
    c.reorder([2, 0, 0])
    assert c.gather(0, reserved=False)[2].tolist() == [0, 7, 52, 97]
    c.release(1)
    assert c.gather(0, reserved=False)[2].tolist() == [0, 7, 7, 52] and c.gather(0)[2].tolist() == [0, 8, 8, 54]
