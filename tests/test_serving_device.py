"""Packed attention and the 4-bit cache launch with their tensors' GPU as the current device and on its current
stream, and take tensors of one GPU only.  On the CPU, with the library, the device switch, the stream lookup and the
tensors' devices replaced by records."""

import contextlib

import pytest
import torch

from reskv_amd import int4, packed
from reskv_amd.int4 import copy_pages, empty_pages, int4_append, int4_attention, int4_gather
from reskv_amd.packed import packed_attention

f16 = dict(dtype=torch.float16)
i32 = dict(dtype=torch.int32)


class _Library:
    def __init__(self, current):
        self.calls, self.current = [], current

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_bytes"):
                return 64
            self.calls.append((name, self.current[-1], args[-1]))
            return 0

        return call


@pytest.fixture
def library(monkeypatch):
    """A process with GPU 0 current, tensors on GPU 3."""
    current = [0]

    @contextlib.contextmanager
    def device(index):
        current.append(index)
        yield
        current.pop()

    lib = _Library(current)
    packed._packed_workspace.cache_clear()
    int4._attention_workspace.cache_clear()
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[-1], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(packed._lib, "lib", lambda: lib)
    for module in (packed, int4):
        monkeypatch.setattr(module, "_same_gpu", lambda *t: 3)
    yield lib
    packed._packed_workspace.cache_clear()
    int4._attention_workspace.cache_clear()


def test_every_launch_is_on_the_tensors_gpu(library):
    pages = empty_pages(4, 2, 64, device="cpu")
    table, starts = torch.zeros(2, 2, **i32), torch.zeros(2, **i32)
    rows, q = torch.zeros(2, 2, 128, **f16), torch.zeros(2, 4, 128, **f16)
    ends = torch.tensor([0, 1, 2], **i32)
    int4_append(pages, table, starts, rows, rows)
    int4_gather(pages, table, starts, ends, 2)
    int4_attention(q, pages, table, starts)
    copy_pages(pages, [0], [1])
    packed_attention(q, rows, rows, ends)
    assert library.calls == [(n, 3, 103) for n in ("reskv_int4_append", "reskv_int4_gather", "reskv_int4_attention",
                                                   "reskv_copy_pages", "reskv_packed_attention")]
    assert library.current == [0]


class _On:
    """Stands for a tensor: where it is."""

    def __init__(self, index):
        self.is_cuda, self.index = index >= 0, index

    def get_device(self):
        return self.index


def test_tensors_must_share_a_gpu():
    assert packed._same_gpu(_On(2), None, _On(2)) == 2
    for tensors in ((_On(0), _On(1)), (_On(1), _On(1), _On(0))):
        with pytest.raises(RuntimeError, match="on the same GPU"):
            packed._same_gpu(*tensors)
    for tensors in ((_On(-1),), (_On(0), _On(-1)), (_On(-1), _On(0))):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            packed._same_gpu(*tensors)


def test_no_gradient_is_recorded(library):
    """Inference operators: tensors that require gradients are read, and nothing is recorded."""
    q = torch.zeros(2, 4, 128, **f16, requires_grad=True)
    rows = torch.zeros(2, 2, 128, **f16, requires_grad=True)
    wide = torch.zeros(2, 2, 256, **f16, requires_grad=True)[..., ::2]  # copied first
    out = packed_attention(q, rows, wide, torch.tensor([0, 1, 2], **i32))
    assert not out.requires_grad and out.shape == q.shape
    pages, table, starts = empty_pages(4, 2, 64, device="cpu"), torch.zeros(2, 2, **i32), torch.zeros(2, **i32)
    assert not int4_attention(torch.nn.Parameter(q.detach()), pages, table, starts).requires_grad
