"""Causal attention of packed sequences of different lengths.

``RandomLlama.prefill`` and the transformers prompt pass take batches of one length;
``packed_attention`` takes sequences one behind the other, without padding, and chunks of
prompts that continue on keys already there.  Like ``attention`` it is an inference
operator: no gradient is recorded.
"""

import ctypes

import torch

from . import _lib
from ._extension import _require, _stream, _workspace

_STRIDES = ctypes.c_int64 * 6


def _rows(name, t, heads=None):
    _require(t.dtype == torch.float16 and t.dim() == 3 and t.shape[2] == 128, f"{name} must be fp16 [rows, heads, 128]")
    _require(heads is None or t.shape[1] == heads, f"{name} has {t.shape[1]} heads, expected {heads}")


def _int32(name, t, count):
    _require(t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous(), f"{name} must be a contiguous int32 vector")
    _require(count is None or t.shape[0] == count, f"{name} has {t.shape[0]} entries, expected {count}")


def _same_gpu(*tensors):
    """Checked last, after every shape, dtype and layout check."""
    _require(all(t is None or t.is_cuda for t in tensors), "every tensor must be a CUDA tensor")
    dev = tensors[0].device
    _require(all(t is None or t.device == dev for t in tensors), "all tensors must be on the same GPU")
    return dev


def _launch(name, dev, *args):
    """Calls the library's ``name`` on the current stream of dev, made the current device meanwhile: a
    launch goes to the current device, whatever the device of its pointers."""
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == dev.index:
        _lib.check(fn(*args, _stream(dev)), name)
    else:
        with torch.cuda.device(dev):
            _lib.check(fn(*args, _stream(dev)), name)


def _kernel_rows(t, most=None):
    """t itself when its rows of 128 channels can be read in place (16-byte aligned; token stride
    below ``most``), else a contiguous copy."""
    token, head, channel = t.stride()
    fits = channel == 1 and token % 8 == 0 and head % 8 == 0 and t.data_ptr() % 16 == 0
    return t if fits and (most is None or token < most) else t.clone(memory_format=torch.contiguous_format)


@torch.no_grad()
def packed_attention(q, k, v, q_offsets, k_offsets=None, *, scaling=None, max_keys=None, out=None):
    """Causal attention of S sequences packed one behind the other.

    q fp16 [Nq, Hq, 128] and k, v fp16 [Nk, Hk, 128] (q and k rotated; any strides with unit channel
    stride are read in place); Hq a multiple of Hk.  Sequence s has the query rows ``q_offsets[s]``
    to ``q_offsets[s + 1]`` (int32 [S + 1] on the GPU) and the key rows that ``k_offsets`` gives
    (default: the same).  Its last query sees all its keys, the one before all but the last, and
    so on: with nq queries and nk keys, query i sees the keys 0 .. i + nk - nq, so that a chunk
    of a prompt, or a single token, attends the keys before it as well; a query that sees none gives zeros.
    What a query does not see does not matter to it, NaN and infinities included.

    ``scaling`` (positive) defaults to 128 ** -0.5; ``max_keys`` bounds the keys of a sequence
    (default: all of k) and only steers how the work is split.  Returns fp16 [Nq, Hq, 128],
    ``out`` when given (contiguous); rows of no sequence are zero, or left as they are in ``out``.

    Scores and sums are fp32; the softmax weights are rounded to fp16 for the product with V.  Offsets
    are not read on the host: values outside the tensors are clamped into them.
    """
    _rows("q", q)
    _rows("k", k)
    _rows("v", v, k.shape[1])
    _require(k.shape[0] == v.shape[0], "k and v must have the same number of rows")
    nq, heads = q.shape[0], q.shape[1]
    nk, kv_heads = k.shape[0], k.shape[1]
    _require(kv_heads > 0 and heads > 0 and heads % kv_heads == 0, "the query heads must be a multiple of the KV heads")
    _int32("q_offsets", q_offsets, None)
    count = q_offsets.shape[0] - 1
    _require(count >= 1, "q_offsets needs the start and the end of at least one sequence")
    if k_offsets is None:
        k_offsets = q_offsets
    else:
        _int32("k_offsets", k_offsets, count + 1)
    scaling = 128 ** -0.5 if scaling is None else float(scaling)
    _require(scaling > 0.0 and scaling < float("inf"), "scaling must be positive")
    most = nk if max_keys is None else int(max_keys)
    _require(most >= 0, "max_keys must not be negative")
    clear = out is None
    if not clear:
        _rows("out", out, heads)
        _require(out.shape[0] == nq and out.is_contiguous(), "out must be contiguous and have a row for every query")
    dev = _same_gpu(q, k, v, q_offsets, k_offsets, out)
    if clear:
        out = torch.empty((nq, heads, 128), dtype=torch.float16, device=dev)
    if nq == 0:
        return out
    if nk == 0:  # nobody sees anything
        if clear:
            return out.zero_()
        k = v = torch.empty((1, kv_heads, 128), dtype=torch.float16, device=dev)
        k_offsets, nk = torch.zeros_like(q_offsets), 1
    q, k, v = _kernel_rows(q), _kernel_rows(k, 1 << 23), _kernel_rows(v, 1 << 23)
    nbytes = _lib.lib().reskv_packed_workspace_bytes(count, nq, heads, kv_heads, most)
    work = _workspace(nbytes, dev) if nbytes else None
    strides = _STRIDES(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2])
    _launch("reskv_packed_attention", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            q_offsets.data_ptr(), k_offsets.data_ptr(), count, nq, nk, heads, kv_heads, strides, scaling, most,
            int(clear), None if work is None else work.data_ptr(), nbytes)
    return out
