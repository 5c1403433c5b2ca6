"""Causal attention of packed sequences of different lengths.

``RandomLlama.prefill`` and the transformers prompt pass take batches of one length;
``packed_attention`` takes sequences one behind the other, without padding, and chunks of
prompts that continue on keys already there.  Like ``attention`` it is an inference
operator: no gradient is recorded.
"""

import struct
from functools import lru_cache

import torch

from . import _lib
from ._extension import _require, _workspace

_INF = float("inf")


# The checks run for every call of a decode step, so that a message is put together only
# where it is needed.
def _rows(name, t, heads=None):
    if t.dtype is not torch.float16 or t.dim() != 3 or t.shape[2] != 128:
        raise RuntimeError(f"{name} must be fp16 [rows, heads, 128]")
    if heads is not None and t.shape[1] != heads:
        raise RuntimeError(f"{name} has {t.shape[1]} heads, expected {heads}")


def _int32(name, t, count):
    if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous int32 vector")
    if count is not None and t.shape[0] != count:
        raise RuntimeError(f"{name} has {t.shape[0]} entries, expected {count}")


def _same_gpu(first, *others):
    """The index of the GPU that all tensors are on.  Checked last, after every shape, dtype and layout check."""
    index = first.get_device() if first.is_cuda else -1
    for t in others:
        if t is not None and (not t.is_cuda or t.get_device() != index):
            index = -1
    if index < 0:
        _require(all(t is None or t.is_cuda for t in (first, *others)), "every tensor must be a CUDA tensor")
        raise RuntimeError("all tensors must be on the same GPU")
    return index


def _launch(name, index, *args):
    """Calls the library's ``name`` on the current stream of GPU ``index``, made the current device
    meanwhile: a launch goes to the current device, whatever the device of its pointers."""
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _launch(name, index, *args)
    status = getattr(_lib.lib(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def _kernel_rows(t, least=0, most=1 << 62):
    """t itself when its rows of 128 channels can be read in place (16-byte aligned; token stride
    from ``least`` to below ``most``), else a contiguous copy."""
    token, head, channel = t.stride()
    if channel == 1 and not (token | head) & 7 and least <= token < most and not t.data_ptr() & 15:
        return t
    return t.detach().clone(memory_format=torch.contiguous_format)


def _new(like, shape):
    """An fp16 tensor (a plain one, also for a subclass's ``like``) on the GPU of ``like``."""
    if type(like) is torch.Tensor:
        return torch.empty_like(like) if like.shape == shape and like.is_contiguous() else like.new_empty(shape)
    return torch.empty(shape, dtype=torch.float16, device=like.device)


_pack = [struct.Struct(f"{2 * n}q").pack for n in range(4)]


def _strides(*tensors):
    """Token and head strides of row tensors, as the library reads them (int64 values in memory)."""
    return _pack[len(tensors)](*(n for t in tensors for n in t.stride()[:2]))


@lru_cache(4096)  # a function of the sizes alone
def _packed_workspace(sequences, queries, heads, kv_heads, most):
    return _lib.lib().reskv_packed_workspace_bytes(sequences, queries, heads, kv_heads, most)


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
    ``out`` when given (contiguous, apart from k and v); rows of no sequence are zero, or left as they are in ``out``.

    Scores and sums are fp32; the softmax weights are rounded to fp16 for the product with V.  Offsets
    are not read on the host: values outside the tensors are clamped into them.
    """
    _rows("q", q)
    _rows("k", k)
    _rows("v", v, k.shape[1])
    _require(k.shape[0] == v.shape[0], "k and v must have the same number of rows")
    nq, heads, _ = q.shape
    nk, kv_heads, _ = k.shape
    _require(kv_heads > 0 and heads > 0 and heads % kv_heads == 0, "the query heads must be a multiple of the KV heads")
    _int32("q_offsets", q_offsets, None)
    count = q_offsets.shape[0] - 1
    _require(count >= 1, "q_offsets needs the start and the end of at least one sequence")
    if k_offsets is None:
        k_offsets = q_offsets
    else:
        _int32("k_offsets", k_offsets, count + 1)
    scaling = 128 ** -0.5 if scaling is None else float(scaling)
    _require(0.0 < scaling < _INF, "scaling must be positive")
    most = nk if max_keys is None else int(max_keys)
    _require(most >= 0, "max_keys must not be negative")
    clear = out is None
    if not clear:
        _rows("out", out, heads)
        _require(out.shape[0] == nq and out.is_contiguous(), "out must be contiguous and have a row for every query")
    index = _same_gpu(q, k, v, q_offsets, k_offsets, out)
    if clear:
        out = _new(q, (nq, heads, 128))
    if nq == 0:
        return out
    if nk == 0:  # nobody sees anything
        if clear:
            return out.zero_()
        k = v = _new(q, (1, kv_heads, 128))
        k_offsets, nk = torch.zeros_like(q_offsets), 1
    q, k, v = _kernel_rows(q), _kernel_rows(k, 128, 1 << 23), _kernel_rows(v, 128, 1 << 23)
    nbytes = _packed_workspace(count, nq, heads, kv_heads, most)
    work = _workspace(nbytes, q.device) if nbytes else None
    _launch("reskv_packed_attention", index, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            q_offsets.data_ptr(), k_offsets.data_ptr(), count, nq, nk, heads, kv_heads, _strides(q, k, v), scaling, most,
            clear, None if work is None else work.data_ptr(), nbytes)
    return out
