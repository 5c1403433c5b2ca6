"""Trees of drafted tokens: their masks, and which of them a target model accepts.

A sequence's tree has up to 64 nodes, parents before children, one row each in packed tensors.  Node 0 is its root, the token
that was sampled last; the others are drafts, a chain or a tree.  A decoding step runs all nodes through the model
(``int4_append_rope`` puts their keys into the cache, ``int4_tree_attention`` attends them), lets ``verify_drafts`` find
what the model agrees with, and keeps that (``Int4Cache.keep``); ``GreedyDecoder.step_drafts`` does it.

Like the cache's operators these read their offsets, parents and tokens on the GPU only, and may be captured.
"""

from functools import lru_cache

import torch

from . import _lib
from ._extension import _require, _workspace
from .int4 import TREE_NODES
from .packed import _INF, _int32, _launch, _same_gpu


def draft_tree(parents, offsets, starts=None):
    """(seen, positions) of trees: rows ``offsets[s]`` to ``offsets[s + 1]`` (int32 [S + 1]) of ``parents`` (int32 [N]) name
    the parent of every node of sequence s, a node before it; anything else is none.

    ``seen`` (int64 [N]) has bit j set in the mask of node i where j is i or an ancestor of it, as ``int4_tree_attention``
    takes it; ``positions`` (int32 [N]) is a node's depth, with ``starts`` (int32 [S]) behind that many tokens, as ``int4_append_rope``
    takes them.  Rows of no sequence, and nodes from the 64th on, get zeros.
    """
    _int32("parents", parents, None)
    _int32("offsets", offsets, None)
    sequences = offsets.shape[0] - 1
    _require(sequences >= 1, "offsets needs the start and the end of at least one sequence")
    if starts is not None:
        _int32("starts", starts, sequences)
    index = _same_gpu(parents, offsets, starts)
    n = parents.shape[0]
    seen = torch.zeros(n, dtype=torch.int64, device=parents.device)
    positions = torch.zeros(n, dtype=torch.int32, device=parents.device)
    if n:
        _launch("reskv_draft_tree", index, parents.data_ptr(), offsets.data_ptr(), None if starts is None else starts.data_ptr(),
                sequences, n, seen.data_ptr(), positions.data_ptr())
    return seen, positions


@lru_cache(4096)  # a function of the sizes alone
def _verify_workspace(sequences, rows, vocab):
    return _lib.lib().reskv_verify_workspace_bytes(sequences, rows, vocab)


def _matrix(name, t, dtypes, shape):
    """t must be a matrix of the shape with contiguous rows that do not overlap; returns its row stride."""
    if t.dtype not in dtypes or t.dim() != 2:
        raise RuntimeError(f"{name} must be a matrix of {' or '.join(str(d)[6:] for d in dtypes)}")
    rows, columns = t.shape
    if shape is not None and (rows, columns) != shape:
        raise RuntimeError(f"{name} must be [{shape[0]}, {shape[1]}]")
    row, column = t.stride()
    if not (column == 1 or columns == 1) or (rows > 1 and row < columns):
        raise RuntimeError(f"{name} must have contiguous rows")
    return row if rows > 1 else columns


def verify_drafts(logits, tokens, parents, offsets, accept=None, sample=None, *, draft=None, temperature=1.0):
    """Which nodes of every sequence's tree the target model accepts, and the token behind them: (path, counts, token).

    Row ``offsets[s] + i`` (int32 [S + 1]) of ``logits`` (fp16 or fp32 [N, V]) is what the target says behind node i of
    sequence s, of ``tokens`` (int64 [N]) and ``parents`` (int32 [N]) its token and its parent.  The walk starts at the root
    with r = softmax(logits / temperature) and goes through the nodes in their order.  A child x of the node
    reached, with token t, drawn from the distribution q (``draft[row]``, fp32 [N, V]; None: x was not drawn, q is one at t), is
    accepted if ``accept[row] * q(t) < r(t) / sum(r)``; the walk goes on from it with its own r.  Else r becomes ``max(r / sum(r)
    - q, 0)`` (or stays, where that leaves nothing).  The token at the end is the first with ``r(0) + .. + r(t) > sample[s] * sum(r)``.
    With ``accept`` (fp32 [N]) and ``sample`` (fp32 [S]) uniform on [0, 1), accepted tokens and the one behind them are
    distributed as the target model's own, whatever the drafts are.

    With temperature 0 the child is accepted whose token is the argmax (the lowest of equals), which is the token at the end;
    ``accept``, ``sample`` and ``draft`` are not read.

    ``path`` (int32 [S, 64]) lists the nodes reached, the root first and -1 behind them, ``counts`` (int32 [S]) says how many,
    ``token`` is int64 [S].  A node whose token is outside the vocabulary is passed over.  A token is -1 where the row reached
    has no distribution (a NaN, plus infinity, or nothing but minus infinity; with temperature 0 a NaN), and where a sequence has no
    nodes (its count is 0).  Sums and probabilities are 64 bits.
    """
    stride = _matrix("logits", logits, (torch.float16, torch.float32), None)
    n, vocab = logits.shape
    _require(0 < vocab < 1 << 30, "logits must have a column for every token")
    _require(tokens.dtype is torch.int64 and tokens.dim() == 1 and tokens.is_contiguous() and tokens.shape[0] == n,
             "tokens must be a contiguous int64 vector with a token for every row of logits")
    _int32("parents", parents, n)
    _int32("offsets", offsets, None)
    sequences = offsets.shape[0] - 1
    _require(sequences >= 1, "offsets needs the start and the end of at least one sequence")
    temperature = float(temperature)
    _require(0.0 <= temperature < _INF, "temperature must be finite and not negative")
    _require(temperature == 0.0 or temperature >= 1e-30, "a temperature that is not 0 must be 1e-30 or more")
    draft_stride = 0
    if temperature == 0.0:
        accept = sample = draft = None
    else:
        for name, t, count in (("accept", accept, n), ("sample", sample, sequences)):
            if t is None or t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != count or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous fp32 vector of {count} random numbers")
        if draft is not None:
            draft_stride = _matrix("draft", draft, (torch.float32,), (n, vocab))
    index = _same_gpu(logits, tokens, parents, offsets, accept, sample, draft)
    device = logits.device
    path = torch.empty((sequences, TREE_NODES), dtype=torch.int32, device=device)
    counts = torch.empty((sequences,), dtype=torch.int32, device=device)
    token = torch.empty((sequences,), dtype=torch.int64, device=device)
    if n == 0:
        return path.fill_(-1), counts.zero_(), token.fill_(-1)
    if logits.data_ptr() & 15:
        logits = logits.detach().clone(memory_format=torch.contiguous_format)
        stride = vocab
    nbytes = _verify_workspace(sequences, n, vocab)
    work = _workspace(nbytes, device)
    _launch("reskv_verify_drafts", index, logits.data_ptr(), logits.dtype is torch.float32, stride, tokens.data_ptr(),
            parents.data_ptr(), offsets.data_ptr(), None if accept is None else accept.data_ptr(),
            None if sample is None else sample.data_ptr(), None if draft is None else draft.data_ptr(), draft_stride, temperature,
            sequences, n, vocab, path.data_ptr(), counts.data_ptr(), token.data_ptr(), work.data_ptr(), nbytes)
    return path, counts, token
