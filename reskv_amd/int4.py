"""Paged cache of 4-bit keys and values, and the operators on its pages.

A pool is a uint8 tensor [pages, KV heads, bytes] (``empty_pages``; 160 bytes per token and head, K and V
together, against 512 in fp16); a sequence's tokens lie in the pages that its row of an
int32 page table names.  Every row of 128 channels is quantised in groups of 32: ``low`` is
the group's smallest value and ``scale`` a fifteenth of its range, both fp16, and a channel is stored as the
nearest of the sixteen values ``code * scale + low``.

* ``int4_append`` puts rows of K and V into pages, prompts and single tokens alike;
* ``int4_gather`` gives them back in fp16, for a prompt that continues on cached tokens;
* ``int4_attention`` attends one token of every sequence over its pages;
* ``copy_pages`` copies pages in every layer's pool at once;
* ``Int4Cache`` keeps the pages of a decoder stack: which sequence has which, forks that share
  them, their release and compaction.

K is stored as it is given: rotated keys, as the dense ring of ``ResKVLayerCache`` has them.
Like ``attention`` these are inference operators: no gradient is recorded.  Page tables, positions and
lengths stay on the GPU and are not read on the host: a page number outside the pool, or a position outside
the table, stands for a token that is not there, which appends leave out and reads pass over.
"""

import ctypes
from functools import lru_cache

import torch

from . import _lib
from ._extension import _require, _workspace
from .packed import _INF, _int32, _kernel_rows, _launch, _new, _rows, _same_gpu, _strides

BLOCK_TOKENS = 32
TOKEN_BYTES = 160  # of one KV head, K and V


def _page_bytes(page_tokens):
    page_tokens = int(page_tokens)
    _require(page_tokens >= BLOCK_TOKENS and page_tokens % BLOCK_TOKENS == 0,
             f"a page must hold a positive multiple of {BLOCK_TOKENS} tokens")
    return page_tokens * TOKEN_BYTES


def empty_pages(pages, kv_heads, page_tokens=64, layers=None, device="cuda"):
    """A pool of unused pages: uint8 [pages, kv_heads, bytes], or [layers, pages, kv_heads, bytes]."""
    shape = (int(pages), int(kv_heads), _page_bytes(page_tokens))
    _require(shape[0] > 0 and shape[1] > 0, "a pool needs pages and KV heads")
    return torch.zeros(shape if layers is None else (int(layers), *shape), dtype=torch.uint8, device=device)


def _pool(pages):
    """(pages, tokens per page, KV heads) of a pool."""
    _require(pages.dtype is torch.uint8 and pages.dim() == 3 and pages.is_contiguous(),
             "pages must be a contiguous uint8 tensor [pages, KV heads, bytes]")
    count, heads, nbytes = pages.shape
    if not (count > 0 and heads > 0 and nbytes > 0 and nbytes % (BLOCK_TOKENS * TOKEN_BYTES) == 0):
        raise RuntimeError(f"a page must hold a positive multiple of {BLOCK_TOKENS} tokens of {TOKEN_BYTES} bytes")
    return count, nbytes // TOKEN_BYTES, heads


def _table(table):
    _require(table.dtype is torch.int32 and table.dim() == 2 and table.is_contiguous() and table.shape[1] > 0,
             "table must be a contiguous int32 matrix [sequences, pages]")
    return table.shape


def int4_append(pages, table, starts, k, v, offsets=None):
    """Quantises rows of k and v, fp16 [N, Hk, 128] (any strides with unit channel stride), into pages.

    Without ``offsets``, row s becomes token ``starts[s]`` of sequence s (a decode step); with them
    (int32 [S + 1]), row ``offsets[s] + i`` becomes token ``starts[s] + i``.  ``starts`` is int32 [S], ``table`` int32 [S,
    pages of a sequence].  Tokens of a block before and behind the new ones keep their values.  A group of
    channels that holds a NaN or an infinity reads as NaN.  No two sequences of a call may write to one page.
    """
    count, tokens, heads = _pool(pages)
    sequences, width = _table(table)
    _int32("starts", starts, sequences)
    _rows("k", k, heads)
    _rows("v", v, heads)
    n = k.shape[0]
    _require(v.shape[0] == n, "k and v must have the same number of rows")
    if offsets is None:
        _require(n == sequences, "without offsets there must be one row for every sequence")
    else:
        _int32("offsets", offsets, sequences + 1)
    index = _same_gpu(pages, table, starts, k, v, offsets)
    if n == 0 or sequences == 0:
        return
    k, v = _kernel_rows(k), _kernel_rows(v)
    _launch("reskv_int4_append", index, pages.data_ptr(), count, tokens, heads, table.data_ptr(), width, sequences,
            starts.data_ptr(), None if offsets is None else offsets.data_ptr(), k.data_ptr(), v.data_ptr(), n,
            _strides(k, v))


def int4_gather(pages, table, starts, offsets, rows, out=None):
    """The stored values of tokens, as (k, v) fp16 [rows, Hk, 128]: row ``offsets[s] + i`` is token
    ``starts[s] + i`` of sequence s (``rows`` is what ``offsets`` ends with; the host does not read it).

    ``out`` = (k, v) to write to, contiguous; rows of no token are zero, or left as they are in ``out``.
    """
    count, tokens, heads = _pool(pages)
    sequences, width = _table(table)
    _int32("starts", starts, sequences)
    _int32("offsets", offsets, sequences + 1)
    rows = int(rows)
    _require(rows >= 0, "rows must not be negative")
    clear = out is None
    if not clear:
        for name, t in zip(("out k", "out v"), out):
            _rows(name, t, heads)
            _require(t.shape[0] == rows and t.is_contiguous(), f"{name} must be contiguous and have {rows} rows")
    k, v = (None, None) if clear else out
    index = _same_gpu(pages, table, starts, offsets, k, v)
    if clear:
        shape = (rows, heads, 128)
        k, v = pages.new_empty(shape, dtype=torch.float16), pages.new_empty(shape, dtype=torch.float16)
    if rows == 0:
        return k, v
    if sequences == 0:
        return (k.zero_(), v.zero_()) if clear else (k, v)
    _launch("reskv_int4_gather", index, pages.data_ptr(), count, tokens, heads, table.data_ptr(), width, sequences,
            starts.data_ptr(), offsets.data_ptr(), k.data_ptr(), v.data_ptr(), rows, clear)
    return k, v


@lru_cache(4096)  # a function of the sizes alone
def _attention_workspace(sequences, heads, kv_heads, most):
    return _lib.lib().reskv_int4_workspace_bytes(sequences, heads, kv_heads, most)


def int4_attention(q, pages, table, lengths, *, scaling=None, max_length=None, out=None):
    """Attention of one token of every sequence: q fp16 [B, Hq, 128] (rotated) against the first
    ``lengths[b]`` (int32 [B]) tokens of sequence b; fp16 [B, Hq, 128], ``out`` when given (contiguous).

    Hq is any multiple of the pool's KV heads.  A sequence without tokens gives zeros.  ``max_length`` bounds
    the lengths (default: what the table can hold; a longer length is cut to it) and steers how the work
    is split over the GPU; a captured call keeps it.  Scores, softmax and sums are fp32; a weight times a scale of V is
    rounded to fp16, once, for the product with V's codes (where it is 2^-20 of the largest such product of its query head and
    channel group, or less, to 2^-31 of that).
    """
    count, tokens, kv_heads = _pool(pages)
    sequences, width = _table(table)
    _int32("lengths", lengths, sequences)
    _rows("q", q)
    heads = q.shape[1]
    _require(q.shape[0] == sequences, "q must have one row for every sequence")
    _require(heads > 0 and heads % kv_heads == 0, "the query heads must be a multiple of the KV heads")
    scaling = 128 ** -0.5 if scaling is None else float(scaling)
    _require(-_INF < scaling < _INF, "scaling must be finite")
    most = width * tokens if max_length is None else int(max_length)
    _require(most >= 0, "max_length must not be negative")
    if out is not None:
        _rows("out", out, heads)
        _require(out.shape[0] == sequences and out.is_contiguous(), "out must be contiguous and shaped like q")
    index = _same_gpu(q, pages, table, lengths, out)
    if out is None:
        out = _new(q, (sequences, heads, 128))
    if sequences == 0:
        return out
    if not q.is_contiguous() or q.data_ptr() & 15:
        q = q.detach().clone(memory_format=torch.contiguous_format)
    most = min(most, width * tokens)
    nbytes = _attention_workspace(sequences, heads, kv_heads, most)
    work = _workspace(nbytes, q.device)
    _launch("reskv_int4_attention", index, q.data_ptr(), pages.data_ptr(), count, tokens, table.data_ptr(), width,
            lengths.data_ptr(), sequences, heads, kv_heads, scaling, most, out.data_ptr(),
            work.data_ptr(), nbytes)
    return out


def copy_pages(pages, source, target):
    """Copies page ``source[i]`` to page ``target[i]`` (host sequences of page numbers) in a pool [pages, ...]
    or in every layer's pool [layers, pages, KV heads, bytes], in one launch per 384 pages.

    A target may be neither a source nor named twice: what it would hold then depends on the order.
    """
    _require(pages.dtype is torch.uint8 and pages.dim() in (3, 4) and pages.is_contiguous(),
             "pages must be a contiguous uint8 tensor [pages, KV heads, bytes] or [layers, pages, KV heads, bytes]")
    source, target = list(map(int, source)), list(map(int, target))
    _require(len(source) == len(target), "every source page needs a target page")
    layers, count = (1, pages.shape[0]) if pages.dim() == 3 else pages.shape[:2]
    nbytes = pages.shape[-2] * pages.shape[-1]
    _require(nbytes > 0 and nbytes % 16 == 0, "a page must be a multiple of 16 bytes")
    if source and not (0 <= min(source) and max(source) < count and 0 <= min(target) and max(target) < count):
        raise RuntimeError(f"page numbers must be in 0 .. {count - 1}")
    written = set(target)
    _require(len(written) == len(target) and written.isdisjoint(source),
             "a target page may be neither a source nor named twice")
    index = _same_gpu(pages)
    n = len(source)
    if n == 0 or layers == 0:
        return
    pairs = ctypes.c_int32 * n
    _launch("reskv_copy_pages", index, pages.data_ptr(), layers, count, nbytes, pairs(*source), pairs(*target), n)


class Int4Cache:
    """Paged 4-bit K/V cache of a decoder stack: ``sequences`` rows of up to ``max_length`` tokens over one pool
    of pages per layer, with one page table for all layers.

    A step reserves its tokens once, then every layer appends and attends::

        cache.reserve(1)                       # or one count per sequence
        for layer in range(layers):
            cache.append(layer, k, v)          # rotated K, V [sequences, Hk, 128]
            out = cache.attend(layer, q)       # rotated Q [sequences, Hq, 128]

    Which page belongs to whom is kept on the host; ``table``, ``starts`` (of the reserved tokens) and
    ``lengths`` (with them) are its copies on the GPU, at fixed addresses, so that appends and attention
    may be captured into a graph and replayed after every ``reserve``, which itself stays outside.  Sequences that
    were forked share pages; ``reserve`` gives a sequence a copy of its last page before it writes to a shared one.
    """

    def __init__(self, layers, kv_heads, sequences, max_length, *, page_tokens=64, pages=None, device="cuda"):
        _require(int(layers) > 0 and int(sequences) > 0 and int(max_length) > 0,
                 "a cache needs layers, sequences and a length")
        _page_bytes(page_tokens)
        self.page_tokens, self.max_length = int(page_tokens), int(max_length)
        width = -(-self.max_length // self.page_tokens)
        self.pool = empty_pages(int(sequences) * width if pages is None else pages, kv_heads, page_tokens, layers, device)
        self._table = torch.full((int(sequences), width), -1, dtype=torch.int32)
        self.table = self._table.to(device, copy=True)
        self.starts = torch.zeros(int(sequences), dtype=torch.int32, device=device)
        self.lengths = torch.zeros_like(self.starts)
        self._pages = [[] for _ in range(int(sequences))]
        self._lengths = [0] * int(sequences)
        self._counts = [0] * int(sequences)          # tokens reserved last
        self._forked = False                         # rows may share pages that the reserved tokens lie in
        self._users = [0] * self.pool.shape[1]       # sequences that have a page
        self._free = list(range(self.pool.shape[1] - 1, -1, -1))  # the lowest number last

    # -- state ---------------------------------------------------------------
    @property
    def sequences(self) -> int:
        return len(self._lengths)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def get_seq_length(self, sequence=0) -> int:
        return self._lengths[sequence]

    def _row(self, sequence):
        _require(0 <= int(sequence) < self.sequences, f"sequence {sequence} is not in 0 .. {self.sequences - 1}")
        return int(sequence)

    def _publish(self, rows):
        """The page table's changed rows, to the GPU."""
        for s in rows:
            self._table[s] = -1
            self._table[s, : len(self._pages[s])] = torch.tensor(self._pages[s], dtype=torch.int32)
        if rows:
            self.table.copy_(self._table)

    def _publish_lengths(self):
        starts = [n - c for n, c in zip(self._lengths, self._counts)]
        both = torch.tensor([starts, self._lengths], dtype=torch.int32).to(self.lengths.device)
        self.starts.copy_(both[0])
        self.lengths.copy_(both[1])

    def _drop(self, pages):
        freed = False
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                self._free.append(p)
                freed = True
        if freed:
            self._free.sort(reverse=True)

    # -- tokens ----------------------------------------------------------------
    def reserve(self, counts):
        """Makes room for ``counts`` more tokens (one number for every sequence, or one for each); the
        appends that follow fill it.  Raises before any change when a sequence would pass
        ``max_length`` or the pool has too few free pages."""
        _require(not (self.pool.is_cuda and torch.cuda.is_current_stream_capturing()),
                 "reserve works on the host and cannot be captured")
        same = isinstance(counts, int)
        counts = [counts] * self.sequences if same else [int(c) for c in counts]
        _require(len(counts) == self.sequences and min(counts) >= 0, "reserve needs a count of tokens for every sequence")
        ends = [n + c for n, c in zip(self._lengths, counts)]
        _require(max(ends) <= self.max_length, f"a sequence would pass {self.max_length} tokens")
        size, need, shared, users = self.page_tokens, 0, [], {}
        for s, (n, c) in enumerate(zip(self._lengths, counts)):
            need += -(-ends[s] // size) - len(self._pages[s])
            if c and n % size:  # writes to its last page
                last = self._pages[s][-1]
                left = users.get(last, self._users[last])
                if left > 1:  # of those who share it, the last one keeps it
                    shared.append(s)
                    users[last] = left - 1
        need += len(shared)
        _require(need <= len(self._free), f"{need} pages are needed and {len(self._free)} are free")
        if shared:
            source = [self._pages[s][-1] for s in shared]
            target = [self._free.pop() for _ in shared]
            copy_pages(self.pool, source, target)
            for s, a, b in zip(shared, source, target):
                self._users[a] -= 1
                self._users[b] = 1
                self._pages[s][-1] = b
        changed = set(shared)
        for s, end in enumerate(ends):
            while len(self._pages[s]) * size < end:
                p = self._free.pop()
                self._users[p] = 1
                self._pages[s].append(p)
                changed.add(s)
        self._publish(sorted(changed))
        self._lengths, self._counts, self._forked = ends, counts, False
        if same:
            self.starts.copy_(self.lengths)
            self.lengths.add_(counts[0])
        else:
            self._publish_lengths()

    def append(self, layer, k, v, offsets=None):
        """The reserved tokens of one layer (``int4_append``): one row per sequence, or rows packed by ``offsets``
        (on the GPU, so that their counts are not compared with the reserved ones)."""
        _require(not self._forked, "sequences were forked: reserve tokens before the next append")
        int4_append(self.pool[layer], self.table, self.starts, k, v, offsets)

    def attend(self, layer, q, *, scaling=None, out=None):
        """Attention of one token per sequence over all its tokens (``int4_attention``)."""
        return int4_attention(q, self.pool[layer], self.table, self.lengths, scaling=scaling, out=out)

    def gather(self, layer, *, reserved=True):
        """(k, v, offsets): the stored values of all tokens, packed (``int4_gather``), as
        ``packed_attention`` takes them for a prompt that continues.

        The tokens reserved last are among them, so they have to be appended to this layer first.  With
        ``reserved=False`` they are left out: what the cache held before, for a chunk whose own fp16 rows
        are put behind each sequence's.
        """
        ends = self._lengths if reserved else [n - c for n, c in zip(self._lengths, self._counts)]
        ends = torch.tensor([0, *ends], dtype=torch.int64).cumsum(0)
        offsets = ends.to(torch.int32).to(self.table.device)
        k, v = int4_gather(self.pool[layer], self.table, torch.zeros_like(self.starts), offsets, int(ends[-1]))
        return k, v, offsets

    # -- sequences ---------------------------------------------------------------
    def reorder(self, index):
        """Row i takes the tokens of row ``index[i]`` (beams): pages are shared, not copied."""
        index = [self._row(s) for s in (index.tolist() if torch.is_tensor(index) else index)]
        _require(len(index) == self.sequences, "reorder needs a row for every sequence")
        pages = [list(self._pages[s]) for s in index]
        for row in pages:
            for p in row:
                self._users[p] += 1
        self._forked |= len(set(index)) < len(index)
        old, self._pages = self._pages, pages
        self._drop(p for row in old for p in row)
        self._lengths = [self._lengths[s] for s in index]
        self._counts = [self._counts[s] for s in index]
        self._publish(list(range(self.sequences)))
        self._publish_lengths()

    def fork(self, source, target):
        """Row ``target`` gives up its tokens and shares those of row ``source``."""
        index = list(range(self.sequences))
        index[self._row(target)] = self._row(source)
        self.reorder(index)

    def release(self, sequence):
        """Row ``sequence`` gives up its tokens; pages that no other row shares are free again."""
        s = self._row(sequence)
        pages, self._pages[s] = self._pages[s], []
        self._lengths[s] = self._counts[s] = 0
        self._drop(pages)
        self._publish([s])
        self._publish_lengths()

    def compact(self):
        """Moves pages in use to the lowest numbers, so that the rest of the pool is free in one piece;
        returns how many were moved."""
        used = len(self._users) - len(self._free)
        source = [p for p in range(used, len(self._users)) if self._users[p]]
        target = [p for p in range(used) if not self._users[p]]
        copy_pages(self.pool, source, target)
        move = dict(zip(source, target))
        for s, t in move.items():
            self._users[t], self._users[s] = self._users[s], 0
        self._free = [p for p in range(len(self._users) - 1, -1, -1) if not self._users[p]]
        changed = [s for s, row in enumerate(self._pages) if any(p in move for p in row)]
        for s in changed:
            self._pages[s] = [move.get(p, p) for p in self._pages[s]]
        self._publish(changed)
        return len(source)
