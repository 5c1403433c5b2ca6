"""Argument checks of the operators of drafted decoding, on the CPU: every mismatch is refused before a pointer reaches a
kernel (shape, dtype and layout first, then the device), and launches go to the tensors' GPU."""

import contextlib
import ctypes

import pytest
import torch

from reskv_amd import _lib, drafts, int4, packed
from reskv_amd.drafts import draft_tree, verify_drafts
from reskv_amd.int4 import empty_pages, int4_append_rope, int4_keep, int4_tree_attention

f16, f32, i32 = dict(dtype=torch.float16), dict(dtype=torch.float32), dict(dtype=torch.int32)


def ints(*x):
    return torch.tensor(x, **i32)


def pool():
    return empty_pages(3, 2, 64, device="cpu")


def append(**changes):
    kw = dict(pages=pool(), table=torch.zeros(2, 2, **i32), starts=ints(0, 5), q=torch.zeros(6, 4, 128, **f16),
              k=torch.zeros(6, 2, 128, **f16), v=torch.zeros(6, 2, 128, **f16), cos=torch.zeros(9, 64), sin=torch.zeros(9, 64),
              offsets=ints(0, 2, 6))
    return int4_append_rope(**{**kw, **changes})


@pytest.mark.parametrize("changes,match", [
    (dict(pages=torch.zeros(3, 2, 60 * 160, dtype=torch.uint8)), "positive multiple of 32 tokens"),
    (dict(table=torch.zeros(2, 2)), "table must be a contiguous int32 matrix"),
    (dict(starts=ints(0)), "starts has 1 entries, expected 2"),
    (dict(k=torch.zeros(6, 1, 128, **f16)), "k has 1 heads, expected 2"),
    (dict(v=torch.zeros(6, 2, 64, **f16)), "v must be fp16"),
    (dict(v=torch.zeros(5, 2, 128, **f16)), "k and v must have the same number of rows"),
    (dict(q=torch.zeros(6, 4, 128)), "q must be fp16"),
    (dict(q=torch.zeros(5, 4, 128, **f16)), "q and k must have the same number of rows"),
    (dict(q=torch.zeros(6, 3, 128, **f16)), "multiple of the KV heads"),
    (dict(q=torch.zeros(6, 0, 128, **f16)), "multiple of the KV heads"),
    (dict(offsets=None), "one row for every sequence"),
    (dict(offsets=ints(0, 6)), "offsets has 2 entries, expected 3"),
    (dict(positions=ints(0, 1)), "positions has 2 entries, expected 6"),
    (dict(positions=torch.zeros(6, dtype=torch.int64)), "positions must be a contiguous int32 vector"),
    (dict(cos=torch.zeros(9, 64, **f16)), "cos must be a contiguous fp32 matrix"),
    (dict(sin=torch.zeros(64, 9).t()), "sin must be a contiguous fp32 matrix"),
    (dict(sin=torch.zeros(8, 64)), "the same shape"),
    (dict(cos=torch.zeros(0, 64), sin=torch.zeros(0, 64)), "a row for every position"),
    (dict(cos=torch.zeros(9, 60), sin=torch.zeros(9, 60)), "multiple of 16, up to 128"),
    (dict(cos=torch.zeros(9, 72), sin=torch.zeros(9, 72)), "multiple of 16, up to 128"),
    (dict(cos=torch.zeros(9, 0), sin=torch.zeros(9, 0)), "multiple of 16, up to 128"),
    (dict(out=torch.zeros(6, 2, 128, **f16)), "out has 2 heads, expected 4"),
    (dict(out=torch.zeros(4, 6, 128, **f16).transpose(0, 1)), "out must be contiguous"),
    (dict(q=None, out=torch.zeros(6, 4, 128, **f16)), "out is for the queries"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_append_rope_checks(changes, match):
    with pytest.raises(RuntimeError, match=match):
        append(**changes)


def attend(**changes):
    kw = dict(q=torch.zeros(6, 4, 128, **f16), pages=pool(), table=torch.zeros(2, 2, **i32), lengths=ints(5, 9),
              offsets=ints(0, 2, 6), seen=torch.zeros(6, dtype=torch.int64))
    return int4_tree_attention(**{**kw, **changes})


@pytest.mark.parametrize("changes,match", [
    (dict(q=torch.zeros(6, 4, 64, **f16)), "q must be fp16"),
    (dict(q=torch.zeros(6, 3, 128, **f16)), "multiple of the KV heads"),
    (dict(lengths=ints(1, 2, 3)), "lengths has 3 entries, expected 2"),
    (dict(offsets=ints(0, 6)), "offsets has 2 entries, expected 3"),
    (dict(seen=torch.zeros(6, **i32)), "a mask for every row of q"),
    (dict(seen=torch.zeros(5, dtype=torch.int64)), "a mask for every row of q"),
    (dict(seen=torch.zeros(12, dtype=torch.int64)[::2]), "a mask for every row of q"),
    (dict(scaling=0.0), "scaling must be positive"),
    (dict(scaling=-1.0), "scaling must be positive"),
    (dict(scaling=float("nan")), "scaling must be positive"),
    (dict(max_length=-1), "max_length must not be negative"),
    (dict(max_nodes=0), r"max_nodes must be in 1 \.\. 64"),
    (dict(max_nodes=65), r"max_nodes must be in 1 \.\. 64"),
    (dict(out=torch.zeros(5, 4, 128, **f16)), "shaped like q"),
    (dict(table=torch.zeros(2, 0, **i32)), "table must be"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_tree_attention_checks(changes, match):
    with pytest.raises(RuntimeError, match=match):
        attend(**changes)


def verify(**changes):
    kw = dict(logits=torch.zeros(6, 50, **f16), tokens=torch.zeros(6, dtype=torch.int64), parents=torch.zeros(6, **i32),
              offsets=ints(0, 2, 6), accept=torch.zeros(6), sample=torch.zeros(2))
    return verify_drafts(**{**kw, **changes})


@pytest.mark.parametrize("changes,match", [
    (dict(logits=torch.zeros(6, 50, dtype=torch.bfloat16)), "logits must be a matrix of float16 or float32"),
    (dict(logits=torch.zeros(6, 5, 10)), "logits must be a matrix"),
    (dict(logits=torch.zeros(50, 6).t()), "logits must have contiguous rows"),
    (dict(logits=torch.zeros(1, 50).expand(6, 50)), "logits must have contiguous rows"),
    (dict(logits=torch.zeros(6, 0)), "a column for every token"),
    (dict(tokens=torch.zeros(6, **i32)), "tokens must be a contiguous int64 vector"),
    (dict(tokens=torch.zeros(5, dtype=torch.int64)), "a token for every row"),
    (dict(parents=torch.zeros(5, **i32)), "parents has 5 entries, expected 6"),
    (dict(offsets=ints(0)), "at least one sequence"),
    (dict(accept=None), "accept must be a contiguous fp32 vector of 6"),
    (dict(accept=torch.zeros(6, dtype=torch.float64)), "accept must be"),
    (dict(sample=torch.zeros(6)), "sample must be a contiguous fp32 vector of 2"),
    (dict(draft=torch.zeros(6, 50, **f16)), "draft must be a matrix of float32"),
    (dict(draft=torch.zeros(6, 49)), r"draft must be \[6, 50\]"),
    (dict(draft=torch.zeros(1, 50).expand(6, 50)), "draft must have contiguous rows"),
    (dict(temperature=-0.5), "temperature must be finite and not negative"),
    (dict(temperature=1e-31), "must be 1e-30 or more"),
    (dict(temperature=float("inf")), "temperature must be finite and not negative"),
    (dict(temperature=float("nan")), "temperature must be finite and not negative"),
    (dict(), "every tensor must be a CUDA tensor"),
    (dict(temperature=0.0, accept=None, sample=None), "every tensor must be a CUDA tensor"),
])
def test_verify_checks(changes, match):
    with pytest.raises(RuntimeError, match=match):
        verify(**changes)


@pytest.mark.parametrize("changes,match", [
    (dict(pages=torch.zeros(3, 2, 60 * 160, dtype=torch.uint8)), "positive multiple of 32 tokens"),
    (dict(pages=torch.zeros(2, 3, 2, 64 * 160)), "pages must be a contiguous uint8 tensor"),
    (dict(starts=ints(1)), "starts has 1 entries, expected 2"),
    (dict(counts=torch.zeros(2)), "counts must be a contiguous int32 vector"),
    (dict(path=torch.zeros(2, 65, **i32)), "up to 64"),
    (dict(path=torch.zeros(3, 8, **i32)), "path must be a contiguous int32 matrix"),
    (dict(path=torch.zeros(8, 2, **i32).t()), "path must be a contiguous int32 matrix"),
    (dict(), "every tensor must be a CUDA tensor"),
])
def test_keep_checks(changes, match):
    kw = dict(pages=pool(), table=torch.zeros(2, 2, **i32), starts=ints(0, 5), path=torch.zeros(2, 8, **i32), counts=ints(1, 2))
    with pytest.raises(RuntimeError, match=match):
        int4_keep(**{**kw, **changes})


@pytest.mark.parametrize("args,match", [
    ((torch.zeros(4), ints(0, 4)), "parents must be a contiguous int32 vector"),
    ((ints(-1, 0), ints(0)), "at least one sequence"),
    ((ints(-1, 0), ints(0, 2), ints(1, 2)), "starts has 2 entries, expected 1"),
    ((ints(-1, 0), ints(0, 2)), "every tensor must be a CUDA tensor"),
])
def test_tree_checks(args, match):
    with pytest.raises(RuntimeError, match=match):
        draft_tree(*args)


def err(status):
    assert status != 0
    return _lib.lib().reskv_last_error().decode()


def test_the_library_refuses_by_name():
    """The C entry points' own checks; nothing is launched."""
    lib, p, odd = _lib.lib(), ctypes.c_void_p(16), ctypes.c_void_p(24)
    six = (ctypes.c_int64 * 6)(*([128] * 6))
    bad = (ctypes.c_int64 * 6)(128, 128, 128, 128, 132, 128)

    def rope(pages=p, positions=None, q=p, hq=4, k=p, n=2, strides=six, rows=9, rotary=128, s=2, offsets=None, page=64):
        return lib.reskv_int4_append_rope(pages, 3, page, 2, p, 2, s, p, offsets, positions, q, hq, k, p, n, strides, p, p, rows, rotary, 0, p,
                                          1, None)

    assert "null" in err(rope(pages=None)) and "null" in err(rope(k=None))
    assert "multiple of 32 tokens" in err(rope(page=40))
    assert "bad sizes" in err(rope(n=3)) and "bad sizes" in err(rope(s=0))
    assert "multiple of the KV heads" in err(rope(hq=3))
    assert "multiple of 16" in err(rope(rotary=24)) and "multiple of 16" in err(rope(rotary=144)) and "tables have rows" in err(rope(rows=0))
    assert "16-byte aligned" in err(rope(k=odd)) and "16-byte aligned" in err(rope(strides=bad)) and "16-byte aligned" in err(rope(q=odd))
    assert "too many rows or sequences" in err(rope(offsets=p, s=1 << 23, n=1 << 29))

    def tree(q=p, lengths=p, hq=4, n=4, scaling=1.0, most=100, nodes=64, work=p, nbytes=1 << 40, width=2, s=2):
        return lib.reskv_int4_tree_attention(q, p, 3, 64, p, width, lengths, p, None, s, n, hq, 2, scaling, most, nodes, 1, p, work, nbytes, None)

    assert "null" in err(tree(q=None)) and "null" in err(tree(lengths=None))
    assert "bad sizes" in err(tree(hq=5)) and "bad sizes" in err(tree(n=0))
    assert "1 to 64 nodes" in err(tree(nodes=65)) and "1 to 64 nodes" in err(tree(nodes=0))
    assert "must not be negative" in err(tree(most=-1))
    assert "scaling must be positive" in err(tree(scaling=0.0)) and "scaling must be positive" in err(tree(scaling=float("nan")))
    assert "16-byte aligned" in err(tree(q=odd))
    assert "workspace is too small" in err(tree(work=None)) and "workspace is too small" in err(tree(nbytes=100))
    assert "too many tokens" in err(tree(width=1 << 24, most=1 << 30, s=1 << 12))
    assert "too many tokens" in err(tree(n=1 << 29, hq=64))
    assert lib.reskv_int4_tree_workspace_bytes(2, 4, 5, 2, 100, 64) == 0
    assert lib.reskv_int4_tree_workspace_bytes(2, 4, 4, 2, 100, 64) > 0

    def check(logits=p, accept=p, draft=None, temperature=1.0, n=4, v=10, work=p, nbytes=1 << 40, stride=10):
        return lib.reskv_verify_drafts(logits, 0, stride, p, p, p, accept, p, draft, 10, temperature, 2, n, v, p, p, p, work, nbytes, None)

    assert "null" in err(check(logits=None)) and "null" in err(check(accept=None))
    assert "bad sizes" in err(check(n=0)) and "bad sizes" in err(check(v=0)) and "bad sizes" in err(check(v=1 << 30)) and "bad sizes" in err(check(n=1 << 24))
    assert "strides" in err(check(stride=-1))
    assert "temperature" in err(check(temperature=-1.0)) and "temperature" in err(check(temperature=float("nan")))
    assert "16-byte aligned" in err(check(logits=odd))
    assert "workspace is too small" in err(check(nbytes=10)) and "workspace is too small" in err(check(work=None))

    def keep(starts=p, layers=1, width=8, s=2, page=64):
        return lib.reskv_int4_keep(p, layers, 3, page, 2, p, 2, s, starts, p, width, p, None)

    assert "null" in err(keep(starts=None)) and "bad sizes" in err(keep(layers=0)) and "bad sizes" in err(keep(width=65))
    assert "bad sizes" in err(keep(layers=1 << 16)) and "too many sequences" in err(keep(s=1 << 24)) and "multiple of 32" in err(keep(page=33))
    assert "null" in err(lib.reskv_draft_tree(None, p, None, 1, 1, p, None, None))
    assert "bad sizes" in err(lib.reskv_draft_tree(p, p, None, 0, 1, p, None, None))


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
    sizes = (int4._tree_workspace, drafts._verify_workspace)
    for f in sizes:
        f.cache_clear()
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[-1], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(packed._lib, "lib", lambda: lib)
    for module in (int4, drafts):
        monkeypatch.setattr(module, "_same_gpu", lambda *t: 3)
    yield lib
    for f in sizes:
        f.cache_clear()


def test_every_launch_is_on_the_tensors_gpu(library):
    append()
    attend()
    verify()
    verify(temperature=0.0, accept=None, sample=None)
    int4_keep(pool(), torch.zeros(2, 2, **i32), ints(0, 5), torch.zeros(2, 8, **i32), ints(1, 2))
    draft_tree(ints(-1, 0), ints(0, 2))
    names = ["reskv_int4_append_rope", "reskv_int4_tree_attention", "reskv_verify_drafts", "reskv_verify_drafts", "reskv_int4_keep",
             "reskv_draft_tree"]
    assert library.calls == [(n, 3, 103) for n in names] and library.current == [0]


def test_nothing_to_do_launches_nothing(library):
    none = torch.zeros(0, 2, 128, **f16)
    assert append(q=torch.zeros(0, 4, 128, **f16), k=none, v=none, offsets=ints(0, 0, 0)).shape == (0, 4, 128)
    assert append(q=None, k=none, v=none, offsets=ints(0, 0, 0)) is None
    assert attend(q=torch.zeros(0, 4, 128, **f16), seen=None).shape == (0, 4, 128)
    path, counts, token = verify(logits=torch.zeros(0, 50), tokens=torch.zeros(0, dtype=torch.int64), parents=torch.zeros(0, **i32),
                                 accept=torch.zeros(0))
    assert (path == -1).all() and path.shape == (2, 64) and counts.tolist() == [0, 0] and token.tolist() == [-1, -1]
    int4_keep(pool(), torch.zeros(2, 2, **i32), ints(0, 5), torch.zeros(2, 0, **i32), ints(1, 2))
    assert draft_tree(torch.zeros(0, **i32), ints(0, 0))[0].shape == (0,)
    assert library.calls == []


def test_no_gradient_is_recorded(library):
    q = torch.zeros(6, 4, 128, **f16, requires_grad=True)
    assert not append(q=q).requires_grad and not attend(q=q).requires_grad
    wide = torch.zeros(6, 4, 256, **f16, requires_grad=True)[..., ::2]  # copied first
    assert not append(q=wide).requires_grad and not attend(q=wide).requires_grad
    verify(logits=torch.zeros(6, 50, requires_grad=True))


@pytest.mark.parametrize("rows", [1, 7, 33, 34, 100, 558, 1000, 5000])
def test_a_row_has_a_segment_for_every_lane_at_most(rows):
    """The walk of verify_drafts takes a row's segments one per lane of a wave: 64, whatever the vocabulary is.  The workspace
    holds 16 bytes per row and segment, 8 per sequence and segment, and 24 per sequence."""
    size = _lib.lib().reskv_verify_workspace_bytes
    around = [(64 << k) + i for k in range(10, 23) for i in range(-20, 21)] + [(1 << k) + i for k in range(21) for i in range(-9, 10)]
    for vocab in {v for v in around if v > 0} | set(range(1, 200000, 97)):
        segments = (size(3, rows, vocab) - 3 * 24) / (16 * rows + 3 * 8)
        assert segments == int(segments) and 1 <= segments <= 64, vocab


@pytest.mark.parametrize("sequences,rows,heads,per_head,refused", [
    (1 << 21, 4, 4, 2, True),        # few rows: 1024 threads for every four of them, or every sequence
    ((1 << 21) - 4, 4, 4, 2, False),
    (1 << 21, 2048, 4, 2, True),     # 1024 threads for every 16 rows
    (1 << 22, 257, 4, 4, True),
    (1 << 22, 8192, 4, 2, False),    # 256 threads
    (1 << 23, 8192, 4, 2, True),
])
def test_a_launch_of_the_merge_has_fewer_than_2_to_the_32_threads(sequences, rows, heads, per_head, refused):
    """Looked at before anything is launched; a workspace that is too small stops the calls that pass."""
    p = ctypes.c_void_p(16)
    said = err(_lib.lib().reskv_int4_tree_attention(p, p, 3, 64, p, 1, p, p, None, sequences, rows, heads, heads // per_head, 1.0, 64, 1, 1, p, p,
                                                    0, None))
    assert ("pass a launch's 2^32 threads" if refused else "workspace is too small") in said
