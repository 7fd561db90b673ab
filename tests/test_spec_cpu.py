"""The speculative-step entry points without a GPU: what they refuse (before any
device call), and the index arithmetic of qg_kv_index.h on tables, lengths, row
starts and parents that hold anything."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from nebula_amd import qg

ROOT = Path(__file__).resolve().parent.parent
INVALID = 1  # hipErrorInvalidValue
A = 1 << 20   # a well-aligned address that is never read


def cache(**kw):
    d = dict(k=A, v=2 * A, type=1, layers=2, pages=10, kv_heads=2, page_tokens=16, head_dim=64, refs=3 * A, table=4 * A, length=5 * A,
             sequences=3, table_pages=4)
    return qg.KvCache(**(d | kw))


def batch(**kw):
    return qg.KvBatch(**(dict(rows=9, max_rows=5, start=6 * A, parent=7 * A) | kw))


def rows(**kw):
    d = dict(q=8 * A, k=9 * A, v=10 * A, q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, rows=9, q_heads=4, kv_heads=2,
             head_dim=64, q_norm=11 * A, k_norm=12 * A, eps=1e-6, rope_dims=64, freq=13 * A)
    return qg.QkRows(**(d | kw))


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=A + 8), dict(table=None), dict(length=None), dict(table=A + 2), dict(type=2), dict(type=-1),
             dict(layers=0), dict(pages=0), dict(kv_heads=0), dict(kv_heads=129), dict(page_tokens=12), dict(page_tokens=4), dict(page_tokens=2048),
             dict(head_dim=96), dict(head_dim=0), dict(sequences=0), dict(sequences=1025), dict(table_pages=0),
             dict(table_pages=1 << 25), dict(layers=1 << 30, pages=1 << 30)]
BAD_BATCH = [dict(start=None), dict(start=A + 1), dict(rows=0), dict(rows=1 << 17), dict(max_rows=0), dict(max_rows=10), dict(rows=100, max_rows=65),
             dict(parent=A + 2)]


def ref(x):
    return C.byref(x) if x is not None else None


@pytest.fixture(scope="module")
def lib():
    return qg.lib()


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_refused_caches(lib, kw):
    c, b = cache(**kw), batch()
    assert lib.qg_kv_workspace_bytes(ref(c)) == 0
    assert lib.qg_tree_attention_workspace_bytes(ref(c), ref(b), 4) == 0
    assert lib.qg_tree_attention(20 * A, 21 * A, 4, 1.0, ref(c), 0, ref(b), 22 * A, 1 << 30) == INVALID
    assert lib.qg_qk_norm_rope(20 * A, None, ref(rows()), ref(c), 0, ref(b)) == INVALID
    assert lib.qg_kv_reserve(ref(c), ref(b), A, 22 * A, 1 << 30) == INVALID
    assert lib.qg_kv_fork(ref(c), A, A, 1, 22 * A, 1 << 30) == INVALID
    assert lib.qg_kv_truncate(ref(c), None) == INVALID
    assert lib.qg_kv_compact(ref(c), ref(b), A, A, 23 * A) == INVALID
    assert lib.qg_kv_copy_pages(ref(c), A, A, 1) == INVALID


@pytest.mark.parametrize("kw", BAD_BATCH)
def test_refused_batches(lib, kw):
    c, b = cache(), batch(**kw)
    assert lib.qg_tree_attention_workspace_bytes(ref(c), ref(b), 4) == 0
    assert lib.qg_tree_attention(20 * A, 21 * A, 4, 1.0, ref(c), 0, ref(b), 22 * A, 1 << 30) == INVALID
    assert lib.qg_qk_norm_rope(20 * A, None, ref(rows(rows=max(b.rows, 1))), ref(c), 0, ref(b)) == INVALID
    assert lib.qg_kv_reserve(ref(c), ref(b), A, 22 * A, 1 << 30) == INVALID
    assert lib.qg_kv_compact(ref(c), ref(b), A, A, 23 * A) == INVALID
    assert lib.qg_verify_drafts(A, A, A, A, A, A, A, A, 100, 3, ref(b), 22 * A, 1 << 30) == INVALID


@pytest.mark.parametrize("args", [
    (None, 21 * A, 4, 1.0, 0, 22 * A), (20 * A, None, 4, 1.0, 0, 22 * A), (20 * A, 21 * A, 3, 1.0, 0, 22 * A), (20 * A, 21 * A, 0, 1.0, 0, 22 * A),
    (20 * A, 21 * A, 258, 1.0, 0, 22 * A), (20 * A, 21 * A, 4, float("nan"), 0, 22 * A), (20 * A, 21 * A, 4, float("inf"), 0, 22 * A),
    (20 * A, 21 * A, 4, 1.0, 2, 22 * A), (20 * A, 21 * A, 4, 1.0, -1, 22 * A), (20 * A, 21 * A, 4, 1.0, 0, None), (20 * A + 4, 21 * A, 4, 1.0, 0, 22 * A),
    (20 * A, 21 * A + 8, 4, 1.0, 0, 22 * A), (20 * A, 20 * A, 4, 1.0, 0, 22 * A), (20 * A, 20 * A + 64, 4, 1.0, 0, 22 * A),
    (20 * A, 21 * A, 4, 1.0, 0, 21 * A), (20 * A, 21 * A, 4, 1.0, 0, 22 * A + 4)])
def test_refused_attention(lib, args):
    out, q, heads, scale, layer, ws = args
    c, b = cache(), batch()
    assert lib.qg_tree_attention(out, q, heads, scale, ref(c), layer, ref(b), ws, 1 << 30) == INVALID


def test_refused_workspaces(lib):
    c, b = cache(), batch()
    n = lib.qg_tree_attention_workspace_bytes(ref(c), ref(b), 4)
    assert n and lib.qg_tree_attention(20 * A, 21 * A, 4, 1.0, ref(c), 0, ref(b), 22 * A, n - 1) == INVALID
    n = lib.qg_kv_workspace_bytes(ref(c))
    assert n >= 4 * 3 * (4 + 2) and lib.qg_kv_fork(ref(c), A, A, 1, 22 * A, n - 1) == INVALID
    assert lib.qg_kv_reserve(ref(c), ref(b), A, 22 * A, n - 1) == INVALID
    n = lib.qg_softmax_workspace_bytes(3, 1000)
    assert n and lib.qg_softmax(A, 2 * A, 3, 1000, 1.0, 22 * A, n - 1) == INVALID
    n = lib.qg_verify_workspace_bytes(3, 1000)
    assert n and lib.qg_verify_drafts(A, A, A, A, A, A, A, A, 1000, 3, ref(b), 22 * A, n - 1) == INVALID
    # a workspace serves every batch of no more rows; too many rows x heads for one launch are refused
    sizes = [lib.qg_tree_attention_workspace_bytes(ref(cache(head_dim=128)), ref(batch(rows=64, max_rows=m)), 16) for m in range(1, 65)]
    assert len(set(sizes)) == 1
    assert all(0 < lib.qg_tree_attention_workspace_bytes(ref(c), ref(batch(rows=r, max_rows=1)), 4) <= n0
               for n0 in [lib.qg_tree_attention_workspace_bytes(ref(c), ref(batch(rows=40, max_rows=40, parent=None)), 4)] for r in range(1, 41))
    assert lib.qg_tree_attention_workspace_bytes(ref(c), ref(batch(rows=65536, max_rows=9)), 256) > 0
    assert lib.qg_tree_attention_workspace_bytes(ref(cache(kv_heads=128)), ref(batch(rows=65536, max_rows=9)), 1024) == 0
    for rows_, cols in ((0, 5), (5, 0), (65537, 5), (5, (1 << 24) + 1), (-1, -1), (4096, 1 << 24)):
        assert lib.qg_softmax_workspace_bytes(rows_, cols) == 0
    for seq, cols in ((0, 5), (1025, 5), (5, 0), (5, (1 << 24) + 1)):
        assert lib.qg_verify_workspace_bytes(seq, cols) == 0


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(k=None), dict(v=None), dict(rows=0), dict(rows=8), dict(head_dim=128), dict(head_dim=63), dict(q_heads=0), dict(kv_heads=3),
    dict(rope_dims=63), dict(rope_dims=4), dict(rope_dims=72), dict(rope_dims=-8), dict(freq=None), dict(freq=A + 4), dict(eps=-1.0),
    dict(eps=float("nan")), dict(q_row=258), dict(q_head=-64), dict(k_row=1 << 50), dict(q=8 * A + 4), dict(q_norm=A + 4), dict(position=A + 2)])
def test_refused_rows(lib, kw):
    c, b = cache(), batch()
    assert lib.qg_qk_norm_rope(20 * A, 21 * A, ref(rows(**kw)), ref(c), 0, ref(b)) == INVALID


def test_refused_rope_calls(lib):
    c, b, r = cache(), batch(), rows()
    call = lib.qg_qk_norm_rope
    assert call(None, None, ref(r), ref(c), 0, ref(b)) == INVALID
    assert call(20 * A, None, None, ref(c), 0, ref(b)) == INVALID
    assert call(20 * A, None, ref(r), ref(c), 2, ref(b)) == INVALID
    assert call(20 * A, None, ref(r), ref(c), 0, None) == INVALID
    assert call(20 * A, None, ref(r), None, 0, ref(b)) == INVALID      # a batch without its cache
    assert call(20 * A, None, ref(r), None, 0, None) == INVALID         # a rotation without positions
    # outputs over inputs: q_out in another layout's place, over k or v, over k_out
    for q_out, k_out, kw in ((8 * A, None, dict(q_row=512)), (8 * A + 256, None, {}), (9 * A, None, {}), (10 * A, None, {}), (20 * A, 20 * A + 1024, {}),
                             (20 * A, 8 * A, {}), (20 * A, 9 * A, dict(k_head=128, k_row=256)), (20 * A, 10 * A + 512, {})):
        assert call(q_out, k_out, ref(rows(**kw)), ref(c), 0, ref(b)) == INVALID, (q_out, k_out, kw)


def test_refused_calls(lib):
    c, b = cache(), batch()
    W, N = 22 * A, 1 << 30
    for args in ((None, 2 * A, 3, 100, 1.0, W, N), (A, None, 3, 100, 1.0, W, N), (A, 2 * A, 3, 100, -1.0, W, N), (A, 2 * A, 3, 100, float("nan"), W, N),
                 (A, 2 * A, 3, 100, float("inf"), W, N), (A, 2 * A, 3, 100, 1.0, None, N), (A, A + 4, 3, 100, 1.0, W, N), (A + 2, 2 * A, 3, 100, 1.0, W, N),
                 (A, 2 * A, 0, 100, 1.0, W, N), (A, 2 * A, 3, 100, 1.0, W + 4, N)):
        assert lib.qg_softmax(*args) == INVALID, args
    good = [A, 2 * A, 3 * A, 4 * A, 5 * A, 6 * A, 7 * A, 8 * A, 100, 3, ref(b), W, N]
    for i, bad in ((0, None), (1, None), (2, None), (3, None), (5, None), (6, None), (7, None), (3, A + 2), (4, A + 1), (8, 0), (9, 0), (9, 1025), (10, None),
                   (11, None), (11, W + 8)):
        args = list(good)
        args[i] = bad
        assert lib.qg_verify_drafts(*args) == INVALID, (i, bad)
    for args in ((None, A, 1, W, N), (A, None, 1, W, N), (A, A, 0, W, N), (A, A, 4, W, N), (A, A, 1, None, N), (A + 2, A, 1, W, N)):
        assert lib.qg_kv_fork(ref(c), *args) == INVALID
    for args in ((None, W, N), (A, None, N), (A + 1, W, N)):
        assert lib.qg_kv_reserve(ref(c), ref(b), *args) == INVALID
    for args in ((None, A, 23 * A), (A, None, 23 * A), (A, A, None), (A, A, 23 * A + 2), (A, A, 5 * A + 4)):
        assert lib.qg_kv_compact(ref(c), ref(b), *args) == INVALID
    for args in ((None, A, 1), (A, None, 1), (A, A, 0), (A, A, 4097), (A + 2, A, 1)):
        assert lib.qg_kv_copy_pages(ref(c), *args) == INVALID
    no_refs = cache(refs=None)
    assert lib.qg_kv_truncate(ref(no_refs), None) == INVALID and lib.qg_kv_reserve(ref(no_refs), ref(b), A, W, N) == INVALID
    assert lib.qg_kv_truncate(ref(c), A + 2) == INVALID


def test_refused_overlaps(lib):
    """Arrays that a call reads in one workgroup and writes in another, and sizes past an index."""
    c, b = cache(), batch()
    W, N = 60 * A, 1 << 30
    assert lib.qg_kv_truncate(ref(c), c.length + 4) == INVALID and lib.qg_kv_truncate(ref(c), c.length - 8) == INVALID
    good = [30 * A, 31 * A, 32 * A, 33 * A, 34 * A, 35 * A, 36 * A, 37 * A, 100, 3, ref(b), W, N]
    for i, bad in ((0, 31 * A), (0, 31 * A + 4), (0, 32 * A), (1, 32 * A - 4), (0, 33 * A), (1, 34 * A + 16), (2, 33 * A + 8), (0, W), (1, W + 64), (2, W + 4),
                   (3, W), (4, W + 4)):
        args = list(good)
        args[i] = bad
        assert lib.qg_verify_drafts(*args) == INVALID, (i, bad)
    huge = cache(layers=65537)
    assert lib.qg_tree_attention_workspace_bytes(ref(huge), ref(b), 4) == 0 and lib.qg_kv_copy_pages(ref(huge), A, A, 1) == INVALID
    assert lib.qg_tree_attention(20 * A, 21 * A, 4, 3e38, ref(c), 0, ref(b), 22 * A, 1 << 30) == INVALID


HARNESS = r"""
#include "qg_kv_index.h"
extern "C" int page(const int *table, int pages, int shift, int sequences, int table_pages, const int *length, int s, int t, int *len, long long *at) {
    KvView c{};
    c.table = (int *)table; c.length = (int *)length; c.pages = pages; c.shift = shift; c.sequences = sequences; c.table_pages = table_pages;
    c.layers = 3; c.heads = 5; c.dim = 64;
    *len = kv_length(c, s);
    const int p = kv_page(c, s, t);
    *at = p < 0 ? -1 : (long long)kv_at(c, 2, p, 4, t & ((1 << shift) - 1));
    return p;
}
extern "C" void rows(const int *start, int total, int most, int s, int *first, int *n) {
    BatchView b{start, nullptr, total, most};
    batch_rows(b, s, *first, *n);
}
extern "C" int parent(int p, int i) { return tree_parent(p, i); }
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_index")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", f"-I{ROOT / 'nebula_amd' / 'csrc'}", str(d / "h.cpp"), "-o", str(d / "h.so")], check=True)
    return C.CDLL(str(d / "h.so"))


def test_index_arithmetic_stays_inside(index):
    rng = np.random.default_rng(0)
    wild = np.array([0, 1, -1, -2, 2 ** 31 - 1, -2 ** 31, 2 ** 30, 7, 100], np.int32)
    n, first, count, at = C.c_int(), C.c_int(), C.c_int(), C.c_longlong()
    for _ in range(3000):
        shift, pages, B, width = int(rng.integers(3, 11)), int(rng.integers(1, 9)), 4, int(rng.integers(1, 6))
        table = np.where(rng.random((B, width)) < 0.6, rng.integers(0, pages, (B, width)), rng.choice(wild, (B, width))).astype(np.int32)
        length = np.where(rng.random(B) < 0.5, rng.integers(0, width << shift, B), rng.choice(wild, B)).astype(np.int32)
        s = int(rng.integers(0, B))
        t = int(rng.choice([rng.integers(0, width << shift), rng.choice(wild), (width << shift) - 1, width << shift]))
        p = index.page(table.ctypes.data_as(C.c_void_p), pages, shift, B, width, length.ctypes.data_as(C.c_void_p), s, t, C.byref(n), C.byref(at))
        inside = 0 <= t < width << shift
        want = int(table[s, t >> shift]) if inside and 0 <= table[s, t >> shift] < pages else -1
        assert p == want
        assert n.value == min(max(int(length[s]), 0), width << shift)
        if p >= 0:
            assert at.value == (((2 * pages + p) * 5 + 4) * (1 << shift) + t % (1 << shift)) * 64
            assert at.value + 64 <= 3 * pages * 5 * (1 << shift) * 64
        total, most = int(rng.integers(1, 50)), int(rng.integers(1, 50))
        start = np.where(rng.random(B + 1) < 0.6, np.sort(rng.integers(0, total + 1, B + 1)), rng.choice(wild, B + 1)).astype(np.int32)
        index.rows(start.ctypes.data_as(C.c_void_p), total, most, s, C.byref(first), C.byref(count))
        assert 0 <= first.value <= total and 0 <= count.value <= most and first.value + count.value <= total
        i, q = int(rng.integers(0, 64)), int(rng.choice(np.concatenate([wild, rng.integers(-2, 70, 4).astype(np.int32)])))
        assert index.parent(q, i) == (q if 0 <= q < i else -1)


OWN = r"""
#include "qg_kv_index.h"
extern "C" int shared(const int *table, int *refs, int pages, int t) {
    KvView c{};
    c.table = (int *)table; c.refs = refs; c.pages = pages; c.shift = 3; c.sequences = 1; c.table_pages = 4;
    return kv_shared(c, kv_page(c, 0, t));
}
"""


def test_pages_that_may_be_written(tmp_path):
    """A page that another table entry holds too is shared; without counts none is, and no page is none."""
    (tmp_path / "h.cpp").write_text(OWN)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", f"-I{ROOT / 'nebula_amd' / 'csrc'}", str(tmp_path / "h.cpp"), "-o", str(tmp_path / "h.so")], check=True)
    shared = C.CDLL(str(tmp_path / "h.so")).shared
    table, refs = (C.c_int * 4)(2, 0, -1, 7), (C.c_int * 3)(2, 0, 1)
    assert [shared(table, refs, 3, t) for t in (0, 7, 8, 16, 24, 32, -1)] == [0, 0, 1, 0, 0, 0, 0]
    assert [shared(table, None, 3, t) for t in (0, 7, 8, 16, 24, 32, -1)] == [0] * 7


def test_refused_temperatures(lib):
    for t in (1e-40, 2.0 ** -127, -0.5, float("-inf")):
        assert lib.qg_softmax(A, 2 * A, 3, 100, t, 22 * A, 1 << 30) == INVALID, t


def test_refused_overlaps_of_page_calls(lib):
    """What a page call writes and what its other workgroups read, cache arrays among it; sizes of the caches above:
    3 sequences, tables of 4 entries, 10 pages."""
    c, b = cache(), batch()
    W, N = 60 * A, lib.qg_kv_workspace_bytes(ref(c))
    path, count, out = 30 * A, 31 * A, 32 * A
    for new in (path, path + 4 * 14, count, count + 8, count - 8, b.start, b.start + 12, c.table + 44, c.table - 8, c.refs + 36, c.length + 8, c.length - 8):
        assert lib.qg_kv_compact(ref(c), ref(b), path, count, new) == INVALID, hex(new)
    for own in (dict(count=c.length), dict(path=c.length - 4), dict(start=c.length + 4)):   # the cache's lengths as the new ones
        p, n, starts = own.get("path", path), own.get("count", count), own.get("start", b.start)
        assert lib.qg_kv_compact(ref(c), ref(batch(start=starts)), p, n, c.length) == INVALID, own
    for new in (c.table + 44, c.table - 8, c.refs, c.refs + 36):
        assert lib.qg_kv_truncate(ref(c), new) == INVALID, hex(new)
    for status, ws in ((W, W), (W + N - 4, W), (c.length, W), (c.table + 44, W), (c.refs + 36, W), (b.start + 12, W), (out, c.length - N + 4), (out, c.table),
                       (out, c.refs + 36), (out, b.start + 12)):
        assert lib.qg_kv_reserve(ref(c), ref(b), status, ws, N) == INVALID, (hex(status), hex(ws))
    for dst, src, n, ws in ((c.length, path, 1, W), (path, c.length + 8, 1, W), (c.table + 40, path, 2, W), (path, c.refs + 32, 3, W), (W + 4, path, 1, W),
                            (path, W + N - 4, 1, W), (path, count, 1, c.length - 4), (path, count, 1, c.table + 44), (path, count, 1, c.refs)):
        assert lib.qg_kv_fork(ref(c), dst, src, n, ws, N) == INVALID, (hex(dst), hex(src))


def test_refused_overlaps_of_verification(lib):
    """Outputs over what the last kernel reads, the workspace over any input."""
    b, W = batch(), 60 * A
    N = lib.qg_verify_workspace_bytes(3, 100)
    good = [30 * A, 31 * A, 32 * A, 33 * A, 34 * A, 35 * A, 36 * A, 37 * A, 100, 3, ref(b), W, N]
    for i, bad in ((0, 37 * A), (1, 37 * A + 8), (2, 37 * A - 8), (0, b.start), (1, b.start + 12), (2, b.start - 8), (5, W), (6, W + N - 4), (7, W + 16)):
        args = list(good)
        args[i] = bad
        assert lib.qg_verify_drafts(*args) == INVALID, (i, hex(bad))
    for kw in (dict(start=W), dict(parent=W + N - 4)):
        args = list(good)
        args[10] = ref(batch(**kw))
        assert lib.qg_verify_drafts(*args) == INVALID, kw


@pytest.mark.parametrize("cols", [1, 4096, 4097, 40960, 40961, 50000, 131072, 135168, 135169, 151936, 300001, 1 << 24])
def test_workspaces_serve_smaller_batches(lib, cols):
    """A workspace for the largest batch is enough for every smaller one, and none is smaller than what a call of that
    size lays out in it."""
    rows = [lib.qg_softmax_workspace_bytes(r, cols) for r in range(1, 1200)]
    assert rows == sorted(rows) and rows[0] > 0
    seqs = [lib.qg_verify_workspace_bytes(s, cols) for s in range(1, 1025)]
    assert seqs == sorted(seqs)
    blocks = -(-cols // 4096)
    for s, n in enumerate(seqs, 1):
        pieces = -(-blocks // -(-blocks * s // 2048))
        assert n >= 2 * s * (8 * pieces + 48) + s * 64 * 20, (s, n)
    for r, n in enumerate(rows, 1):
        if cols > 135168 or (cols > 40960 and r * cols < 13000000):
            assert n >= 16 * r * -(-cols // 4096), (r, n)


def test_refused_page_counts(lib):
    """Page numbers are marked as -2 - page and counted 16384 at a time: both stay inside an int up to 2^30 pages."""
    small = dict(layers=1, kv_heads=1, page_tokens=8)
    assert lib.qg_kv_workspace_bytes(ref(cache(pages=1 << 30, **small))) == 4 * (2 + 2 * 3 + (1 << 30))
    for pages in ((1 << 30) + 1, 2 ** 31 - 1):
        c = cache(pages=pages, **small)
        assert lib.qg_kv_workspace_bytes(ref(c)) == 0
        assert lib.qg_kv_reserve(ref(c), ref(batch()), 30 * A, 60 * A, 1 << 40) == INVALID
