"""qg_kv_prefixes and qg_prefix_attention without a GPU: what they refuse, and the reads of a
buffer that holds anything (qg_prefix_index.h)."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from nebula_amd import qg
from test_spec_cpu import A, BAD_BATCH, BAD_CACHE, INVALID, batch, cache, ref

ROOT = Path(__file__).resolve().parent.parent
N = 1 << 40


@pytest.fixture(scope="module")
def lib():
    return qg.lib()


def attend(lib, c, b, out=20 * A, q=21 * A, heads=4, scale=1.0, layer=0, prefixes=23 * A, pn=1 << 20, ws=1 << 32, n=N):
    return lib.qg_prefix_attention(out, q, heads, scale, ref(c), layer, ref(b), prefixes, pn, ws, n)


@pytest.mark.parametrize("c,b", [(kw, {}) for kw in BAD_CACHE] + [({}, kw) for kw in BAD_BATCH])
def test_refused_caches_and_batches(lib, c, b):
    c, b = cache(**c), batch(**b)
    assert lib.qg_kv_prefixes_bytes(ref(c), ref(b)) == 0
    assert lib.qg_prefix_attention_workspace_bytes(ref(c), ref(b), 4) == 0
    assert lib.qg_kv_prefixes(24 * A, 25 * A, ref(c), ref(b), 23 * A, N) == INVALID
    assert attend(lib, c, b) == INVALID


@pytest.mark.parametrize("kw", [
    dict(out=None), dict(q=None), dict(heads=3), dict(heads=0), dict(heads=258), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38),
    dict(layer=2), dict(layer=-1), dict(ws=None), dict(ws=(1 << 32) + 8), dict(out=20 * A + 4), dict(q=21 * A + 8), dict(q=20 * A), dict(q=20 * A + 64),
    dict(prefixes=None), dict(prefixes=23 * A + 4), dict(pn=16), dict(n=64), dict(out=23 * A), dict(prefixes=20 * A + 16), dict(ws=23 * A - 4096),
    dict(ws=21 * A - 64), dict(ws=20 * A)])
def test_refused_attention(lib, kw):
    assert attend(lib, cache(), batch(), **kw) == INVALID


def test_refused_searches(lib):
    c, b = cache(), batch()
    n = lib.qg_kv_prefixes_bytes(ref(c), ref(b))
    assert n % 4 == 0 and n > 4 * 9
    call = lib.qg_kv_prefixes
    for link, shared, p, size in ((24 * A, 25 * A, None, N), (24 * A, 25 * A, 23 * A + 8, N), (24 * A, 25 * A, 23 * A, n - 1), (24 * A + 2, 25 * A, 23 * A, n),
                                  (24 * A, 25 * A + 1, 23 * A, n), (24 * A, 24 * A + 8, 23 * A, n), (23 * A + 16, 25 * A, 23 * A, n), (24 * A, 23 * A + n - 4, 23 * A, n),
                                  (4 * A, 25 * A, 23 * A, n), (24 * A, 5 * A + 8, 23 * A, n), (6 * A + 12, 25 * A, 23 * A, n), (24 * A, 25 * A, 4 * A, n),
                                  (24 * A, 25 * A, 5 * A, n), (24 * A, 25 * A, 6 * A, n)):
        assert call(link, shared, ref(c), ref(b), p, size) == INVALID, (link, shared, p, size)


def test_least_saving(lib):
    """A thread's own setting."""
    import threading
    first = lib.qg_prefix_least_saving(5)
    assert first == 48 << 20 and lib.qg_prefix_least_saving(0) == 5 and lib.qg_prefix_least_saving(1 << 62) == 0
    seen = []
    t = threading.Thread(target=lambda: seen.append(lib.qg_prefix_least_saving(7)))
    t.start()
    t.join()
    assert seen == [48 << 20]
    assert lib.qg_prefix_least_saving(-1) == 1 << 60 and lib.qg_prefix_least_saving(-1) == 48 << 20


def test_workspaces(lib):
    c = cache(head_dim=128, sequences=64)
    sizes = [lib.qg_prefix_attention_workspace_bytes(ref(c), ref(batch(rows=r, max_rows=m, parent=None)), 16)
             for r, m in ((1, 1), (2, 1), (64, 1), (64, 64), (1000, 17), (1024, 1), (1025, 1), (5000, 9), (6000, 1), (65536, 1))]
    assert all(sizes) and sizes == sorted(sizes)
    n = sizes[2]
    b = batch(rows=64, max_rows=1, parent=None)
    assert attend(lib, c, b, heads=16, n=n - 1) == INVALID
    assert lib.qg_prefix_attention_workspace_bytes(ref(cache(kv_heads=128)), ref(batch(rows=65536, max_rows=9)), 1024) == 0


HARNESS = r"""
#include "qg_prefix_index.h"
extern "C" int inside(int *v, int sequences, int table_pages, int shift, int rows, int max_rows) {
    KvView c{};
    BatchView b{nullptr, nullptr, rows, max_rows};
    c.sequences = sequences; c.table_pages = table_pages; c.shift = shift;
    const Segment s = segment_inside(c, b, Segment{v[0], v[1], v[2], v[3], v[4], v[5], v[6], 0});
    v[0] = s.owner; v[1] = s.begin; v[2] = s.end; v[3] = s.row0; v[4] = s.rows; v[5] = s.up;
    PrefixView p{};
    p.head = v + 7;
    return segment_count(c, p);
}
extern "C" int place(const int *p, int heads, int h, int x, int all, long *at) {
    return segment_place(SegmentParts{p[0], p[1], p[2], p[3]}, heads, h, x, all, at[0], at[1]);
}
extern "C" long bytes(int S, int rows) {
    int *p = nullptr;
    const PrefixView v = prefix_view(p, S, rows);
    return (char *)(v.row_of + rows) - (char *)p == (long)prefix_bytes(S, rows) ? (long)prefix_bytes(S, rows) : -1;
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("prefix_index")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", f"-I{ROOT / 'nebula_amd' / 'csrc'}", str(d / "h.cpp"), "-o", str(d / "h.so")], check=True)
    lib = C.CDLL(str(d / "h.so"))
    lib.bytes.restype = C.c_long
    return lib


def test_buffers_of_any_content_stay_inside(index, lib):
    rng = np.random.default_rng(0)
    wild = np.array([0, 1, -1, -2, 2 ** 31 - 1, -2 ** 31, 2 ** 30, 31, 32, 33, 100, 2 ** 28], np.int32)
    for _ in range(5000):
        S, width, shift, rows, most = int(rng.integers(1, 1025)), int(rng.integers(1, 200)), int(rng.integers(3, 11)), int(rng.integers(1, 5000)), int(rng.integers(1, 65))
        v = np.where(rng.random(8) < 0.5, rng.integers(-5, 3000, 8), rng.choice(wild, 8)).astype(np.int32)
        count = index.inside(v.ctypes.data_as(C.c_void_p), S, width, shift, rows, most)
        owner, begin, end, row0, n, up = (int(x) for x in v[:6])
        assert 0 <= count <= 2 * S and 0 <= owner < S and -1 <= up < 2 * S
        assert 0 <= begin <= end <= (width << shift) + most and begin % 32 == 0
        assert 0 <= row0 and 0 <= n and row0 + n <= rows
        p = np.where(rng.random(4) < 0.6, rng.integers(-1, 20, 4), rng.choice(wild, 4)).astype(np.int32)
        heads, tiles, x = int(rng.integers(1, 129)), int(rng.integers(1, 1 << 27)), int(rng.integers(0, 1 << 23))
        h, at = int(rng.integers(0, heads)), (C.c_long * 2)()
        if rng.random() < 0.5:
            x %= 200
        if index.place(p.ctypes.data_as(C.c_void_p), heads, h, x, tiles, at):
            slot, step = at
            assert slot >= 0 and step > 0 and slot + (int(p[1]) - 1) * step < 16 * tiles
            assert slot == 16 * (int(p[0]) + (h * int(p[2]) + x // (16 * int(p[3]))) * int(p[3])) + x % (16 * int(p[3]))
            assert step == heads * int(p[2]) * int(p[3]) * 16
    for S, rows in ((1, 1), (3, 9), (1024, 65536)):
        assert index.bytes(S, rows) == lib.qg_kv_prefixes_bytes(ref(cache(sequences=S)), ref(batch(rows=rows, max_rows=1)))
