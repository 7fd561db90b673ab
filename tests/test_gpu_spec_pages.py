"""qg_kv_reserve / fork / truncate / compact / copy_pages against a model of the
same rules in Python: tables, holders, lengths and every byte of the pages."""
import ctypes as C
import sys

import numpy as np
import pytest

import spec_oracle as O
from nebula_amd import qg
from nebula_amd.qg import Device, call
from spec_oracle import BF16, F16, F32, Batch, Cache

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True, file=sys.stderr)


class Model:
    """The rules, one sequence and one page at a time, on the host copy of a cache."""

    def __init__(self, c):
        self.c = c

    def _let_go(self, p):
        if 0 <= p < self.c.pages:
            self.c.refs[p] -= 1

    def truncate(self, new=None):
        c = self.c
        for s in range(c.B):
            n = int(min(max(c.length[s], 0), c.width * c.P))
            n = n if new is None else min(n, max(int(new[s]), 0))
            for j in range(-(-n // c.P), c.width):
                self._let_go(c.table[s, j])
                c.table[s, j] = -1
            c.length[s] = n

    def fork(self, dst, src):
        c, table, length = self.c, self.c.table.copy(), self.c.length.copy()
        ok = [0 <= d < c.B and 0 <= s < c.B and d != s for d, s in zip(dst, src)]
        for i, (d, s) in enumerate(zip(dst, src)):
            if not ok[i] or any(ok[j] and dst[j] == d for j in range(i + 1, len(dst))):
                continue
            for p in c.table[d]:
                self._let_go(p)
            keep = -(-int(length[s]) // c.P)
            row = np.where((np.arange(c.width) < keep) & (table[s] >= 0) & (table[s] < c.pages), table[s], -1)
            for p in row[row >= 0]:
                c.refs[p] += 1
            c.table[d], c.length[d] = row, length[s]

    def reserve(self, counts):
        c = self.c
        status, need, copies = np.zeros(c.B, np.int32), [], []
        live = [s for s in range(c.B) if counts[s] and c.length[s] + counts[s] <= c.width * c.P]
        for s in range(c.B):
            if counts[s] and s not in live:
                status[s] = 2
        page = {s: c.page_of(s, int(c.length[s])) for s in live if c.length[s] % c.P}
        for s in live:
            L, here = int(c.length[s]), int(c.length[s]) // c.P
            for j in range(here, -(-(L + counts[s]) // c.P)):
                p = int(c.table[s, j])
                if not 0 <= p < c.pages:
                    need.append((s, j, -1))
                elif j == here and s in page:
                    same = [t for t in page if page[t] == p]
                    if c.refs[p] > 1 and (same[0] != s or len(same) < c.refs[p]):
                        need.append((s, j, p))
                elif c.refs[p] > 1:
                    need.append((s, j, p))
        free = [p for p in range(c.pages) if c.refs[p] == 0]
        if len(need) > len(free):
            status[live] = 1
            return status
        for (s, j, old), p in zip(need, free):
            if old >= 0:
                c.refs[old] -= 1
                if j == int(c.length[s]) // c.P and s in page:
                    copies.append((p, old))
            c.table[s, j] = p
            c.refs[p] = 1
        for p, old in copies:
            c.k[:, p], c.v[:, p] = c.k[:, old], c.v[:, old]
        return status

    def compact(self, batch, path, count):
        c, new = self.c, c_length(self.c)
        for s in range(c.B):
            n, L = int(batch.start[s + 1] - batch.start[s]), int(c.length[s])
            before, kept = -1, 0
            for i in range(min(max(int(count[s]), 0), n)):
                p = int(path[s, i])
                if not before < p < n:
                    break
                before, kept = p, kept + 1
                a, b = c.page_of(s, L + p), c.page_of(s, L + i)
                if p != i and a >= 0 and b >= 0:
                    for pool in (c.k, c.v):
                        pool[:, b, :, (L + i) % c.P] = pool[:, a, :, (L + p) % c.P]
            new[s] += kept
        return new


def c_length(c):
    return c.length.copy()


def same(c, pools=True):
    np.testing.assert_array_equal(c.dtable.get(), c.table)
    np.testing.assert_array_equal(c.drefs.get(), c.refs)
    np.testing.assert_array_equal(c.dlength.get(), c.length)
    held = np.bincount(c.table[(c.table >= 0) & (c.table < c.pages)], minlength=c.pages)
    np.testing.assert_array_equal(held, c.refs)
    if pools:
        np.testing.assert_array_equal(c.dk.get().view(np.uint8), c.k.view(np.uint8))
        np.testing.assert_array_equal(c.dv.get().view(np.uint8), c.v.view(np.uint8))


def workspace(c):
    n = qg.lib().qg_kv_workspace_bytes(c.ref)
    return Device(np.full(n, 0xff, np.uint8)), n


def reserve(c, counts):
    batch, status, (ws, n) = Batch(counts), Device(np.full(c.B, 9, np.int32)), workspace(c)
    say(f"reserve {counts[:8]}")
    call("kv_reserve", c.ref, batch.ref, status.p, ws.p, n)
    return status.get()


def fork(c, dst, src):
    d, s, (ws, n) = Device(np.array(dst, np.int32)), Device(np.array(src, np.int32)), workspace(c)
    say(f"fork {dst[:8]} from {src[:8]}")
    call("kv_fork", c.ref, d.p, s.p, len(dst), ws.p, n)


def truncate(c, new=None):
    d = Device(np.array(new, np.int32)) if new is not None else None
    say(f"truncate {new and new[:8]}")
    call("kv_truncate", c.ref, d.p if d else None)


@pytest.mark.parametrize("typ,page,dim,heads,layers", [(F16, 8, 64, 1, 1), (BF16, 32, 128, 3, 2), (F32, 16, 64, 2, 5), (F16, 256, 256, 1, 1)])
def test_pages_random_walk(qgl, typ, page, dim, heads, layers):
    """Forks, reserves, truncations and compactions in random order, with sequences that share pages, run out of pages
    and outgrow their table."""
    rng = np.random.default_rng(page + dim)
    B = 7
    c = Cache(rng, [5 * page // 2, 3, 0, page, 0, 2 * page + 1, 0], [0] * B, typ=typ, layers=layers, kv_heads=heads, page=page, dim=dim,
              spare=9, table_pages=6)
    m = Model(c)
    for step in range(40):
        kind = rng.integers(0, 4)
        if kind == 0:
            n = int(rng.integers(1, B + 1))
            dst, src = (rng.integers(-1, B + 1, n).tolist() for _ in range(2))
            fork(c, dst, src)
            m.fork(dst, src)
        elif kind == 1:
            counts = rng.integers(0, page + 3, B).tolist()
            counts[int(rng.integers(0, B))] = int(rng.integers(0, 3 * page))
            if sum(counts):
                np.testing.assert_array_equal(reserve(c, counts), m.reserve(counts))
        elif kind == 2:
            new = rng.integers(-1, 4 * page, B).tolist() if rng.random() < 0.8 else None
            truncate(c, new)
            m.truncate(new)
        else:
            counts = rng.integers(0, 18, B).tolist()
            counts[0] = max(counts[0], 1)
            status = m.reserve(counts)
            np.testing.assert_array_equal(reserve(c, counts), status)
            counts = [0 if s else n for s, n in zip(status, counts)]
            if not sum(counts):
                continue
            batch = Batch(counts)
            path = np.full((B, batch.max_rows), -1, np.int32)
            count = np.zeros(B, np.int32)
            for s, n in enumerate(counts):
                count[s] = rng.integers(0, n + 1)
                path[s, :count[s]] = np.sort(rng.choice(n, count[s], replace=False)) if n else []
            dp, dc = Device(path), Device(count)
            say("compact", count.tolist())
            call("kv_compact", c.ref, batch.ref, dp.p, dc.p, c.dlength.p)
            c.length = m.compact(batch, path, count)
        same(c)


def test_compact_all_moves(qgl):
    """Paths of every shape: identity, far jumps, overlapping moves across pages, faults; the lengths kept apart."""
    rng = np.random.default_rng(1)
    for page in (8, 64):
        counts = [64, 64, 17, 5, 9, 1, 0, 30]
        c = Cache(rng, [3, 0, 100, 7, 8, 0, 5, 33], counts, typ=BF16, layers=3, kv_heads=2, page=page, dim=64)
        batch = Batch(counts)
        for row, s, place in batch.places():
            for layer in range(3):
                c.put(layer, s, int(c.length[s]) + place, *rng.standard_normal((2, 2, 64)))
        if page == 8:  # a hole among the moved rows
            c.refs[c.table[7, 4]] = 0
            c.table[7, 4] = -1
        c.upload()
        path = np.full((8, 64), -1, np.int32)
        path[0], path[1, :63] = np.arange(64), np.arange(1, 64)
        path[2, :4], path[3, :5] = (0, 9, 10, 16), (0, 2, 2, 3, 4)   # the second repeats a row
        path[4, :3], path[5, 0] = (0, 9, 1), 0                      # and this one leaves its sequence
        path[6, :2], path[7, :10] = (0, 1), np.arange(10) * 3
        count = np.array([64, 63, 4, 5, 3, 1, 2, 1000], np.int32)
        dp, dc, out = Device(path), Device(count), Device(np.zeros(8, np.int32))
        want = Model(c).compact(batch, path, count)
        say(f"compact page={page}")
        call("kv_compact", c.ref, batch.ref, dp.p, dc.p, out.p)
        np.testing.assert_array_equal(out.get(), want)
        same(c)


def test_copy_pages(qgl):
    rng = np.random.default_rng(2)
    c = Cache(rng, [100], [0], typ=F16, layers=4, kv_heads=3, page=16, dim=64, spare=12)
    for pool in (c.k, c.v):
        pool[:] = rng.standard_normal(pool.shape)
    c.upload()
    dst, src = [9, 10, 11, 9, 3, -1, 12, 200], [1, 2, 1, 4, 5, 1, 200, 1]
    # 9 comes twice (the last counts); 3 is a source below? it is not: copied; bad indexes are left out
    dst += [13, 5]
    src += [6, 7]       # 5 is a source of the pair above, so it is not written
    for d, s, ok in zip(dst, src, (0, 1, 1, 1, 1, 0, 0, 0, 1, 0)):
        if ok:
            c.k[:, d], c.v[:, d] = c.k[:, s], c.v[:, s]
    dd, ds = Device(np.array(dst, np.int32)), Device(np.array(src, np.int32))
    say("copy pages")
    call("kv_copy_pages", c.ref, dd.p, ds.p, len(dst))
    np.testing.assert_array_equal(c.dk.get().view(np.uint16), c.k.view(np.uint16))
    np.testing.assert_array_equal(c.dv.get().view(np.uint16), c.v.view(np.uint16))


def test_reserve_many_sequences(qgl):
    """1024 sequences over 40000 pages, some shared, some rows long: the pages come in order."""
    rng = np.random.default_rng(3)
    B = 1024
    lengths = rng.integers(0, 60, B).tolist()
    c = Cache(rng, lengths, [0] * B, typ=F16, kv_heads=1, page=8, dim=64, spare=30000, table_pages=300, fill=False)
    c.k[:], c.v[:] = 0, 0
    c.upload()
    m = Model(c)
    dst, src = rng.permutation(B)[:200].tolist(), rng.integers(0, B, 200).tolist()
    fork(c, dst, src)
    m.fork(dst, src)
    counts = rng.integers(0, 20, B).tolist()
    counts[5], counts[900] = 2000, 2399
    np.testing.assert_array_equal(reserve(c, counts), m.reserve(counts))
    same(c, pools=False)


def test_reserve_keeps_forks_apart(qgl):
    """Two sequences of different lengths in one page: neither's tokens change when both are written behind."""
    rng = np.random.default_rng(4)
    c = Cache(rng, [14, 0, 0], [0, 0, 0], typ=F32, kv_heads=1, page=16, dim=64, spare=3, table_pages=2)
    fork(c, [1], [0])
    truncate(c, [14, 10, 0])
    m = Model(c)
    m.fork([1], [0])
    m.truncate([14, 10, 0])
    same(c)
    # only the shorter one is written: it must not lose the other's tokens; then no page is left for both
    np.testing.assert_array_equal(reserve(c, [0, 2, 0]), m.reserve([0, 2, 0]))
    same(c)
    np.testing.assert_array_equal(reserve(c, [16, 20, 16]), m.reserve([16, 20, 16]))
    same(c)


@pytest.mark.parametrize("n,width", [(1, 4096), (1, 4097), (32, 128), (32, 129), (33, 8), (1000, 9)])
def test_fork_of_few_and_many_entries(qgl, n, width):
    """Pairs that chain (a destination is the next pair's source), repeat and are out of range, over tables on both sides
    of what one workgroup holds."""
    rng = np.random.default_rng(n + width)
    B = min(1024, n + 3)
    lengths = [8 * width - 3, 5] + [0] * (B - 2)
    c = Cache(rng, lengths, [0] * B, typ=F16, kv_heads=1, page=8, dim=64, spare=5, table_pages=width, fill=False)
    m = Model(c)
    for rounds in range(2):
        dst, src = rng.integers(0, B, n).tolist(), rng.integers(0, min(B, 4), n).tolist()
        if n > 5:
            dst[:4], src[:4] = [2, 3, 2, B], [0, 2, 1, 0]
        fork(c, dst, src)
        m.fork(dst, src)
        same(c, pools=False)


def store_rows(c, batch, rng):
    """qg_qk_norm_rope of the batch's rows, neither normalised nor rotated; returns k and v as given."""
    row = 3 * c.H * c.D
    x = rng.standard_normal((batch.rows, row)).astype(np.float32)
    dx, out = Device(x), Device(shape=(batch.rows, c.H, c.D), dtype=np.float32)
    args = qg.QkRows(q=dx.p, k=dx.p + 4 * c.H * c.D, v=dx.p + 8 * c.H * c.D, q_row=row, q_head=c.D, k_row=row, k_head=c.D, v_row=row, v_head=c.D,
                     rows=batch.rows, q_heads=c.H, kv_heads=c.H, head_dim=c.D, eps=1e-6)
    call("qk_norm_rope", out.p, None, C.byref(args), c.ref, 0, batch.ref)
    return x.reshape(batch.rows, 3, c.H, c.D)[:, 1:].swapaxes(0, 1)


@pytest.mark.parametrize("typ", [F16, F32])
def test_rows_without_room_leave_shared_pages(qgl, typ):
    """A step that runs on after reserve found no room: neither the store nor the compaction writes into a page that
    another sequence holds."""
    rng = np.random.default_rng(21)
    c = Cache(rng, [14, 0, 0], [0, 0, 0], typ=typ, kv_heads=2, page=16, dim=64, spare=0, table_pages=2)
    fork(c, [1], [0])
    truncate(c, [14, 10, 0])
    m = Model(c)
    m.fork([1], [0])
    m.truncate([14, 10, 0])
    counts = [0, 5, 0]
    status = m.reserve(counts)
    assert status[1] == 1
    np.testing.assert_array_equal(reserve(c, counts), status)
    batch = Batch(counts)
    store_rows(c, batch, rng)
    same(c)
    for lengths in (c.dlength, Device(np.zeros(3, np.int32))):
        path, count = np.full((3, 5), -1, np.int32), np.array([0, 3, 0], np.int32)
        path[1, :3] = (0, 2, 3)
        dp, dc = Device(path), Device(count)
        say("compact after no room")
        call("kv_compact", c.ref, batch.ref, dp.p, dc.p, lengths.p)
        np.testing.assert_array_equal(lengths.get(), [14, 10, 0])
        same(c)
    # a cache without counts of its own: the caller says where rows go
    desc = qg.KvCache.from_buffer_copy(c.desc)
    desc.refs, c.ref = None, C.byref(desc)
    k, v = store_rows(c, batch, rng)
    for i in range(5):
        c.put(0, 1, 10 + i, k[i], v[i])
    np.testing.assert_array_equal(c.dk.get().view(np.uint8), c.k.view(np.uint8))
    np.testing.assert_array_equal(c.dv.get().view(np.uint8), c.v.view(np.uint8))


@pytest.mark.parametrize("page", [8, 16])
def test_lengths_stop_where_no_row_was_stored(qgl, page):
    """After a status of 1 or 2 the rows that found no page do not count, whatever was accepted of them."""
    rng = np.random.default_rng(22)
    # a page's rest for some rows (sequences 0, 1), a full page (2), none at all (3), a table too short (4)
    lengths, counts = [page - 3, 2 * page - 1, page, 0, 3 * page - 2], [9, 4, 3, 2, 9]
    for full in (False, True):   # the others get pages, or nobody does
        c = Cache(rng, lengths, [0] * 5, typ=BF16, layers=2, kv_heads=1, page=page, dim=64, spare=0 if full else 9, table_pages=3)
        m = Model(c)
        status = m.reserve(counts)
        np.testing.assert_array_equal(status, [1, 1, 1, 1, 2] if full else [0, 0, 0, 0, 2])
        np.testing.assert_array_equal(reserve(c, counts), status)
        batch = Batch(counts)
        paths = [[0, 1, 2, 3, 8], [0, 1, 3], [0, 2], [0, 1], [0, 1, 2, 5]]
        room = [3, 1, 0, 0, 2] if full else [5, 3, 2, 2, 2]   # rows of each path up to the last with a page at both ends
        path, count = np.full((5, 9), -1, np.int32), np.array([len(p) for p in paths], np.int32)
        for s, p in enumerate(paths):
            path[s, :len(p)] = p
        for row, s, place in batch.places():
            for layer in range(2):
                c.put(layer, s, int(c.length[s]) + place, *rng.standard_normal((2, 1, 64)))
        c.upload()
        want = c_length(c) + np.array(room, np.int32)
        dp, dc, out = Device(path), Device(count), Device(np.zeros(5, np.int32))
        m.compact(batch, path, count)
        say(f"compact page={page} full={full}")
        call("kv_compact", c.ref, batch.ref, dp.p, dc.p, out.p)
        np.testing.assert_array_equal(out.get(), want)
        same(c)
        # again into the cache's own lengths: the moved rows lie where they are, so only the lengths change
        identity = np.tile(np.arange(9, dtype=np.int32), (5, 1))
        dp.set(identity)
        dc.set(np.array(room, np.int32))
        call("kv_compact", c.ref, batch.ref, dp.p, dc.p, c.dlength.p)
        c.length = want
        same(c)


class Careful(Model):
    """The rules for steps that run on whatever reserve said."""

    def shared(self, p):
        return p >= 0 and self.c.refs[p] > 1

    def store(self, batch, k, v):
        c = self.c
        for row, s, place in batch.places():
            t = int(c.length[s]) + place
            if not self.shared(c.page_of(s, t)):
                c.put(0, s, t, k[row], v[row])

    def compact(self, batch, path, count):
        c, new = self.c, c_length(self.c)
        for s in range(c.B):
            n, L = int(batch.start[s + 1] - batch.start[s]), int(c.length[s])
            before, rows = -1, []
            for i in range(min(max(int(count[s]), 0), n)):
                p = int(path[s, i])
                a, b = c.page_of(s, L + p), c.page_of(s, L + i)
                if not before < p < n or self.shared(a) or self.shared(b):
                    break
                before = p
                rows.append((p, a, b))
            while rows and (rows[-1][1] < 0 or rows[-1][2] < 0):
                rows.pop()
            for i, (p, a, b) in enumerate(rows):
                if p != i and a >= 0 and b >= 0:
                    for pool in (c.k, c.v):
                        pool[:, b, :, (L + i) % c.P] = pool[:, a, :, (L + p) % c.P]
            new[s] += len(rows)
        return new


@pytest.mark.parametrize("typ,page,heads,seed", [(F16, 8, 1, 1), (BF16, 16, 2, 2), (F32, 8, 2, 3), (F16, 32, 1, 4)])
def test_steps_that_run_on_without_room(qgl, typ, page, heads, seed):
    """Steps of forked sequences over few pages, every call of each step made whatever reserve's status: tables, holders,
    lengths and every byte of the pages."""
    rng = np.random.default_rng(seed)
    B = 5
    c = Cache(rng, [3 * page // 2, 0, 0, page - 1, 2 * page], [0] * B, typ=typ, layers=2, kv_heads=heads, page=page, dim=64, spare=2, table_pages=4)
    m, seen = Careful(c), np.zeros(3, int)
    for step in range(30):
        if rng.random() < 0.5:
            dst, src = rng.integers(0, B, 2).tolist(), rng.integers(0, B, 2).tolist()
            fork(c, dst, src)
            m.fork(dst, src)
        if rng.random() < 0.4:
            new = rng.integers(0, 3 * page, B).tolist()
            truncate(c, new)
            m.truncate(new)
        counts = rng.integers(0, 9, B).tolist()
        counts[int(rng.integers(0, B))] += 1
        status = m.reserve(counts)
        np.testing.assert_array_equal(reserve(c, counts), status)
        seen += np.bincount(status, minlength=3)
        batch = Batch(counts)
        m.store(batch, *store_rows(c, batch, rng))
        path, count = np.full((B, batch.max_rows), -1, np.int32), np.zeros(B, np.int32)
        for s, n in enumerate(counts):
            count[s] = rng.integers(0, n + 1)
            path[s, :count[s]] = np.sort(rng.choice(n, count[s], replace=False)) if n else []
        dp, dc = Device(path), Device(count)
        say("compact", count.tolist(), "status", status.tolist())
        call("kv_compact", c.ref, batch.ref, dp.p, dc.p, c.dlength.p)
        c.length = m.compact(batch, path, count)
        same(c)
    assert (seen[:2] > 3).all(), seen
