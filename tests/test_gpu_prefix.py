"""qg_kv_prefixes and qg_prefix_attention against plain statements of both in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from nebula_amd import qg
from nebula_amd.qg import Device
from prefix_oracle import Forked, prefixes
from spec_oracle import BF16, F16, F32, Batch, attention, decode, encode, random_tree

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def whatever_it_saves(qgl):
    """Small batches share their pages too."""
    before = qgl.qg_prefix_least_saving(0)
    yield
    qgl.qg_prefix_least_saving(before)


class Plan:
    """The buffer of a cache and batch, and what was found."""

    def __init__(self, cache, batch):
        self.bytes = qg.lib().qg_kv_prefixes_bytes(cache.ref, batch.ref)
        assert self.bytes
        self.buffer = Device(np.full(self.bytes, 0xA5, np.uint8))
        self.link, self.shared = (Device(np.full(cache.B, -9, np.int32)) for _ in range(2))
        self.cache, self.batch = cache, batch

    def find(self):
        qg.call("kv_prefixes", self.link.p, self.shared.p, self.cache.ref, self.batch.ref, self.buffer.p, self.bytes)

    def check(self):
        counts = [min(int(b - a), self.batch.max_rows) for a, b in zip(self.batch.start, self.batch.start[1:])]
        link, shared = prefixes(self.cache.table, self.cache.pages, self.cache.P, self.cache.length, counts)
        assert np.array_equal(self.shared.get(), shared), (self.shared.get(), shared)
        assert np.array_equal(self.link.get(), link)


class Attend:
    def __init__(self, cache, batch, q, scale, layer=0):
        self.cache, self.batch, self.q, self.scale, self.layer = cache, batch, np.ascontiguousarray(q, np.float32), scale, layer
        self.plan = Plan(cache, batch)
        self.dq, self.out = Device(self.q), Device(np.full(self.q.shape, 7, np.float32))
        self.bytes = qg.lib().qg_prefix_attention_workspace_bytes(cache.ref, batch.ref, q.shape[1])
        assert self.bytes
        self.ws = Device(np.full(self.bytes, 0xA5, np.uint8))

    def run(self, find=True):
        if find:
            self.plan.find()
        qg.call("prefix_attention", self.out.p, self.dq.p, self.q.shape[1], self.scale, self.cache.ref, self.layer, self.batch.ref, self.plan.buffer.p,
                self.plan.bytes, self.ws.p, self.bytes)
        return self.out.get()

    def check(self):
        got = self.run()
        want, tol, done = attention(self.cache, self.batch, self.q, self.scale, self.layer)
        bad = np.abs(got - want) > tol
        assert not bad[done].any(), (np.argwhere(bad & done[:, None, None])[:5], np.abs(got - want)[done].max(), tol[done].max())
        assert (got[~done] == 7).all()  # rows of no sequence
        return got


def fill_rows(rng, cache, batch, layer=0):
    """Keys and values of the batch's rows behind the cached tokens."""
    for _, s, i in batch.places():
        cache.put(layer, s, int(cache.length[s]) + i, *(rng.standard_normal((cache.H, cache.D)) for _ in range(2)))
    cache.upload()


def build(rng, family, counts, tree=False, heads=8, max_rows=None, rows=None, **kw):
    cache = Forked(rng, family, [max(c, 0) for c in counts], **kw)
    parents = [random_tree(rng, c) if c else [] for c in counts] if tree else None
    batch = Batch(counts, parents, max_rows=max_rows, rows=rows)
    fill_rows(rng, cache, batch)
    q = rng.standard_normal((batch.rows, heads, cache.D)).astype(np.float32)
    return Attend(cache, batch, q, cache.D ** -0.5)


# (from, common, own) of each sequence
FAMILIES = {
    "alone": [(-1, 0, 300)],
    "strangers": [(-1, 0, 40), (-1, 0, 700), (-1, 0, 0)],
    "forks": [(-1, 0, 700)] + [(0, 700, 3)] * 6,
    "forks of whole pages": [(-1, 0, 768), (0, 768, 0), (0, 768, 0), (0, 768, 1)],
    "short": [(-1, 0, 255), (0, 255, 0), (0, 200, 30)],
    "two levels": [(-1, 0, 900), (0, 900, 5), (0, 300, 500), (2, 800, 9), (2, 790, 20), (0, 310, 0), (-1, 0, 20)],
    "branches": [(-1, 0, 1400)] + [(0, c, 17) for c in (300, 1300, 600, 601, 256, 1200, 900, 255)],
    "a line of branches": [(-1, 0, 400), (0, 390, 300), (1, 650, 300), (2, 900, 300), (3, 1190, 300), (1, 660, 10)],
    "late owner": [(-1, 0, 10), (-1, 0, 800), (1, 800, 2), (1, 513, 300), (-1, 0, 0)],
}
COUNTS = {1: lambda i: 1, 3: lambda i: 1 + i % 3, 9: lambda i: (i * 5) % 10}


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("most", COUNTS)
@pytest.mark.parametrize("tree", [False, True])
def test_families(qgl, family, most, tree):
    rng = np.random.default_rng(len(family) * 100 + most)
    f = FAMILIES[family]
    counts = [COUNTS[most](i) for i in range(len(f))]
    if not sum(counts):
        counts[0] = 1
    a = build(rng, f, counts, tree)
    a.check()
    a.plan.check()


def test_what_is_worth_sharing(qgl):
    """Below the least saving each sequence reads for itself: the search's outputs are the same, the attention's within its error."""
    rng = np.random.default_rng(2)
    a = build(rng, FAMILIES["two levels"], [1, 3, 1, 2, 1, 1, 1], kv_heads=2, dim=64, typ=F16)
    outs, heads = [], []
    saved = sum(int(x) // 256 * 256 for x in prefixes(a.cache.table, a.cache.pages, a.cache.P, a.cache.length, [1] * 7)[1]) * 2 * 2 * 64 * 2
    for least in (0, saved, saved + 1, 1 << 40, -1):
        qgl.qg_prefix_least_saving(least)
        outs.append(a.check())
        a.plan.check()
        heads.append(a.plan.buffer.get()[:8].view(np.int32).tolist())  # segments, and those that are shared
    assert heads[0] == heads[1] and heads[0][1] > 0
    assert heads[2] == heads[3] == heads[4] == [7, 0]
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[2], outs[3])


@pytest.mark.parametrize("typ", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (10, 2), (16, 2), (16, 1), (40, 1)])
def test_types_and_heads(qgl, typ, dim, heads, kv_heads):
    rng = np.random.default_rng(dim + heads)
    a = build(rng, FAMILIES["two levels"], [1, 4, 1, 2, 1, 3, 1], heads % 4 == 0, heads, typ=typ, dim=dim, kv_heads=kv_heads, page=32)
    a.check()


@pytest.mark.parametrize("page", [8, 64, 256, 512])
@pytest.mark.parametrize("rows", [1, 17])
def test_pages(qgl, page, rows):
    rng = np.random.default_rng(page)
    family = [(-1, 0, 1300), (0, 1300, 40), (0, 1100, 260), (2, 1280, 5), (0, 520, 1)]
    a = build(rng, family, [rows, 1, rows, 2, 1], rows == 17, page=page)
    a.check()
    a.plan.check()


@pytest.mark.parametrize("counts", [[70, 1, 90, 5], [200, 0, 130, 1]])
def test_chunks(qgl, counts):
    """Chains of more rows than a tree has: chunks of prompts behind a common text."""
    rng = np.random.default_rng(sum(counts))
    build(rng, [(-1, 0, 600), (0, 600, 3), (0, 520, 60), (2, 570, 0)], counts, heads=4).check()


def test_many_sequences(qgl):
    """More segments than a wave has lanes; sequences without rows between."""
    rng = np.random.default_rng(3)
    family = [(-1, 0, 520), (-1, 0, 300)]
    for i in range(2, 150):
        up = int(rng.integers(0, i))
        family.append((up, int(rng.integers(0, 900)), int(rng.integers(0, 120))))
    counts = [int(rng.integers(0, 3)) for _ in family]
    a = build(rng, family, counts, heads=2, kv_heads=1)
    a.check()
    a.plan.check()


def test_more_branches_than_partial_results(qgl):
    """Every sequence leaves the first at a place of its own: the segments get longer until their rows are few enough."""
    rng = np.random.default_rng(4)
    family = [(-1, 0, 256 * 44)] + [(0, 256 * i + 3, 2) for i in range(1, 44)]
    a = build(rng, family, [1] * 44, heads=1, kv_heads=1)
    a.check()
    a.plan.check()


@pytest.mark.parametrize("seed", range(4))
def test_found_prefixes(qgl, seed):
    """Tables of any content: pages shared anywhere, entries that are none, lengths past the table."""
    rng = np.random.default_rng(seed)
    S, W = [(5, 700), (70, 40), (300, 9), (1024, 3)][seed]
    cache = Forked(rng, [(-1, 0, 1)] * S, [1] * S, page=8, kv_heads=1, extra=W - 1)
    base = rng.integers(0, cache.pages, W)
    for s in range(S):
        cut = int(rng.integers(0, W + 1))
        cache.table[s, :cut] = base[:cut]
        cache.table[s, cut:] = rng.integers(-2, cache.pages + 2, W - cut)
        if s and rng.random() < 0.4:
            cache.table[s] = cache.table[rng.integers(0, s)]
        if rng.random() < 0.1:
            cache.table[s, rng.integers(0, W)] = -1
    cache.length = rng.integers(-3, W * 8 + 20, S).astype(np.int32)
    cache.upload()
    plan = Plan(cache, Batch([int(rng.integers(0, 2)) for _ in range(S)], rows=S + 1, max_rows=1))
    plan.find()
    plan.check()
    plan.find()
    plan.check()
    # without the outputs
    qg.call("kv_prefixes", None, None, cache.ref, plan.batch.ref, plan.buffer.p, plan.bytes)
    qg.call("sync")


def test_rows_of_no_sequence_and_cut_batches(qgl):
    """Rows behind the last sequence, and sequences of more rows than max_rows."""
    rng = np.random.default_rng(6)
    a = build(rng, FAMILIES["forks"], [2] * 7, rows=17)
    a.check()
    a = build(rng, FAMILIES["forks"], [2, 5, 1, 0, 0, 3, 2], max_rows=3)
    a.check()


def special(a, what):
    """Puts values of a kind into the shared pages and the own ones."""
    c = a.cache
    k, v = (decode(p, c.typ).astype(np.float32) for p in (c.k, c.v))
    p0, p1 = c.table[0, 2], c.table[1, int(c.length[1]) // c.P]
    if what == "key -inf":
        k[0, p0, :, 3, 5] = -np.inf
    elif what == "value inf":
        v[0, p0, :, 3, 5] = np.inf
    elif what == "value nan of one":
        v[0, p1, :, int(c.length[1]) % c.P, 7] = np.nan
    elif what == "large values":
        v[:] = np.where(np.isnan(v), v, np.sign(v) * 3e38)
    with np.errstate(over="ignore"):
        c.k, c.v = encode(k, c.typ), encode(v, c.typ)
    c.upload()


@pytest.mark.parametrize("what", ["key -inf", "value inf", "value nan of one"])
@pytest.mark.parametrize("typ", [F32, F16, BF16])
def test_values_that_are_no_numbers(qgl, typ, what):
    """Only rows that see such a value with a weight above 0 have it, as in the definition."""
    rng = np.random.default_rng(7)
    a = build(rng, FAMILIES["forks"], [1, 2, 1, 1, 1, 2, 1], typ=typ)
    special(a, what)
    got = a.run()
    with np.errstate(invalid="ignore"):
        want, tol, done = attention(a.cache, a.batch, a.q, a.scale)
    finite = np.isfinite(want)
    assert (np.isfinite(got) == finite).all()
    assert (np.abs(got - want)[finite] <= tol[finite]).all()
    # the same calls of the attention that reads each sequence by itself
    n = qgl.qg_tree_attention_workspace_bytes(a.cache.ref, a.batch.ref, 8)
    ws, out = Device(np.zeros(n, np.uint8)), Device(np.zeros(a.q.shape, np.float32))
    qg.call("tree_attention", out.p, a.dq.p, 8, a.scale, a.cache.ref, 0, a.batch.ref, ws.p, n)
    assert (np.isnan(out.get()) == np.isnan(got)).all() and (np.isinf(out.get()) == np.isinf(got)).all()


@pytest.mark.parametrize("typ", [F32, BF16])
def test_values_near_the_types_end(qgl, typ):
    rng = np.random.default_rng(8)
    a = build(rng, FAMILIES["forks"], [1] * 7, typ=typ)
    special(a, "large values")
    a.check()


def test_rows_that_see_nothing(qgl):
    """Tables without pages, shared ones with a hole, lengths of zero."""
    rng = np.random.default_rng(9)
    a = build(rng, [(-1, 0, 0), (-1, 0, 600), (1, 600, 4), (1, 600, 0)], [1, 2, 1, 1])
    a.cache.table[0, :] = -1
    a.cache.table[1, 4] = a.cache.table[2, 4] = -1
    a.cache.upload()
    got = a.check()
    assert (got[0] == 0).all()
    a.plan.check()


def test_whole_sequence_of_infinite_scores(qgl):
    rng = np.random.default_rng(10)
    a = build(rng, FAMILIES["forks"], [1] * 7)
    q = a.q.copy()
    q[3, 2] = np.nan
    q[5, 1, 0] = np.inf
    a.q = q
    a.dq.set(q)
    got = a.run()
    assert np.isnan(got[3, 2]).all() and np.isnan(got[5, 1]).any()
    clear = np.ones(got.shape[:2], bool)
    clear[3, 2] = clear[5, 1] = False
    q2 = np.where(np.isfinite(q), q, 0).astype(np.float32)
    want, tol, _ = attention(a.cache, a.batch, q2, a.scale)
    assert (np.abs(got - want)[clear] <= tol[clear]).all()


@pytest.mark.parametrize("rows", [1, 5])
def test_replayed(qgl, rows):
    """Search and attention of two layers in one graph: queries, tables and lengths change between replays."""
    rng = np.random.default_rng(11)
    families = [FAMILIES["forks"], [(-1, 0, 500)] * 7, [(-1, 0, 690)] + [(0, 300 + 60 * i, 9) for i in range(6)]]
    caches = [Forked(rng, f, [rows] * 7, layers=2, spare=400 - sum(-(-(x[2] + rows) // 16) for x in f), extra=60) for f in families]
    pages, width = max(c.pages for c in caches), min(c.width for c in caches)
    batch = Batch([rows] * 7, [random_tree(rng, rows) for _ in range(7)])
    first = caches[0]
    attends = None
    graph = C.c_void_p()
    held = {}
    for turn in range(6):
        c = caches[turn % 3]
        for layer in range(2):
            for _, s, i in batch.places():
                c.put(layer, s, int(c.length[s]) + i, *(rng.standard_normal((c.H, c.D)) for _ in range(2)))
        # all in the first cache's buffers
        if turn == 0:
            held["k"], held["v"] = (Device(np.zeros((2, pages) + c.k.shape[2:], c.k.dtype)) for _ in range(2))
            held["table"], held["length"] = Device(np.full((7, width), -1, np.int32)), Device(np.zeros(7, np.int32))
            first.desc = qg.KvCache(k=held["k"].p, v=held["v"].p, type=c.typ, layers=2, pages=pages, kv_heads=c.H, page_tokens=c.P, head_dim=c.D,
                                    refs=None, table=held["table"].p, length=held["length"].p, sequences=7, table_pages=width)
            first.ref = C.byref(first.desc)
            q = rng.standard_normal((2, batch.rows, 8, 64)).astype(np.float32)
            attends = [Attend(first, batch, q[i], 0.125, i) for i in range(2)]
            attends[1].plan = attends[0].plan
            qg.call("graph_begin", C.byref(graph))
            attends[0].plan.find()
            for a in attends:
                qg.call("prefix_attention", a.out.p, a.dq.p, 8, 0.125, first.ref, a.layer, batch.ref, a.plan.buffer.p, a.plan.bytes, attends[0].ws.p,
                        attends[0].bytes)
            qg.call("graph_end", graph)
        for name, pool in (("k", c.k), ("v", c.v)):
            whole = np.zeros((2, pages) + c.k.shape[2:], c.k.dtype)
            whole[:, :c.pages] = pool
            held[name].set(whole)
        assert (c.table[:, width:] == -1).all()
        held["table"].set(c.table[:, :width])
        held["length"].set(c.length)
        for a in attends:
            a.q = rng.standard_normal(a.q.shape).astype(np.float32)
            a.dq.set(a.q)
        qg.call("graph_launch", graph)
        qg.call("sync")
        got = [a.out.get().copy() for a in attends]
        for a, g in zip(attends, got):
            want, tol, _ = attention(c, batch, a.q, 0.125, a.layer)
            assert (np.abs(g - want) <= tol).all(), turn
            assert np.array_equal(a.run(), g)  # eager, the same bits
    qgl.qg_graph_destroy(graph)


@pytest.mark.parametrize("fill", [0, 1, 0xFF])
def test_rows_of_no_sequence_whatever_lay_there(qgl, fill):
    """Rows before the first sequence, between two and behind the last, with a buffer that an earlier batch filled."""
    rng = np.random.default_rng(16)
    for family, counts, most, skip in (("forks", [2, 5, 1, 0, 0, 3, 2], 3, 2), ("two levels", [1, 0, 4, 1, 1, 1, 9], 4, 3), ("strangers", [0, 3, 0], 2, 1)):
        cache = Forked(rng, FAMILIES[family], counts)
        batch = Batch(counts, max_rows=most, rows=sum(counts) + skip + 5)
        batch.start += skip
        batch.dstart.set(batch.start)
        fill_rows(rng, cache, batch)
        a = Attend(cache, batch, rng.standard_normal((batch.rows, 8, cache.D)), cache.D ** -0.5)
        a.plan.buffer.set(np.full(a.plan.bytes, fill, np.uint8))
        a.check()
        a.plan.check()


def test_workspace_and_buffer_of_larger_batches(qgl):
    rng = np.random.default_rng(12)
    a = build(rng, FAMILIES["branches"], [3] * 9)
    big = Batch([7] * 9)
    assert qgl.qg_kv_prefixes_bytes(a.cache.ref, big.ref) >= a.plan.bytes
    n = qgl.qg_prefix_attention_workspace_bytes(a.cache.ref, big.ref, 8)
    assert all(0 < qgl.qg_prefix_attention_workspace_bytes(a.cache.ref, Batch([r], rows=r + 3).ref, 8) <= n for r in range(1, 60))
    a.bytes, a.ws = n, Device(np.full(n, 0x5A, np.uint8))
    a.check()


def test_buffer_of_another_batch(qgl):
    """A buffer that no longer fits its batch: other rows stay untouched and the next right call is right."""
    rng = np.random.default_rng(13)
    a = build(rng, FAMILIES["two levels"], [5, 1, 2, 1, 3, 1, 2])
    a.plan.find()
    other = build(rng, FAMILIES["alone"], [2], extra=40)
    buffer = a.plan.buffer
    assert a.plan.bytes >= other.plan.bytes
    qg.call("prefix_attention", other.out.p, other.dq.p, 8, other.scale, other.cache.ref, 0, other.batch.ref, buffer.p, a.plan.bytes, other.ws.p, other.bytes)
    qg.call("sync")
    for fill in (0xFF, 0x7F, 0x01):
        buffer.set(np.full(a.plan.bytes, fill, np.uint8))
        qg.call("prefix_attention", a.out.p, a.dq.p, 8, a.scale, a.cache.ref, 0, a.batch.ref, buffer.p, a.plan.bytes, a.ws.p, a.bytes)
        qg.call("sync")
    a.check()
    other.check()


def test_starts_outside_the_rows(qgl):
    """Row starts below the first row and behind the last are cut to what there is; starts that run backwards, lengths that are none:
    nothing outside is touched, and the next right call is right."""
    rng = np.random.default_rng(17)
    counts = [2, 0, 5, 5]
    cache = Forked(rng, [(-1, 0, 700), (0, 600, 3), (0, 530, 60), (2, 580, 9)], counts)
    batch = Batch(counts, rows=14, max_rows=5)
    batch.start = np.array([-7, 2, 2, 9, 1 << 30], np.int32)
    batch.places = lambda: [(0, 0, 0), (1, 0, 1)] + [(2 + i, 2, i) for i in range(5)] + [(9 + i, 3, i) for i in range(5)]
    batch.dstart.set(batch.start)
    fill_rows(rng, cache, batch)
    a = Attend(cache, batch, rng.standard_normal((14, 8, 64)), 0.125)
    a.check()
    for starts in ([5, -3, 900, 2, 1 << 30], [14, 9, 3, 1, 0], [1 << 30] * 5, [-(1 << 31)] * 5, [0, 14, 0, 14, 0]):
        batch.dstart.set(np.array(starts, np.int32))
        for lengths in ([1 << 30, -5, -(1 << 31), cache.width * cache.P + 1], list(cache.length)):
            cache.dlength.set(np.array(lengths, np.int32))
            a.run()
    batch.dstart.set(batch.start)
    a.out.set(np.full(a.q.shape, 7, np.float32))
    a.check()


@pytest.mark.parametrize("sequences", [300, 700, 1024])
def test_hundreds_of_segments(qgl, sequences):
    """As many segments as a workgroup of the attention has threads, and more, shared ones among them."""
    rng = np.random.default_rng(18)
    family = [(-1, 0, 600)]
    for i in range(1, sequences):
        family.append((int(rng.integers(0, i)), int(rng.integers(200, 900)), int(rng.integers(0, 400))))
    a = build(rng, family, [int(rng.integers(0, 4)) for _ in family], heads=4, kv_heads=1)
    a.check()
    a.plan.check()
    count, shared = a.plan.buffer.get()[:8].view(np.int32)
    assert count >= 256 and shared > 16


def test_far_layers(qgl):
    """A layer behind more than 4 GiB of others, and pages at the end of the pools: offsets beyond 32 bits."""
    rng = np.random.default_rng(19)
    layers, heads, dim, page, pages = 40, 8, 128, 64, 1024
    cache = Forked(rng, [(-1, 0, 700), (0, 640, 3), (0, 600, 70)], [2, 1, 3], kv_heads=heads, page=page, dim=dim)
    bytes_layer = pages * heads * page * dim * 2
    big = [Device.__new__(Device) for _ in range(2)]
    for d in big:
        d.x, d.p = np.zeros(1, np.uint8), qgl.qg_alloc(layers * bytes_layer)
        assert d.p
    batch = Batch([2, 1, 3])
    fill_rows(rng, cache, batch)
    layer, first = layers - 1, pages - cache.pages
    for d, host in zip(big, (cache.k, cache.v)):
        qg.call("write", d.p + layer * bytes_layer + first * heads * page * dim * 2, np.ascontiguousarray(host).ctypes.data, host.nbytes)
    desc = qg.KvCache.from_buffer_copy(cache.desc)
    table = Device(np.where(cache.table >= 0, cache.table + first, -1).astype(np.int32))
    desc.k, desc.v, desc.layers, desc.pages, desc.table = big[0].p, big[1].p, layers, pages, table.p
    q = rng.standard_normal((6, heads * 2, dim)).astype(np.float32)
    want, tol, _ = attention(cache, batch, q, dim ** -0.5)
    cache.ref = C.byref(desc)
    got = Attend(cache, batch, q, dim ** -0.5, layer).run()
    assert np.all(np.abs(got - want) <= tol)
