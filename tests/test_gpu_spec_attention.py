"""qg_tree_attention against a 64-bit statement of it (spec_oracle.attention)."""
import copy
import ctypes as C
import math
import sys

import numpy as np
import pytest

import spec_oracle as O
from nebula_amd import qg
from nebula_amd.qg import Device, call
from spec_oracle import BF16, F16, F32, U, Batch, Cache

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def store(cache, batch, rng, layer=0, scale=1.0):
    """The batch's own rows, in the host copy."""
    for row, s, place in batch.places():
        cache.put(layer, s, int(cache.length[s]) + place, *(scale * rng.standard_normal((2, cache.H, cache.D))))
    cache.upload()


def attend(cache, batch, q, scale, layer=0, sentinel=np.nan):
    dq = Device(q)
    out = Device(np.full(q.shape, sentinel, np.float32))
    n = qg.lib().qg_tree_attention_workspace_bytes(cache.ref, batch.ref, q.shape[1])
    assert n
    ws = Device(np.full(n, 0xff, np.uint8))  # NaN: nothing of a workspace counts that was not written
    say(f"attention q{q.shape} type={cache.typ} page={cache.P} lengths={list(cache.length)[:8]} rows={batch.rows} tree={batch.parent is not None}")
    call("tree_attention", out.p, dq.p, q.shape[1], scale, cache.ref, layer, batch.ref, ws.p, n)
    return out.get()


def check(cache, batch, q, scale, layer=0):
    got = attend(cache, batch, q, scale, layer)
    want, tol, done = O.attention(cache, batch, q, scale, layer)
    assert np.isnan(got[~done]).all()
    bad = ~(np.abs(got - want) <= tol) & done[:, None, None]
    assert not bad.any(), (np.argwhere(bad)[:5], np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-30)))
    return got


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("dim,heads,group,page", [(64, 1, 1, 8), (64, 2, 8, 16), (128, 2, 5, 64), (128, 1, 16, 32), (256, 2, 4, 16), (128, 4, 3, 1024)])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_shapes(qgl, typ, dim, heads, group, page, tree):
    rng = np.random.default_rng(dim + group + page + typ)
    counts, lengths = [1, 5, 0, 17, 2], [0, 31, 8, 100, 257]
    cache = Cache(rng, lengths, counts, typ=typ, layers=2, kv_heads=heads, page=page, dim=dim)
    batch = Batch(counts, [O.random_tree(rng, n) if n else [] for n in counts] if tree else None, rows=sum(counts) + 3)
    store(cache, batch, rng, layer=1)
    q = rng.standard_normal((batch.rows, heads * group, dim)).astype(np.float32)
    check(cache, batch, q, dim ** -0.5, layer=1)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("length", [0, 1, 7, 8, 31, 32, 33, 63, 64, 127, 128, 129, 1000, 4099])
def test_attention_one_row(qgl, typ, length):
    rng = np.random.default_rng(length)
    cache = Cache(rng, [length], [1], typ=typ, kv_heads=2, page=32, dim=64)
    batch = Batch([1])
    store(cache, batch, rng)
    check(cache, batch, rng.standard_normal((1, 10, 64)).astype(np.float32), 0.125)


@pytest.mark.parametrize("typ,dim", [(F16, 128), (BF16, 64), (F32, 64), (BF16, 256)])
@pytest.mark.parametrize("rows,length", [(64, 0), (64, 77), (33, 2000), (2, 5000)])
def test_attention_trees(qgl, typ, dim, rows, length):
    rng = np.random.default_rng(rows + length)
    for width in (1, 3, 64):
        cache = Cache(rng, [length], [rows], typ=typ, kv_heads=1, page=16, dim=dim)
        batch = Batch([rows], [O.random_tree(rng, rows, width)])
        store(cache, batch, rng)
        check(cache, batch, rng.standard_normal((rows, 4, dim)).astype(np.float32), dim ** -0.5)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
def test_attention_prompt_chunk(qgl, typ):
    """A chain longer than a tree may be: a prompt chunk behind cached tokens, and one at the start."""
    rng = np.random.default_rng(5)
    counts, lengths = [130, 300, 3], [65, 0, 200]
    cache = Cache(rng, lengths, counts, typ=typ, kv_heads=2, page=32, dim=64)
    batch = Batch(counts)
    store(cache, batch, rng)
    check(cache, batch, rng.standard_normal((batch.rows, 6, 64)).astype(np.float32), 0.125)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
def test_attention_many_ragged_sequences(qgl, typ):
    rng = np.random.default_rng(6)
    counts = [int(x) for x in rng.integers(0, 4, 130)]
    lengths = [int(x) for x in rng.integers(0, 90, 129)] + [3000]
    cache = Cache(rng, lengths, counts, typ=typ, kv_heads=1, page=16, dim=64)
    batch = Batch(counts, max_rows=3)
    store(cache, batch, rng)
    check(cache, batch, rng.standard_normal((batch.rows, 4, 64)).astype(np.float32), 0.125)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
def test_attention_holes_and_bad_entries(qgl, typ):
    """Table entries that are no pages hold nothing; a row that sees nothing is zero; lengths and row starts outside
    their range are cut."""
    rng = np.random.default_rng(7)
    counts, lengths = [3, 4, 5, 2], [60, 40, 50, 0]
    cache = Cache(rng, lengths, counts, typ=typ, kv_heads=2, page=16, dim=64)
    batch = Batch(counts, [O.random_tree(rng, n) for n in counts])
    store(cache, batch, rng)
    cache.table[0, 1], cache.table[1, 0], cache.table[1, 1] = cache.pages, -7, 0x7fffffff
    cache.table[2, :] = -1
    cache.upload()
    q = rng.standard_normal((batch.rows, 4, 64)).astype(np.float32)
    got = check(cache, batch, q, 0.125)
    assert (got[7:12] == 0).all()
    # a length beyond the table is the table's; one below zero is none
    cache.table[2, :] = cache.table[0, 2]
    cache.length[:] = [1 << 30, -5, -(1 << 31), cache.width * cache.P + 1]
    cache.upload()
    got = attend(cache, batch, q, 0.125)
    assert (got[3:7] == 0).all()  # neither cached tokens nor a page of their own
    # starts that run backwards or beyond the rows
    batch.dstart.set(np.array([5, -3, 900, 2, 1 << 30], np.int32))
    cache.dlength.set(np.array(lengths, np.int32))
    attend(cache, batch, q, 0.125)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
def test_attention_masked_nonfinite(qgl, typ):
    """NaN and infinities in keys and values reach the rows that see them and no others; behind the last token, in
    free pages and in unused slots (all NaN here) they reach none."""
    rng = np.random.default_rng(8)
    rows, length = 9, 70
    cache = Cache(rng, [length], [rows], typ=typ, kv_heads=1, page=16, dim=64)
    parents = [-1, 0, 0, 1, 1, 2, 2, 5, 5]
    batch = Batch([rows], [parents])
    store(cache, batch, rng)
    for t, what in ((length + 3, np.nan), (length + 6, np.inf)):
        p = cache.page_of(0, t)
        cache.v[0, p, 0, t % 16, 5] = O.encode([what], typ)[0]
        cache.k[0, p, 0, t % 16, 9] = O.encode([np.nan if t == length + 3 else 0], typ)[0]
    cache.upload()
    q = rng.standard_normal((rows, 3, 64)).astype(np.float32)
    got = attend(cache, batch, q, 0.125)
    want, tol, done = O.attention(cache, batch, q, 0.125)
    for r in range(rows):
        if r == 3:
            assert np.isnan(got[r]).all()
        elif r == 6:
            assert (got[r, :, 5] == np.inf).all()
            keep = np.arange(64) != 5
            assert np.all(np.abs(got[r][:, keep] - want[r][:, keep]) <= tol[r][:, keep])
        else:
            assert np.all(np.abs(got[r] - want[r]) <= tol[r]), r


@pytest.mark.parametrize("typ", [F16, BF16, F32])
def test_attention_score_range(qgl, typ):
    """Scores far apart and large, queries of very different sizes, keys of the lowest value and scores of minus infinity."""
    rng = np.random.default_rng(9)
    cache = Cache(rng, [300, 90], [4, 2], typ=typ, kv_heads=1, page=32, dim=128)
    batch = Batch([4, 2])
    store(cache, batch, rng)
    q = rng.standard_normal((6, 4, 128)).astype(np.float32)
    q[0] *= 30
    q[1] *= 1e-6
    q[2, 1] = 0
    q[3, 0, :64] *= 1e-8
    check(cache, batch, q, 128 ** -0.5)
    # the largest score comes late and is far above the others
    for t in (250, 299):
        cache.put(0, 0, t, np.full((1, 128), 3.0), np.full((1, 128), 1.0))
    q[0] = np.abs(q[0]) * 0.2
    cache.upload()
    check(cache, batch, q, 128 ** -0.5)
    # rows whose every score is minus infinity are zero; one finite score takes all
    q[4:] = 0
    q[4:, :, 0] = 1.0
    p, low = cache.page_of, O.encode([-np.inf], typ)[0]
    for t in range(92):
        cache.k[0, p(1, t), 0, t % 32] = 0
        if t != 40:
            cache.k[0, p(1, t), 0, t % 32, 0] = low
    cache.upload()
    got = attend(cache, batch, q, 1.0)
    want = cache.token(cache.v, 0, 1, 40)[0]
    np.testing.assert_array_equal(got[4:], np.broadcast_to(want.astype(np.float32), (2, 4, 128)))
    cache.k[0, p(1, 40), 0, 40 % 32, 0] = low
    cache.upload()
    assert (attend(cache, batch, q, 1.0)[4:] == 0).all()


def test_attention_far_offsets(qgl):
    """A layer behind more than 4 GiB of others: offsets beyond 32 bits."""
    rng = np.random.default_rng(10)
    layers, heads, dim, page = 40, 8, 128, 64
    cache = Cache(rng, [200], [2], typ=F16, kv_heads=heads, page=page, dim=dim, spare=0)
    pages = 1024
    bytes_layer = pages * heads * page * dim * 2
    big = [Device.__new__(Device) for _ in range(2)]
    for d in big:
        d.x, d.p = np.zeros(1, np.uint8), qg.lib().qg_alloc(layers * bytes_layer)
        assert d.p
    batch = Batch([2])
    store(cache, batch, rng)
    layer, first = layers - 1, pages - cache.pages
    for d, host in zip(big, (cache.k, cache.v)):
        at = d.p + layer * bytes_layer + first * heads * page * dim * 2
        call("write", at, np.ascontiguousarray(host).ctypes.data, host.nbytes)
    desc = qg.KvCache.from_buffer_copy(cache.desc)
    table = Device(np.where(cache.table >= 0, cache.table + first, -1).astype(np.int32))
    desc.k, desc.v, desc.layers, desc.pages, desc.table = big[0].p, big[1].p, layers, pages, table.p
    q = rng.standard_normal((2, heads * 2, dim)).astype(np.float32)
    want, tol, _ = O.attention(cache, batch, q, dim ** -0.5)
    cache.ref = C.byref(desc)
    got = attend(cache, batch, q, dim ** -0.5, layer)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
def test_attention_long_context_split(qgl, typ):
    """A long cache beside short ones, so that its work is split and joined; the same answer twice, bit for bit."""
    rng = np.random.default_rng(11)
    cache = Cache(rng, [20000, 3, 500], [5, 5, 1], typ=typ, kv_heads=1, page=64, dim=64)
    batch = Batch([5, 5, 1], [O.random_tree(rng, n) for n in (5, 5, 1)])
    store(cache, batch, rng)
    q = rng.standard_normal((11, 6, 64)).astype(np.float32)
    a = check(cache, batch, q, 0.125)
    np.testing.assert_array_equal(a, attend(cache, batch, q, 0.125))


def test_attention_overlapping_starts(qgl):
    """Row starts that run forwards and backwards give sequences the same rows, more of them than there is work for:
    nothing outside the buffers is touched, and rows of no sequence stay."""
    rng = np.random.default_rng(12)
    B, N = 200, 40
    cache = Cache(rng, [10] * B, [N] * B, typ=F16, kv_heads=1, page=32, dim=64, fill=False)
    cache.k[:], cache.v[:] = 0.5, 0.25
    cache.upload()
    batch = Batch([0] * (B - 1) + [N], rows=N + 2, max_rows=N)
    batch.dstart.set(np.array([0, N] * (B // 2) + [0], np.int32))
    q = rng.standard_normal((N + 2, 8, 64)).astype(np.float32)
    got = attend(cache, batch, q, 0.125)
    assert np.isnan(got[N:]).all()


def test_attention_without_rows(qgl):
    """A batch none of whose rows belongs to a sequence."""
    cache = Cache(np.random.default_rng(13), [10, 0], [0, 0], typ=F16, kv_heads=1, page=8, dim=64)
    batch = Batch([0, 0], rows=4, max_rows=2)
    assert np.isnan(attend(cache, batch, np.ones((4, 2, 64), np.float32), 0.125)).all()


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("length,page", [(90, 16), (9000, 64)])
def test_attention_infinite_keys_and_queries(qgl, typ, length, page):
    """A key whose score is minus infinity has weight 0, whatever bits the query has: random queries, and queries whose
    product with the scale is a power of two (every plane but the first is 0)."""
    rng = np.random.default_rng(length)
    rows, heads, dim = 3, 8, 64
    cache = Cache(rng, [length, 40], [rows, 1], typ=typ, kv_heads=1, page=page, dim=dim)
    batch = Batch([rows, 1])
    store(cache, batch, rng)
    low, skip = O.encode([-np.inf], typ)[0], {0: {0, 1, 33, 64, 89} | set(range(100, length, 97)), 1: set(range(41))}
    for s, positions in skip.items():
        for t in positions:
            cache.k[0, cache.page_of(s, t), 0, t % page, 1 + t % 7] = low
    cache.upload()
    finite = copy.copy(cache)
    finite.page_of = lambda s, t: -1 if t in skip[s] else cache.page_of(s, t)
    for scale, power in ((dim ** -0.5, False), (math.log(2.0), True)):
        q = rng.standard_normal((rows + 1, heads, dim)).astype(np.float32)
        if power:
            q = (np.sign(q) * 2.0 ** np.clip(np.round(np.log2(np.abs(q) + 1e-3)) - 4, -9, -2)).astype(np.float32)
        q[:, :, 1:8] = np.abs(q[:, :, 1:8]) + (0 if power else 2.0 ** -12)
        got = attend(cache, batch, q, scale)
        want, tol, _ = O.attention(finite, batch, q, scale)
        assert np.all(np.abs(got - want) <= tol), (np.isnan(got).sum(), np.nanmax(np.abs(got - want)))
        assert (got[rows] == 0).all()
    # an infinite query whose every score is minus infinity, beside rows with NaN of their own
    for s in range(2):
        for t in range(int(cache.length[s]) + (rows if s == 0 else 1)):
            cache.k[0, cache.page_of(s, t), 0, t % page, 9] = O.encode([-1.0], typ)[0]
            cache.k[0, cache.page_of(s, t), 0, t % page, 1:8] = 0
    cache.upload()
    q[0, 3, 9], q[1, 5, 2] = np.inf, np.nan
    got = attend(cache, batch, q, 0.25)
    want, tol, _ = O.attention(cache, batch, np.nan_to_num(q, nan=0, posinf=0), 0.25)
    assert (got[0, 3] == 0).all() and np.isnan(got[1, 5]).all()
    keep = np.ones(q.shape[:2], bool)
    keep[0, 3] = keep[1, 5] = False
    assert np.all(np.abs(got - want)[keep] <= tol[keep])


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("length", [700, 6000])
@pytest.mark.parametrize("nats", [8, 12, 16, 20])
def test_attention_small_weights_beside_a_sink(qgl, typ, length, nats):
    """Keys far below one in every tile whose value is zero: the output is theirs alone.  A weight is within 2^-22 of
    itself or 2^-38 of the largest (F16 planes; the others within 2^-22), all of one sign here: the errors add up."""
    rng = np.random.default_rng(length + nats)
    dim, page = 64, 32
    cache = Cache(rng, [length], [1], typ=typ, kv_heads=1, page=page, dim=dim)
    batch = Batch([1])
    store(cache, batch, rng)
    z = np.full(length + 1, 0.0)
    for t in range(length + 1):
        sink = t % 32 == 7
        z[t] = O.decode(O.encode([nats if sink else rng.uniform(-1, 1)], typ), typ)[0]
        cache.put(0, 0, t, np.eye(1, dim) * z[t], np.zeros((1, dim)) if sink else rng.uniform(0.5, 1.0, (1, dim)))
    cache.upload()
    q = np.zeros((1, 2, dim), np.float32)
    q[0, :, 0] = (1.0, 0.75)
    got = attend(cache, batch, q, 1.0)
    V = np.stack([cache.token(cache.v, 0, 0, t)[0] for t in range(length + 1)])
    for h in range(2):
        s = z * float(q[0, h, 0])
        p = np.exp(s - s.max())
        want = p @ V / p.sum()
        # a score: log2 e and its product with the query (half a step each), the planes (2^-22), the product's sum (2), the
        # sum with the maximum (of |s| log2 e + 13, in 64 bits ln 2 of that); the exponential (2); then p's planes, and p
        # and its sums in fp32 with their roundings as independent
        ds = (9 * np.abs(s).max() + 11) * U
        rel = 2 * ds + 2.0 ** -22 + 4 * U * (4 + math.sqrt(length))
        tol = want * rel + (2.0 ** -38 * V.sum(0) / p.sum() if typ == F16 else 0)
        assert np.all(np.abs(got[0, h] - want) <= tol), (np.abs(got[0, h] - want).max() / want.max(), (tol / want).max())


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("length,page", [(70, 16), (9000, 64)])
def test_attention_values_near_the_types_end(qgl, typ, length, page):
    """The output is a mean of the values: it is finite where they are, however large."""
    rng = np.random.default_rng(length + 1)
    big = {F16: 6.5e4, BF16: 3.3e38, F32: 3.3e38}[typ]
    cache = Cache(rng, [length], [3], typ=typ, kv_heads=1, page=page, dim=64)
    batch = Batch([3])
    for t in range(length + 3):
        cache.put(0, 0, t, rng.standard_normal((1, 64)), big * np.concatenate([np.ones((1, 32)), rng.uniform(-1, 1, (1, 32))], 1))
    cache.upload()
    check(cache, batch, rng.standard_normal((3, 4, 64)).astype(np.float32), 0.125)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_starts_beyond_the_rows(qgl, typ, tree):
    """Row starts below the first row, of more rows than max_rows and behind the last row are cut to what there is."""
    rng = np.random.default_rng(14)
    counts, lengths = [2, 0, 5, 5], [60, 8, 40, 0]
    cache = Cache(rng, lengths, counts, typ=typ, kv_heads=2, page=16, dim=64)
    batch = Batch(counts, [O.random_tree(rng, n) if n else [] for n in counts] if tree else None, rows=14, max_rows=5)
    if tree:
        batch.parent = np.concatenate([batch.parent[:7], [-1, -1], batch.parent[7:12]]).astype(np.int32)
        batch.dparent.set(batch.parent)
    batch.dstart.set(np.array([-7, 2, 2, 9, 1 << 30], np.int32))
    batch.places = lambda: [(0, 0, 0), (1, 0, 1)] + [(2 + i, 2, i) for i in range(5)] + [(9 + i, 3, i) for i in range(5)]
    store(cache, batch, rng)
    check(cache, batch, rng.standard_normal((14, 6, 64)).astype(np.float32), 0.125)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("dim,length", [(64, 50), (128, 3000), (256, 700)])
def test_attention_nan_rows_beside_others(qgl, typ, dim, length):
    """NaN in a query, in a key and in a value that some rows see and others do not, rows that are taken up again for an
    infinite value, all in one batch over holes: each row's own answer."""
    rng = np.random.default_rng(dim)
    rows, heads, page = 8, 4, 32
    cache = Cache(rng, [length], [rows], typ=typ, kv_heads=2, page=page, dim=dim)
    parents = [-1, 0, 0, 1, 2, 2, 4, 3]      # rows below 1: 1, 3, 7; below 2: 2, 4, 5, 6
    batch = Batch([rows], [parents])
    store(cache, batch, rng)
    at = lambda place: (0, cache.page_of(0, length + place), slice(None), (length + place) % page)
    cache.k[at(1)][:, 3] = O.encode([np.nan], typ)[0]
    cache.v[at(5)][:, 2] = O.encode([np.nan], typ)[0]
    cache.v[at(4)][:, 7] = O.encode([np.inf], typ)[0]
    if length > 100:
        cache.table[0, 1] = -1
    cache.upload()
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    q[2, 1, 5] = np.nan
    got = attend(cache, batch, q, dim ** -0.5)
    want, tol, _ = O.attention(cache, batch, np.nan_to_num(q, nan=0.0), dim ** -0.5)
    assert np.isnan(got[[1, 3, 7]]).all() and np.isnan(got[2, 1]).all() and np.isnan(got[5, :, 2]).all()
    assert (got[[4, 6], :, 7] == np.inf).all()
    keep = np.ones(q.shape, bool)
    keep[[1, 3, 7]], keep[2, 1], keep[5, :, 2], keep[4, :, 7], keep[6, :, 7] = False, False, False, False, False
    assert np.all(np.abs(got[keep] - want[keep]) <= tol[keep])
