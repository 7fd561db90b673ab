"""qg_qk_norm_rope, qg_softmax and qg_verify_drafts against 64-bit statements of
the same operators (spec_oracle.py)."""
import ctypes as C
import math
import sys

import numpy as np
import pytest

import spec_oracle as O
from nebula_amd import qg
from nebula_amd.qg import Device, call
from spec_oracle import BF16, F16, F32, HALF_STEP, TINY, U, Batch, Cache

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True, file=sys.stderr)


# ---------------- norm, rotation, store ----------------

# Roundings of one output: the sum of squares (4 fused steps and 6 additions, halved by the root), root, division and two
# products 10; the angle (a turn fraction in fp32) 2, sine and cosine 4, products and sum 3: 19, counted as 20.
ROPE_TOL = 20 * U


def rope_rows(rng, N, Hq, Hkv, D, gated, pad):
    """A packed projection: q heads (each followed by a gate), k heads, v heads, then unused columns."""
    Wq = 2 * D if gated else D
    x = rng.standard_normal((N, Hq * Wq + 2 * Hkv * D + pad)).astype(np.float32)
    q = x[:, :Hq * Wq].reshape(N, Hq, Wq)[:, :, :D]
    k = x[:, Hq * Wq:Hq * Wq + Hkv * D].reshape(N, Hkv, D)
    v = x[:, Hq * Wq + Hkv * D:Hq * Wq + 2 * Hkv * D].reshape(N, Hkv, D)
    dx = Device(x)
    row = x.shape[1]
    args = qg.QkRows(q=dx.p, k=dx.p + 4 * Hq * Wq, v=dx.p + 4 * (Hq * Wq + Hkv * D), q_row=row, q_head=Wq, k_row=row, k_head=D,
                     v_row=row, v_head=D, rows=N, q_heads=Hq, kv_heads=Hkv, head_dim=D, eps=1e-6)
    return args, dx, q, k, v


@pytest.mark.parametrize("D,rope,interleaved,typ,page,tree,gated", [
    (64, 64, 0, F16, 8, False, False), (128, 128, 1, BF16, 16, True, True), (128, 32, 0, F32, 64, False, True),
    (256, 64, 1, BF16, 32, True, False), (64, 8, 0, F32, 16, True, False), (256, 256, 0, F16, 1024, False, False), (128, 0, 0, F16, 16, True, False)])
def test_rope_into_cache(qgl, D, rope, interleaved, typ, page, tree, gated):
    rng = np.random.default_rng(D + rope + typ)
    counts, lengths = [3, 0, 17, 1, 5], [0, 9, 70, 1, 33]
    Hq, Hkv, layers = 5 if D == 64 else 4, 5 if D == 64 else 2, 3
    cache = Cache(rng, lengths, counts, typ=typ, layers=layers, kv_heads=Hkv, page=page, dim=D)
    cache.table[4, :] = -1          # a sequence without pages: its rows are not stored
    cache.table[3, 0] = cache.pages  # and one with an entry that is no page
    cache.upload()
    batch = Batch(counts, [O.random_tree(rng, n) if n else [] for n in counts] if tree else None, rows=sum(counts) + 2)
    N = batch.rows
    args, keep, q, k, v = rope_rows(rng, N, Hq, Hkv, D, gated, 8)
    freq = 10000.0 ** (-2 * np.arange(max(rope // 2, 1)) / max(rope, 1))
    wq, wk = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32), (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    dwq, dwk, dfreq = Device(wq), Device(wk), Device(freq)
    args.q_norm, args.k_norm, args.rope_dims, args.interleaved, args.freq = dwq.p, dwk.p, rope, interleaved, dfreq.p
    qo, ko = Device(np.full((N, Hq, D), np.nan, np.float32)), Device(np.full((N, Hkv, D), np.nan, np.float32))
    say(f"rope D={D} rope={rope} type={typ}")
    call("qk_norm_rope", qo.p, ko.p, C.byref(args), cache.ref, 1, batch.ref)
    gq, gk = qo.get(), ko.get()
    gk_cache, gv_cache = cache.dk.get(), cache.dv.get()
    want_v, left = cache.v.copy(), cache.k.copy()
    seen = np.zeros(N, bool)
    for row, s, place in batch.places():
        seen[row] = True
        L = int(cache.length[s])
        pos = L + len(batch.line(row, place)) - 1
        page_id, slot = cache.page_of(s, L + place), (L + place) % page
        for h in range(Hq):
            y, size = O.norm_rope(q[row, h], wq, 1e-6, pos, freq, rope, interleaved)
            assert np.all(np.abs(gq[row, h] - y) <= ROPE_TOL * size), (row, h, np.abs(gq[row, h] - y).max())
        for h in range(Hkv):
            y, size = O.norm_rope(k[row, h], wk, 1e-6, pos, freq, rope, interleaved)
            assert np.all(np.abs(gk[row, h] - y) <= ROPE_TOL * size)
            if page_id >= 0:
                got = O.decode(gk_cache[1, page_id, h, slot], typ)
                assert np.all(np.abs(got - y) <= ROPE_TOL * size * 1.01 + HALF_STEP[typ] * np.abs(y) + TINY[typ])
                left[1, page_id, h, slot] = gk_cache[1, page_id, h, slot]
        cache.put(1, s, L + place, np.zeros((Hkv, D)), v[row])
    want_v = cache.v
    np.testing.assert_array_equal(gv_cache.view(np.uint8), want_v.view(np.uint8))      # v as rounded, nothing else touched
    np.testing.assert_array_equal(gk_cache.view(np.uint8), left.view(np.uint8))
    assert np.isnan(gq[~seen]).all() and np.isnan(gk[~seen]).all() and seen.sum() == sum(counts)


@pytest.mark.parametrize("position", [0, 1, 98303, 1 << 20, -5])
def test_rope_without_cache_far_positions(qgl, position):
    """Angles of far positions, and the outputs in their inputs' place."""
    rng = np.random.default_rng(3)
    N, Hq, Hkv, D = 70, 3, 1, 128
    q, k = (rng.standard_normal((N, h, D)).astype(np.float32) for h in (Hq, Hkv))
    pos = (position + np.arange(N) * 3).astype(np.int32)
    freq = 1e6 ** (-2 * np.arange(64) / 128)
    dq, dk, dpos, dfreq = Device(q), Device(k), Device(pos), Device(freq)
    args = qg.QkRows(q=dq.p, k=dk.p, q_row=Hq * D, q_head=D, k_row=Hkv * D, k_head=D, rows=N, q_heads=Hq, kv_heads=Hkv, head_dim=D, eps=1e-5,
                     rope_dims=D, freq=dfreq.p, position=dpos.p)
    say(f"rope in place position={position}")
    call("qk_norm_rope", dq.p, dk.p, C.byref(args), None, 0, None)
    for got, x in ((dq.get(), q), (dk.get(), k)):
        for r in range(N):
            for h in range(x.shape[1]):
                y, size = O.norm_rope(x[r, h], None, 0, pos[r], freq, D, 0)
                assert np.all(np.abs(got[r, h] - y) <= ROPE_TOL * size)


def test_rope_many_sequences(qgl):
    """More sequences than a wave has lanes, most of them without rows."""
    rng = np.random.default_rng(9)
    counts = [int(x) for x in rng.integers(0, 3, 300)]
    lengths = [int(x) for x in rng.integers(0, 20, 300)]
    cache = Cache(rng, lengths, counts, typ=F32, kv_heads=1, page=8, dim=64)
    batch = Batch(counts)
    args, keep, q, k, v = rope_rows(rng, batch.rows, 1, 1, 64, False, 0)
    out = Device(shape=(batch.rows, 1, 64), dtype=np.float32)
    say("rope 300 sequences")
    call("qk_norm_rope", out.p, None, C.byref(args), cache.ref, 0, batch.ref)
    np.testing.assert_array_equal(out.get()[:, 0], q[:, 0])  # neither norm nor rotation: a copy
    for row, s, place in batch.places():
        cache.put(0, s, int(cache.length[s]) + place, k[row], v[row])
    np.testing.assert_array_equal(cache.dk.get().view(np.uint32), cache.k.view(np.uint32))
    np.testing.assert_array_equal(cache.dv.get().view(np.uint32), cache.v.view(np.uint32))


def norm_rope_rows(x, w, eps, pos, freq, rope, interleaved):
    """spec_oracle.norm_rope of every row and head at once."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    y, size, half = x.copy(), np.abs(x), rope // 2
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = pos.astype(np.float64)[:, None, None] * freq[:half]
    c, s = np.cos(angle), np.sin(angle)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, size


@pytest.mark.parametrize("D,Hq,Hkv,rope,interleaved,typ", [(64, 19, 2, 64, 0, F16), (64, 19, 2, 32, 1, F32), (128, 9, 2, 32, 0, BF16), (128, 9, 2, 128, 1, F16),
                                                           (256, 5, 1, 256, 0, BF16), (256, 5, 1, 64, 1, F32)])
@pytest.mark.parametrize("shape", ["chunk", "trees", "positions"])
def test_rope_of_many_rows(qgl, D, Hq, Hkv, rope, interleaved, typ, shape):
    """Batches whose waves take five groups of heads each, the last group in part: a prompt chunk beside short chains, many
    trees, and rows without a cache."""
    rng = np.random.default_rng(D + rope + typ)
    counts = [3, 1700, 1, 0, 40] if shape != "trees" else [33, 0] + [int(x) for x in rng.integers(25, 41, 52)]
    groups = -(-(Hq + Hkv * (1 if shape == "positions" else 2)) // (256 // D))
    assert sum(counts) * groups > 8192 and groups % 5
    lengths = [int(x) for x in rng.integers(0, 70, len(counts))]
    cache = Cache(rng, lengths, counts, typ=typ, layers=1, kv_heads=Hkv, page=32, dim=D, fill=False)
    batch = Batch(counts, [O.random_tree(rng, n) if n else [] for n in counts] if shape == "trees" else None, rows=sum(counts) + 3)
    N = batch.rows
    args, keep, q, k, v = rope_rows(rng, N, Hq, Hkv, D, False, 4)
    freq = 10000.0 ** (-2 * np.arange(rope // 2) / rope)
    wq, wk = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32), (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    dwq, dwk, dfreq = Device(wq), Device(wk), Device(freq)
    args.q_norm, args.k_norm, args.rope_dims, args.interleaved, args.freq = dwq.p, dwk.p, rope, interleaved, dfreq.p
    qo, ko = Device(np.full((N, Hq, D), np.nan, np.float32)), Device(np.full((N, Hkv, D), np.nan, np.float32))
    say(f"rope D={D} rows={N} {shape}")
    pos, seen = np.zeros(N, np.int32), np.zeros(N, bool)
    if shape == "positions":
        pos, seen = rng.integers(0, 200000, N).astype(np.int32), ~seen
        dpos = Device(pos)
        args.position = dpos.p
        call("qk_norm_rope", qo.p, ko.p, C.byref(args), None, 0, None)
    else:
        call("qk_norm_rope", qo.p, ko.p, C.byref(args), cache.ref, 0, batch.ref)
        for row, s, place in batch.places():
            seen[row] = True
            pos[row] = lengths[s] + len(batch.line(row, place)) - 1 if shape == "trees" else lengths[s] + place
    for got, x, w in ((qo.get(), q, wq), (ko.get(), k, wk)):
        y, size = norm_rope_rows(x, w, 1e-6, pos, freq, rope, interleaved)
        assert np.all((np.abs(got - y) <= ROPE_TOL * size)[seen]), np.argwhere((np.abs(got - y) > ROPE_TOL * size) & seen[:, None, None])[:5]
        assert np.isnan(got[~seen]).all()
    if shape == "positions":
        return
    # the cache: the keys that were given out, rounded, the values as they came, nothing else
    stored = ko.get()
    for row, s, place in batch.places():
        cache.put(0, s, lengths[s] + place, stored[row], v[row])
    for got, want in ((cache.dk.get(), cache.k), (cache.dv.get(), cache.v)):
        np.testing.assert_array_equal(got.view(np.uint8), want.view(np.uint8))


# ---------------- softmax ----------------

def softmax(x, T, out=None):
    rows, cols = x.shape
    dx = Device(x)
    do = dx if out is None else out
    n = qg.lib().qg_softmax_workspace_bytes(rows, cols)
    ws = Device(nbytes=n)
    say(f"softmax {rows}x{cols} T={T}")
    call("softmax", do.p, dx.p, rows, cols, T, ws.p, n)
    return do.get()


def softmax_oracle(x, T):
    """Values in 64 bits, and the relative error of fp32: the exponent's rounding (of the difference and of its product,
    three half steps of it), the exponential, the sum (its roundings as independent: root, four times) and the division."""
    x = x.astype(np.float64)
    z = (x - x.max(-1, keepdims=True)) / T
    e = np.exp(z)
    tol = U * (3 * np.abs(np.where(np.isfinite(z), z, 0)) + 8 + 4 * math.sqrt(x.shape[1]) / 8)
    return e / e.sum(-1, keepdims=True), tol


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 63), (5, 1000), (2, 4097), (17, 32003), (1, 151936), (300, 1025), (2, 300001), (1000, 7), (130, 20011), (129, 140003), (3, 40960), (3, 40961), (200, 70001), (140, 131072)])
@pytest.mark.parametrize("T", [0.7, 1.0, 30.0])
def test_softmax(qgl, rows, cols, T):
    rng = np.random.default_rng(rows * 7 + cols)
    x = (rng.standard_normal((rows, cols)) * 5).astype(np.float32)
    x[0, rng.integers(0, cols, cols // 3)] = -np.inf
    x[0, 0] = 1.5
    want, tol = softmax_oracle(x, T)
    for out in (None, Device(np.full((rows, cols), np.nan, np.float32))):  # in place, and elsewhere
        got = softmax(x, T, out)
        assert np.all(np.abs(got - want) <= tol * want + 2.0 ** -126), np.max(np.abs(got - want) / (tol * want + 2.0 ** -126))


@pytest.mark.parametrize("rows,cols", [(6, 5), (6, 5000), (6, 131072), (600, 4100), (130, 20001), (129, 140003), (300, 50001)])
def test_softmax_special_rows(qgl, rows, cols):
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[0] = -np.inf
    x[1, cols // 2] = np.nan
    x[2, cols - 1] = np.inf
    x[3] = np.float32(3e38) * np.sign(x[3])       # differences beyond the type's range
    x[4] = np.finfo(np.float32).min               # a mask of the lowest value
    x[5, :] = -np.inf
    x[5, cols - 1] = -2e38
    got = softmax(x, 0.5)
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and np.isnan(got[2]).all()
    np.testing.assert_allclose(got[3], np.where(x[3] == x[3].max(), 1 / (x[3] == x[3].max()).sum(), 0), rtol=1e-5)
    np.testing.assert_allclose(got[4], 1 / cols, rtol=1e-5)
    np.testing.assert_array_equal(got[5], (np.arange(cols) == cols - 1).astype(np.float32))
    want, tol = softmax_oracle(x[6:], 0.5) if rows > 6 else (np.zeros((0, cols)), 0)
    assert np.all(np.abs(got[6:] - want) <= tol * want + 2.0 ** -126)


@pytest.mark.parametrize("rows,cols", [(4, 1), (5, 4099), (2, 151937), (700, 1500), (128, 20001), (300, 50001)])
def test_softmax_greedy(qgl, rows, cols):
    """Temperature 0: one at the lowest index of the largest value."""
    rng = np.random.default_rng(cols)
    x = rng.integers(-3, 4, (rows, cols)).astype(np.float32)  # ties
    x[1 % rows] = -np.inf
    if rows > 3:
        x[3, cols // 2] = np.nan
    got = softmax(x, 0.0)
    want = (np.arange(cols) == x.argmax(-1)[:, None]).astype(np.float32)
    want[1 % rows] = 0
    if rows > 3:
        want[3] = np.nan
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("rows,cols", [(130, 131071), (140, 98305), (140, 98304), (128, 135168), (700, 20001), (300, 4097)])
def test_softmax_greedy_where_the_row_is_kept(qgl, rows, cols):
    """Temperature 0 of rows held in registers and shared memory (from value 98304 on): the largest, ties of it and NaN on
    either side of every border."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    borders = [b for b in (1024, 2048, 16384, 40960, 98304, 99328, 131072) if b < cols] + [cols]
    for r in range(rows):
        at = sorted({int(rng.choice(borders)) + int(d) for d in rng.integers(-2, 2, int(rng.integers(1, 4)))} | {int(rng.integers(0, cols))})
        x[r, [a for a in at if r % 3 and 0 <= a < cols] or [at[-1] % cols]] = 9.0
    x[1], x[2, cols - 1] = -np.inf, np.inf
    x[3] = -np.inf
    x[3, cols - 1] = -3e38
    x[4, cols - 1] = x[5, min(98304, cols - 1)] = np.nan
    x[6, :] = 0.0
    x[7, :] = -1.0
    x[7, cols - 2:] = 0.0
    for out in (None, Device(np.full((rows, cols), np.nan, np.float32))):
        got = softmax(x, 0.0, out)
        want = (np.arange(cols) == x.argmax(-1)[:, None]).astype(np.float32)
        want[1] = 0
        want[[2, 4, 5]] = np.nan
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("rows,cols", [(3, 300), (3, 5000), (3, 30000), (3, 100003), (140, 100003)])
@pytest.mark.parametrize("T,size", [(3e38, 3.4e38), (1e38, 1e38), (2.0 ** 64, 1e22), (1e19, 1e22), (2.0 ** -126, 2.0 ** -124), (1e-30, 1e-29)])
def test_softmax_temperatures_near_the_types_ends(qgl, rows, cols, T, size):
    """Values on the temperature's own scale, whose differences may pass the type's range or be below its normal numbers."""
    rng = np.random.default_rng(cols)
    x = (rng.uniform(-1, 1, (rows, cols)) * size).astype(np.float32)
    x[1] = np.where(rng.random(cols) < 0.5, -np.inf, x[1])
    x[2, :2] = np.float32(size), np.float32(-size)
    T = float(np.float32(T))
    want, tol = softmax_oracle(x, T)
    got = softmax(x, T)
    assert np.all(np.abs(got - want) <= tol * want + 2.0 ** -126), np.max(np.abs(got - want) / (tol * want + 2.0 ** -126))


# ---------------- verification ----------------

def verify(p, q, token, u, u_last, batch):
    B, cols = len(u_last), p.shape[1]
    tokens, path = (Device(np.full((B, batch.max_rows), 77, np.int32)) for _ in range(2))
    count = Device(np.full(B, 77, np.int32))
    dp, dq, dt, du, dl = Device(p), Device(q) if q is not None else None, Device(token), Device(u), Device(u_last)
    n = qg.lib().qg_verify_workspace_bytes(B, cols)
    ws = Device(np.full(n, 0xff, np.uint8))
    say(f"verify {B} sequences, {batch.rows} rows, {cols} tokens")
    call("verify_drafts", tokens.p, path.p, count.p, dp.p, dq.p if dq else None, dt.p, du.p, dl.p, cols, B, batch.ref, ws.p, n)
    return tokens.get(), path.get(), count.get()


def draft_case(rng, counts, cols, tree, greedy, noise=0.7):
    parents = [O.random_tree(rng, n) if n else [] for n in counts] if tree else None
    batch = Batch(counts, parents)
    x = rng.standard_normal((batch.rows, cols)) * 3
    soft = lambda z: (np.exp(z - z.max(-1, keepdims=True)) / np.exp(z - z.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(np.float32)
    p, q = soft(x), soft(x + noise * rng.standard_normal(x.shape))
    token = np.zeros(batch.rows, np.int32)
    for row, s, place in batch.places():
        if place == 0:
            continue
        up = row - place + (place - 1 if parents is None else parents[s][place])
        token[row] = rng.choice(np.argsort(-q[up])[:3]) if greedy else rng.choice(cols, p=q[up].astype(np.float64) / q[up].sum(dtype=np.float64))
    return batch, p, None if greedy else q, token, rng.random(batch.rows, np.float32), rng.random(len(counts), np.float32)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("counts,cols", [([1], 5), ([17], 1000), ([3, 0, 17, 1, 64], 4097), ([17] * 20, 300), ([9, 2], 32003), ([17], 151936)])
def test_verify(qgl, counts, cols, tree, greedy):
    rng = np.random.default_rng(len(counts) * 1000 + cols + tree)
    for _ in range(2 if cols > 5000 else 5):
        case = draft_case(rng, counts, cols, tree, greedy)
        for got, want in zip(verify(*case[1:], case[0]), O.verify(*case[1:], case[0])):
            np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("greedy", [False, True])
def test_verify_pieces_of_several_blocks(qgl, tree, greedy):
    """More blocks of the vocabulary in all than there are workgroups for: a piece is two of them."""
    rng = np.random.default_rng(71 + tree)
    case = draft_case(rng, [3] * 65, 131072, tree, greedy)
    case[5][:3] = 0.0, np.float32(1 - 2 ** -24), 0.5
    for got, want in zip(verify(*case[1:], case[0]), O.verify(*case[1:], case[0])):
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("cols", [262144, 262145, 300001, 600000])
def test_verify_more_pieces_than_lanes(qgl, cols, tree, greedy):
    """Sums over more than 64 pieces, some of them with nothing in them, and tokens drawn from either end."""
    rng = np.random.default_rng(cols)
    for sparse in (False, True):
        batch, p, q, token, u, last = draft_case(rng, [5, 0, 4, 3], cols, tree, greedy)
        if sparse:  # mass in a few blocks alone, before and behind the 64th
            keep = np.zeros(cols, bool)
            for at in (4096 * 3, 4096 * 63 + 4000, cols - 5):
                keep[at:at + 100] = True
            p = np.where(keep, p, 0).astype(np.float32)
            p /= p.sum(-1, keepdims=True)
            token[rng.random(len(token)) < 0.5] = cols - 3
        for lasts in (last, np.zeros(4, np.float32), np.full(4, 1 - 2 ** -24, np.float32)):
            for got, want in zip(verify(p, q, token, u, lasts, batch), O.verify(p, q, token, u, lasts, batch)):
                np.testing.assert_array_equal(got, want)


def test_verify_special_rows(qgl):
    """Equal distributions (nothing is left after a rejection), certain and impossible drafts, tokens outside the
    vocabulary, zeros and NaN, siblings with the same token."""
    cols = 40
    batch = Batch([4] * 8, [[-1, 0, 0, 1]] * 8)
    rng = np.random.default_rng(2)
    p = rng.random((32, cols)).astype(np.float32)
    p /= p.sum(-1, keepdims=True)
    q = p.copy()
    token, u, last = rng.integers(0, cols, 32).astype(np.int32), rng.random(32, np.float32), rng.random(8, np.float32)
    u[4:8] = 0.0
    q[8], p[8] = 0, 0
    p[8, 3] = 1.0                                    # certain token, never drafted
    p[12], q[12, token[13]] = np.nan, 0.5
    token[17], token[18] = -1, cols
    p[20] = 0                                         # nothing to draw from
    token[25] = token[26]
    last[6], last[7] = 0.0, np.float32(1 - 2 ** -24)
    p[28, cols // 2:] = 0                              # no probability at the end, where u_last points
    token[29] = token[30] = cols - 1
    for qq in (q, None):
        for got, want in zip(verify(p, qq, token, u, last, batch), O.verify(p, qq, token, u, last, batch)):
            np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("tree", [False, True])
def test_verify_keeps_the_targets_distribution(qgl, tree):
    """Whatever the drafts are drawn from, the first token said is distributed as the target says: 40960 draws of 6
    tokens, frequencies within five standard deviations."""
    cols, B = 6, 1024
    rng = np.random.default_rng(4)
    p = np.array([.35, .05, .25, .02, .13, .2], np.float32)
    q = np.array([.1, .3, .2, .2, .15, .05], np.float32)
    counts = np.zeros(cols)
    parents = [[-1, 0, 0, 0, 1]] * B if tree else None
    n = 5 if tree else 3
    batch = Batch([n] * B, parents)
    for _ in range(40):
        token = rng.choice(cols, (B, n), p=q / q.sum(dtype=np.float64)).astype(np.int32)
        t, path, c = verify(np.tile(p, (B * n, 1)), np.tile(q, (B * n, 1)), token.reshape(-1), rng.random(B * n, np.float32),
                            rng.random(B, np.float32), batch)
        counts += np.bincount(t[:, 0], minlength=cols)
    total = counts.sum()
    assert total == 40 * B
    assert np.all(np.abs(counts / total - p) <= 5 * np.sqrt(p * (1 - p) / total)), counts / total
