"""Several answers of one prompt, as they are made: the prompt's pages forked, the first tokens drawn, then steps that take
all of them on together (room, norm and rotation with the store, pages that are shared, attention, truncated
probabilities, verification, compaction); eager against the statements, captured and replayed, and the host
driver's stack with shared pages."""
import ctypes as C

import numpy as np
import pytest

import spec_oracle as O
from nebula_amd import qg
from nebula_amd.qg import Device, call
from prefix_oracle import prefixes
from spec_oracle import BF16, F16, F32, Batch, Cache
from test_gpu_sampling import BORDER, stays
from test_gpu_spec_pages import Model, same
from test_gpu_spec_step import HD, HK, HQ, LAYERS, WIDTH, Step, make_stack, stack_parts, step_inputs  # noqa: F401

pytestmark = pytest.mark.gpu
ASKS = [(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.02), (0.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0)]


@pytest.fixture(autouse=True)
def whatever_it_saves(qgl):
    """Small batches share their pages too."""
    before = qgl.qg_prefix_least_saving(0)
    yield
    qgl.qg_prefix_least_saving(before)


class ForkStep(Step):
    """A Step whose attention reads shared pages once and whose probabilities are truncated by each row's request."""

    def __init__(self, cache, rows, max_rows, Hq, cols, tree):
        super().__init__(cache, rows, max_rows, Hq, cols, tree)
        lib = qg.lib()
        self.pn = lib.qg_kv_prefixes_bytes(cache.ref, self.batch)
        self.prefixes, self.link, self.shared = Device(np.full(self.pn, 0xff, np.uint8)), Device(shape=(cache.B,), dtype=np.int32), Device(shape=(cache.B,), dtype=np.int32)
        self.bytes = max(self.bytes, lib.qg_prefix_attention_workspace_bytes(cache.ref, self.batch, Hq), lib.qg_sample_workspace_bytes(rows, cols))
        self.ws = Device(np.full(self.bytes, 0xff, np.uint8))
        self.asks = [ASKS[i % len(ASKS)] for i in range(rows)]
        self.arrays = [Device(np.array(v, t)) for v, t in zip(zip(*self.asks), (np.float32, np.int32, np.float32, np.float32))]
        self.sampling = qg.Sampling(*[a.p for a in self.arrays])
        self.drawn, self.logprob, self.du = Device(shape=(rows, 2), dtype=np.int32), Device(shape=(rows, 2), dtype=np.float32), Device(shape=(rows, 2), dtype=np.float32)

    def set(self, rng, counts, parents):
        flat = super().set(rng, counts, parents)
        self.du.set(rng.random((self.rows, 2), np.float32))
        return flat

    def attend(self):
        c, ws, n = self.c, self.ws.p, self.bytes
        call("kv_reserve", c.ref, self.batch, self.status.p, ws, n)
        call("kv_prefixes", self.link.p, self.shared.p, c.ref, self.batch, self.prefixes.p, self.pn)
        call("qk_norm_rope", self.q.p, None, C.byref(self.args), c.ref, 0, self.batch)
        call("prefix_attention", self.out.p, self.q.p, self.Hq, c.D ** -0.5, c.ref, 0, self.batch, self.prefixes.p, self.pn, ws, n)

    def accept(self):
        c, ws, n = self.c, self.ws.p, self.bytes
        call("sampling_softmax", self.p.p, self.x.p, self.rows, self.cols, C.byref(self.sampling), ws, n)
        call("sampling_softmax", self.pq.p, self.y.p, self.rows, self.cols, C.byref(self.sampling), ws, n)
        call("sample", self.drawn.p, self.logprob.p, self.y.p, self.rows, self.cols, 2, C.byref(self.sampling), self.du.p, ws, n)
        call("verify_drafts", self.tokens.p, self.path.p, self.count.p, self.p.p, self.pq.p, self.token.p, self.u.p, self.last.p, self.cols,
             c.B, self.batch, ws, n)
        call("kv_compact", c.ref, self.batch, self.path.p, self.count.p, c.dlength.p)

    def results(self):
        return super().results() + [d.get() for d in (self.link, self.shared, self.drawn, self.logprob)]


def forked_cache(rng, lengths, forks, **kw):
    """Sequences with tokens of their own, and forks of them (empty before)."""
    cache = Cache(rng, list(lengths) + [0] * len(forks), [0] * (len(lengths) + len(forks)), **kw)
    dst, src = Device(np.arange(len(lengths), len(lengths) + len(forks), dtype=np.int32)), Device(np.array(forks, np.int32))
    n = qg.lib().qg_kv_workspace_bytes(cache.ref)
    ws = Device(np.zeros(n, np.uint8))
    call("kv_fork", cache.ref, dst.p, src.p, len(forks), ws.p, n)
    call("sync")
    cache.table, cache.refs, cache.length = cache.dtable.get().copy(), cache.drefs.get().copy(), cache.dlength.get().copy()
    return cache


@pytest.mark.parametrize("typ,dim,page", [(F16, 64, 16), (BF16, 128, 64), (F32, 64, 8)])
@pytest.mark.parametrize("tree", [False, True])
def test_steps_of_forks(qgl, typ, dim, page, tree):
    rng = np.random.default_rng(page + typ)
    most, Hq, cols = 5, 6, 700
    cache = forked_cache(rng, [610, 40], [0, 0, 1, 0], typ=typ, kv_heads=2, page=page, dim=dim, spare=80, table_pages=100)
    B = cache.B
    model = Model(cache)
    s = ForkStep(cache, B * most, most, Hq, cols, tree)
    for step in range(3):
        counts, parents = step_inputs(rng, B, most, tree)
        s.set(rng, counts, parents)
        s.attend()
        np.testing.assert_array_equal(s.status.get(), model.reserve(counts))
        q, out = s.q.get(), s.out.get()
        # the pages as reserve left them, the rows as they were stored
        cache.table, cache.refs = cache.dtable.get().copy(), cache.drefs.get().copy()
        cache.k, cache.v = cache.dk.get().copy(), cache.dv.get().copy()
        link, shared = prefixes(cache.table, cache.pages, page, cache.length, counts)
        np.testing.assert_array_equal(s.link.get(), link)
        np.testing.assert_array_equal(s.shared.get(), shared)
        assert step or shared.max() >= 512
        batch = Batch(counts, parents, max_rows=most, rows=B * most)
        want, tol, done = O.attention(cache, batch, q, dim ** -0.5)
        assert np.all(np.abs(out - want)[done] <= tol[done])
        s.accept()
        p, pq, tokens, path, count = (d.get() for d in (s.p, s.pq, s.tokens, s.path, s.count))
        for got, xs in ((p, s.x.get()), (pq, s.y.get())):
            for r in range(s.rows):
                w, close = stays(xs[r], *s.asks[r])
                assert close or (np.abs(got[r] - w / w.sum()) <= w / w.sum() * 2.0 ** -23 + 2.0 ** -149).all(), (r, s.asks[r])
        for got, want in zip((tokens, path, count), O.verify(p, pq, s.token.get(), s.u.get(), s.last.get(), batch)):
            np.testing.assert_array_equal(got, want)
        # a token is drawn only where its probability is above 0, and its logarithm is that probability's
        drawn, logs = s.drawn.get(), s.logprob.get()
        chance = np.take_along_axis(pq.astype(np.float64), drawn.astype(np.int64), 1)
        assert (chance > 0).all()
        np.testing.assert_allclose(logs, np.log(chance), rtol=2.0 ** -22, atol=2.0 ** -22)
        cache.length = model.compact(batch, path, count)
        cache.dlength.set(cache.length)
        cache.table, cache.refs = cache.dtable.get().copy(), cache.drefs.get().copy()
        cache.k, cache.v = cache.dk.get().copy(), cache.dv.get().copy()
        model.__init__(cache)


@pytest.mark.parametrize("typ,dim", [(F16, 128), (BF16, 256), (F32, 64)])
def test_forks_captured_and_replayed(qgl, typ, dim):
    """One graph of the whole step, replayed on new rows, trees, lengths and tables, bit for bit the eager step."""
    most, Hq = 9, 4
    caches = [forked_cache(np.random.default_rng(1), [900, 0, 40], [0, 0, 2, 0], typ=typ, kv_heads=1, page=16, dim=dim, spare=120, table_pages=90)
              for _ in range(2)]
    B = caches[0].B
    steps = [ForkStep(c, B * most, most, Hq, 5000, True) for c in caches]
    rng = np.random.default_rng(2)
    counts, parents = step_inputs(rng, B, most, True)
    steps[0].set(rng, counts, parents)
    graph = C.c_void_p()
    call("graph_begin", C.byref(graph))
    steps[0].run()
    call("graph_end", graph)
    try:
        for replay in range(5):
            counts, parents = step_inputs(rng, B, most, True)
            for s in steps:
                s.set(np.random.default_rng(100 + replay), counts, parents)
            call("graph_launch", graph)
            call("sync")
            steps[1].run()
            for a, b in zip(steps[0].results(), steps[1].results()):
                np.testing.assert_array_equal(a.view(np.uint8), b.view(np.uint8))
            assert (steps[0].status.get() == 0).all() and steps[0].shared.get().max() >= 880
    finally:
        call("sync")
        qg.lib().qg_graph_destroy(graph)


def test_stack_with_shared_pages(stack_parts):  # noqa: F811
    """nm_stack_share: the stack's calls one by one give the same bits; off again, the stack is as it was; graphs follow."""
    layers, qkv, out, norms, freq = stack_parts
    h, lib = qg.host(), qg.lib()
    rng = np.random.default_rng(4)

    def cache_of():
        return forked_cache(np.random.default_rng(7), [600], [0, 0, 0], typ=F16, layers=LAYERS, kv_heads=HK, page=16, dim=HD, spare=40, table_pages=50)
    caches = [cache_of() for _ in range(3)]
    counts = [2, 1, 3, 1]
    batches = [Batch(counts) for _ in caches]
    N = sum(counts)
    h0 = rng.standard_normal((N, WIDTH)).astype(np.float32)
    n = lib.qg_kv_workspace_bytes(caches[0].ref)
    for c, b in zip(caches, batches):
        ws, status = Device(np.zeros(n, np.uint8)), Device(np.zeros(c.B, np.int32))
        call("kv_reserve", c.ref, b.ref, status.p, ws.p, n)
        assert (status.get() == 0).all()
    # call by call
    c, b, row = caches[0], batches[0], (HQ + 2 * HK) * HD
    d = [Device(h0), *[Device(shape=s, dtype=np.float32) for s in ((N, WIDTH), (N, row), (N, HQ, HD), (N, HQ, HD), (N, 10))], Device(shape=(N, 10), dtype=np.int32)]
    hid, x, p, q, a, w, ids = d
    pn, an, mn = lib.qg_kv_prefixes_bytes(c.ref, b.ref), lib.qg_prefix_attention_workspace_bytes(c.ref, b.ref, HQ), lib.qg_moe_workspace_bytes(WIDTH, 512, N)
    pre, aws, mws = Device(nbytes=pn), Device(nbytes=an), Device(nbytes=mn)
    shared = Device(np.zeros(c.B, np.int32))
    call("kv_prefixes", None, shared.p, c.ref, b.ref, pre.p, pn)
    assert shared.get().max() >= 512
    for l in range(LAYERS):
        args = qg.QkRows(q=p.p, k=p.p + 4 * HQ * HD, v=p.p + 4 * (HQ + HK) * HD, q_row=row, q_head=HD, k_row=row, k_head=HD, v_row=row, v_head=HD,
                         rows=N, q_heads=HQ, kv_heads=HK, head_dim=HD, q_norm=norms[0].p, k_norm=norms[1].p, eps=1e-6, rope_dims=HD // 2, freq=freq.p)
        call("norm", x.p, hid.p, None, WIDTH, 1, N, 0, 0, 1e-6)
        call("matmul", p.p, qkv[l].p, 12, row, WIDTH, x.p, N)
        call("qk_norm_rope", q.p, None, C.byref(args), c.ref, l, b.ref)
        call("prefix_attention", a.p, q.p, HQ, HD ** -0.5, c.ref, l, b.ref, pre.p, pn, aws.p, an)
        call("matmul", x.p, out[l].p, 12, WIDTH, HQ * HD, a.p, N)
        call("binary", hid.p, hid.p, x.p, N * WIDTH, 0)
        call("moe_forward_residual", hid.p, ids.p, w.p, None, None, None, None, N, C.byref(layers[l].desc), mws.p, mn)
    want = hid.get().copy()
    stacks = [make_stack(stack_parts, c, 17) for c in caches[1:]]
    plain = None
    try:
        def step(stack, batch, graph):
            hidden = h.nm_stack_hidden(stack)
            src = Device(h0)
            call("copy", hidden, src.p, h0.nbytes)
            assert h.nm_stack_verify(stack, batch.ref, graph) == 0, h.nm_last_error()
            call("sync")
            got = np.empty_like(h0)
            call("read", got.ctypes.data, hidden, got.nbytes)
            return got
        plain = step(stacks[0], batches[1], 1)
        assert h.nm_stack_share(stacks[0], 1) == 0, h.nm_last_error()
        for graph in (0, 1, 1, 1):
            assert np.array_equal(step(stacks[0], batches[1], graph), want)
        assert h.nm_stack_share(stacks[0], 1) == 0
        assert np.array_equal(step(stacks[0], batches[1], 1), want)
        assert h.nm_stack_share(stacks[0], 0) == 0
        assert np.array_equal(step(stacks[0], batches[1], 1), plain)
        assert np.array_equal(step(stacks[1], batches[2], 0), plain)
        # refused inside a capture, and without attention
        graph = C.c_void_p()
        call("graph_begin", C.byref(graph))
        assert h.nm_stack_share(stacks[0], 1) == -1
        lib.qg_graph_destroy(graph)
        assert h.nm_stack_share(None, 1) == -1
        bare = h.nm_stack_create((qg.MoeLayer * LAYERS)(*[L.desc for L in layers]), LAYERS, 17, 0)
        assert h.nm_stack_share(bare, 1) == -1
        h.nm_stack_destroy(bare)
    finally:
        call("sync")
        for s in stacks:
            h.nm_stack_destroy(s)
