"""The operators of a speculative step together, as they are used: whole steps
against the 64-bit statements, the same steps captured into one graph and
replayed, and the host driver's stack with attention (nm_stack_verify)."""
import ctypes as C
import sys

import numpy as np
import pytest

import spec_oracle as O
from nebula_amd import qg, synth
from nebula_amd.qg import Device, call
from spec_oracle import BF16, F16, F32, HALF_STEP, TINY, U, Batch, Cache
from test_gpu_spec_pages import Model, same

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True, file=sys.stderr)


class Step:
    """One layer's step over a cache, every buffer allocated once: reserve, norm and rotation with the store, attention,
    softmax of two sets of logits, verification, compaction."""

    def __init__(self, cache, rows, max_rows, Hq, cols, tree, cap=64):
        D, H, B = cache.D, cache.H, cache.B
        self.c, self.rows, self.max_rows, self.Hq, self.cols = cache, rows, max_rows, Hq, cols
        self.width = (Hq + 2 * H) * D
        self.qkv = Device(shape=(rows, self.width), dtype=np.float32)
        self.start, self.parent = Device(shape=(B + 1,), dtype=np.int32), Device(shape=(rows,), dtype=np.int32)
        self.token, self.u, self.last = Device(shape=(rows,), dtype=np.int32), Device(shape=(rows,), dtype=np.float32), Device(shape=(B,), dtype=np.float32)
        self.x, self.y = Device(shape=(rows, cols), dtype=np.float32), Device(shape=(rows, cols), dtype=np.float32)
        self.p, self.pq = Device(shape=(rows, cols), dtype=np.float32), Device(shape=(rows, cols), dtype=np.float32)
        self.q, self.out = Device(shape=(rows, Hq, D), dtype=np.float32), Device(shape=(rows, Hq, D), dtype=np.float32)
        self.tokens, self.path = Device(shape=(B, max_rows), dtype=np.int32), Device(shape=(B, max_rows), dtype=np.int32)
        self.count, self.status = Device(shape=(B,), dtype=np.int32), Device(shape=(B,), dtype=np.int32)
        self.w = [Device((1 + 0.1 * np.random.default_rng(i).standard_normal(D)).astype(np.float32)) for i in range(2)]
        self.freq = Device(1e4 ** (-2 * np.arange(D // 2) / D))
        self.desc = qg.KvBatch(rows=rows, max_rows=max_rows, start=self.start.p, parent=self.parent.p if tree else None)
        self.batch = C.byref(self.desc)
        at = self.qkv.p
        self.args = qg.QkRows(q=at, k=at + 4 * Hq * D, v=at + 4 * (Hq + H) * D, q_row=self.width, q_head=D, k_row=self.width, k_head=D,
                              v_row=self.width, v_head=D, rows=rows, q_heads=Hq, kv_heads=H, head_dim=D, q_norm=self.w[0].p, k_norm=self.w[1].p,
                              eps=1e-6, rope_dims=D, freq=self.freq.p)
        lib = qg.lib()
        sizes = [lib.qg_kv_workspace_bytes(cache.ref), lib.qg_tree_attention_workspace_bytes(cache.ref, self.batch, Hq),
                 lib.qg_softmax_workspace_bytes(rows, cols), lib.qg_verify_workspace_bytes(B, cols)]
        self.bytes = max(sizes)
        self.ws = Device(np.full(self.bytes, 0xff, np.uint8))

    def set(self, rng, counts, parents):
        self.counts = counts
        self.host_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        flat = np.full(self.rows, -1, np.int32)
        flat[:sum(counts)] = [p for q in parents for p in q]
        self.start.set(self.host_start)
        self.parent.set(flat)
        self.host_qkv = rng.standard_normal((self.rows, self.width)).astype(np.float32)
        self.qkv.set(self.host_qkv)
        x = (3 * rng.standard_normal((self.rows, self.cols))).astype(np.float32)
        self.x.set(x)
        self.y.set((x + 0.5 * rng.standard_normal(x.shape)).astype(np.float32))
        self.token.set(rng.integers(0, 12, self.rows).astype(np.int32))
        self.u.set((rng.random(self.rows) * 0.7).astype(np.float32))
        self.last.set(rng.random(self.c.B, np.float32))
        return flat

    def run(self):
        self.attend()
        self.accept()

    def attend(self):
        c, ws, n = self.c, self.ws.p, self.bytes
        call("kv_reserve", c.ref, self.batch, self.status.p, ws, n)
        call("qk_norm_rope", self.q.p, None, C.byref(self.args), c.ref, 0, self.batch)
        call("tree_attention", self.out.p, self.q.p, self.Hq, c.D ** -0.5, c.ref, 0, self.batch, ws, n)

    def accept(self):
        c, ws, n = self.c, self.ws.p, self.bytes
        call("softmax", self.p.p, self.x.p, self.rows, self.cols, 0.8, ws, n)
        call("softmax", self.pq.p, self.y.p, self.rows, self.cols, 0.8, ws, n)
        call("verify_drafts", self.tokens.p, self.path.p, self.count.p, self.p.p, self.pq.p, self.token.p, self.u.p, self.last.p, self.cols,
             c.B, self.batch, ws, n)
        call("kv_compact", c.ref, self.batch, self.path.p, self.count.p, c.dlength.p)

    def results(self):
        c = self.c
        return [d.get() for d in (self.status, self.q, self.out, self.p, self.pq, self.tokens, self.path, self.count, c.dk, c.dv, c.dtable, c.drefs,
                                  c.dlength)]


def step_inputs(rng, B, most, tree):
    counts = [int(x) for x in rng.integers(0, most + 1, B)]
    counts[0] = most
    return counts, [O.random_tree(rng, n) if tree and n else list(range(-1, n - 1)) for n in counts]


@pytest.mark.parametrize("typ,dim,page", [(F16, 64, 16), (BF16, 128, 64), (F32, 64, 8)])
@pytest.mark.parametrize("tree", [False, True])
def test_steps_against_the_statements(qgl, typ, dim, page, tree):
    rng = np.random.default_rng(page + typ)
    B, most, Hq = 4, 9, 6
    cache = Cache(rng, [70, 0, 5, 33], [0] * B, typ=typ, kv_heads=2, page=page, dim=dim, spare=60, table_pages=40)
    model = Model(cache)
    s = Step(cache, B * most, most, Hq, 300, tree)
    for step in range(3):
        counts, parents = step_inputs(rng, B, most, tree)
        s.set(rng, counts, parents)
        say(f"step {step} type={typ} rows={counts}")
        s.attend()
        np.testing.assert_array_equal(s.status.get(), model.reserve(counts))
        q, out, k, v = s.q.get(), s.out.get(), cache.dk.get(), cache.dv.get()
        batch = Batch(counts, parents, max_rows=most, rows=B * most)
        # the rows as stored, within a rounding of the 64-bit values; from here on as they are
        D, w, freq = dim, [d.get() for d in s.w], s.freq.get()
        for row, b, place in batch.places():
            L = int(cache.length[b])
            pos, page_id, slot = L + len(batch.line(row, place)) - 1, cache.page_of(b, L + place), (L + place) % page
            x = s.host_qkv[row].reshape(-1, D)
            for h in range(Hq):
                y, size = O.norm_rope(x[h], w[0], 1e-6, pos, freq, D, 0)
                assert np.all(np.abs(q[row, h] - y) <= 20 * U * size)
            for h in range(2):
                y, size = O.norm_rope(x[Hq + h], w[1], 1e-6, pos, freq, D, 0)
                got = O.decode(k[0, page_id, h, slot], typ)
                assert np.all(np.abs(got - y) <= 20 * U * size * 1.01 + HALF_STEP[typ] * np.abs(y) + TINY[typ])
            cache.put(0, b, L + place, np.zeros((2, D)), x[Hq + 2:Hq + 4])
            cache.k[0, page_id, :, slot] = k[0, page_id, :, slot]
        same(cache)
        want, tol, done = O.attention(cache, batch, q, D ** -0.5)
        assert np.all(np.abs(out - want)[done] <= tol[done])
        s.accept()
        _, _, _, p, pq, tokens, path, count, *_ = s.results()
        for got, xs in ((p, s.x.get()), (pq, s.y.get())):
            z = np.exp((xs - xs.max(-1, keepdims=True)).astype(np.float64) / np.float32(0.8))
            np.testing.assert_allclose(got, z / z.sum(-1, keepdims=True), rtol=3e-5, atol=1e-12)
        for got, want in zip((tokens, path, count), O.verify(p, pq, s.token.get(), s.u.get(), s.last.get(), batch)):
            np.testing.assert_array_equal(got, want)
        cache.length = model.compact(batch, path, count)
        same(cache)


@pytest.mark.parametrize("typ,dim", [(F16, 128), (BF16, 64), (F32, 64)])
def test_step_captured_and_replayed(qgl, typ, dim):
    """One graph of the whole step, replayed on new rows, trees, lengths and tables, with eager work in between: bit for
    bit the eager step on a cache of its own."""
    B, most, Hq = 3, 17, 4
    caches = [Cache(np.random.default_rng(1), [300, 0, 40], [0] * B, typ=typ, kv_heads=1, page=16, dim=dim, spare=80, table_pages=60) for _ in range(2)]
    steps = [Step(c, B * most, most, Hq, 5000, True) for c in caches]
    # without a captured step's side effects: the capture records, it does not run
    rng = np.random.default_rng(2)
    counts, parents = step_inputs(rng, B, most, True)
    steps[0].set(rng, counts, parents)
    graph = C.c_void_p()
    say("capture a step")
    call("graph_begin", C.byref(graph))
    steps[0].run()
    call("graph_end", graph)
    try:
        for replay in range(5):
            counts, parents = step_inputs(rng, B, most, True)
            for s in steps:
                s.set(np.random.default_rng(100 + replay), counts, parents)
            say(f"replay {replay}")
            call("graph_launch", graph)
            call("sync")
            steps[1].run()
            for a, b in zip(steps[0].results(), steps[1].results()):
                np.testing.assert_array_equal(a.view(np.uint8), b.view(np.uint8))
            assert (steps[0].status.get() == 0).all() and steps[0].count.get()[0] >= 1
    finally:
        call("sync")
        qg.lib().qg_graph_destroy(graph)


# ---------------- nm_stack_verify ----------------

WIDTH, HQ, HK, HD, LAYERS = 2048, 4, 1, 128, 2


@pytest.fixture(scope="module")
def stack_parts(qgl):
    layers = [synth.build_layer(synth.LayerSpec(seed=40 + l)) for l in range(LAYERS)]
    qkv = [Device(nbytes=(HQ + 2 * HK) * HD * qg.row_bytes(12, WIDTH)) for _ in layers]
    out = [Device(nbytes=WIDTH * qg.row_bytes(12, HQ * HD)) for _ in layers]
    for l in range(LAYERS):
        call("synth_matrix", qkv[l].p, 12, 50, l, (HQ + 2 * HK) * HD, WIDTH, 0.03)
        call("synth_matrix", out[l].p, 12, 51, l, WIDTH, HQ * HD, 0.03)
    rng = np.random.default_rng(3)
    norms = [Device((1 + 0.1 * rng.standard_normal(HD)).astype(np.float32)) for _ in range(2)]
    freq = Device(1e4 ** (-2 * np.arange(HD // 4) / (HD // 2)))
    return layers, qkv, out, norms, freq


def make_stack(parts, cache, tokens):
    layers, qkv, out, norms, freq = parts
    h = qg.host()
    stack = h.nm_stack_create((qg.MoeLayer * LAYERS)(*[L.desc for L in layers]), LAYERS, tokens, 0)
    assert stack, h.nm_last_error()
    al = (qg.AttentionLayer * LAYERS)(*[qg.AttentionLayer(qkv=qkv[l].p, out=out[l].p, qkv_type=12, out_type=12, q_norm=norms[0].p, k_norm=norms[1].p)
                                        for l in range(LAYERS)])
    a = qg.Attention(q_heads=HQ, rope_dims=HD // 2, interleaved=0, freq=freq.p, scale=HD ** -0.5)
    assert h.nm_stack_attend(stack, al, C.byref(a), cache.ref) == 0, h.nm_last_error()
    return stack


def explicit(parts, cache, batch, h0):
    """The same layers by the library's calls one by one; returns the last hidden state and the first layer's parts."""
    layers, qkv, out, norms, freq = parts
    N, row = batch.rows, (HQ + 2 * HK) * HD
    h, x, p, q, a = Device(h0), Device(shape=(N, WIDTH), dtype=np.float32), Device(shape=(N, row), dtype=np.float32), \
        Device(shape=(N, HQ, HD), dtype=np.float32), Device(shape=(N, HQ, HD), dtype=np.float32)
    ids, w = Device(shape=(N, 10), dtype=np.int32), Device(shape=(N, 10), dtype=np.float32)
    lib = qg.lib()
    n = lib.qg_tree_attention_workspace_bytes(cache.ref, batch.ref, HQ)
    m = lib.qg_moe_workspace_bytes(WIDTH, 512, N)
    ws, mws = Device(nbytes=n), Device(nbytes=m)
    first = None
    for l in range(LAYERS):
        args = qg.QkRows(q=p.p, k=p.p + 4 * HQ * HD, v=p.p + 4 * (HQ + HK) * HD, q_row=row, q_head=HD, k_row=row, k_head=HD, v_row=row, v_head=HD,
                         rows=N, q_heads=HQ, kv_heads=HK, head_dim=HD, q_norm=norms[0].p, k_norm=norms[1].p, eps=1e-6, rope_dims=HD // 2, freq=freq.p)
        call("norm", x.p, h.p, None, WIDTH, 1, N, 0, 0, 1e-6)
        call("matmul", p.p, qkv[l].p, 12, row, WIDTH, x.p, N)
        call("qk_norm_rope", q.p, None, C.byref(args), cache.ref, l, batch.ref)
        call("tree_attention", a.p, q.p, HQ, HD ** -0.5, cache.ref, l, batch.ref, ws.p, n)
        call("matmul", x.p, out[l].p, 12, WIDTH, HQ * HD, a.p, N)
        call("binary", h.p, h.p, x.p, N * WIDTH, 0)
        if l == 0:
            first = p.get(), q.get(), a.get(), h.get()
        call("moe_forward_residual", h.p, ids.p, w.p, None, None, None, None, N, C.byref(layers[l].desc), mws.p, m)
    return h.get(), first


def dequant(dev, rows, cols):
    f = Device(shape=(rows, cols), dtype=np.float32)
    call("dequant", f.p, dev.p, 12, rows, cols)
    return f.get().astype(np.float64)


def test_stack_verify(stack_parts):
    rng = np.random.default_rng(5)
    counts, lengths = [9, 5, 3], [200, 0, 17]
    make = lambda: Cache(np.random.default_rng(6), lengths, counts, typ=BF16, layers=LAYERS, kv_heads=HK, page=32, dim=HD)
    host = qg.host()
    ref, eager, graphed = make(), make(), make()
    stacks = [make_stack(stack_parts, c, 17) for c in (eager, graphed)]
    batches = [Batch(counts, [O.random_tree(np.random.default_rng(7), n) for n in counts]) for _ in range(3)]
    try:
        for step in range(4):
            N = sum(counts)
            h0 = rng.standard_normal((N, WIDTH)).astype(np.float32)
            want, first = explicit(stack_parts, ref, batches[0], h0)
            for i, stack in enumerate(stacks):
                call("write", host.nm_stack_hidden(stack), h0.ctypes.data, h0.nbytes)
                say(f"stack verify step {step} graph={i}")
                assert host.nm_stack_verify(stack, batches[1 + i].ref, i) == 0, host.nm_last_error()
                call("sync")
                got = np.empty_like(h0)
                call("read", got.ctypes.data, host.nm_stack_hidden(stack), got.nbytes)
                np.testing.assert_array_equal(got.view(np.uint32), want.view(np.uint32))
            for c in (eager, graphed):
                np.testing.assert_array_equal(c.dk.get(), ref.dk.get())
                np.testing.assert_array_equal(c.dv.get(), ref.dv.get())
            if step == 0:  # the attention block itself, in 64 bits
                p, q, a, h1 = first
                x = synth.rmsnorm(h0).astype(np.float64)
                wq = dequant(stack_parts[1][0], (HQ + 2 * HK) * HD, WIDTH)
                np.testing.assert_allclose(p, x @ wq.T, rtol=1e-4, atol=1e-4)
                ref.k, ref.v = ref.dk.get(), ref.dv.get()
                o, tol, done = O.attention(ref, batches[0], q, HD ** -0.5)
                assert done.all() and np.all(np.abs(a - o) <= tol)
                wo = dequant(stack_parts[2][0], WIDTH, HQ * HD)
                np.testing.assert_allclose(h1, h0 + a.reshape(N, -1).astype(np.float64) @ wo.T, rtol=1e-4, atol=1e-4)
            # the next step: other lengths and other trees in the same arrays
            lengths2 = np.array([180 + step, step, 20 - step], np.int32)
            for c in (ref, eager, graphed):
                c.dlength.set(lengths2)
                c.length = lengths2.copy()
            tree = np.concatenate([O.random_tree(np.random.default_rng(20 + step), n) for n in counts]).astype(np.int32)
            for b in batches:
                b.dparent.set(tree)
                b.parent = tree
    finally:
        for stack in stacks:
            host.nm_stack_destroy(stack)


def test_stack_verify_other_batches(stack_parts):
    """A chain after a tree, other row counts, other arrays with the same row count: each its own graph."""
    rng = np.random.default_rng(8)
    make = lambda: Cache(np.random.default_rng(9), [60, 7], [17, 17], typ=F16, layers=LAYERS, kv_heads=HK, page=16, dim=HD)
    host = qg.host()
    ref, mine = make(), make()
    stack = make_stack(stack_parts, mine, 17)
    try:
        for counts, parents in (([5, 4], [O.random_tree(rng, 5), O.random_tree(rng, 4)]), ([5, 4], None), ([1, 0], None), ([0, 17], None),
                                ([5, 4], [O.random_tree(rng, 5), O.random_tree(rng, 4)])):
            batch = Batch(counts, parents)
            h0 = rng.standard_normal((batch.rows, WIDTH)).astype(np.float32)
            want, _ = explicit(stack_parts, ref, batch, h0)
            call("write", host.nm_stack_hidden(stack), h0.ctypes.data, h0.nbytes)
            say(f"stack verify rows={counts}")
            assert host.nm_stack_verify(stack, batch.ref, 1) == 0, host.nm_last_error()
            call("sync")
            got = np.empty_like(h0)
            call("read", got.ctypes.data, host.nm_stack_hidden(stack), got.nbytes)
            np.testing.assert_array_equal(got.view(np.uint32), want.view(np.uint32))
        # refusals: more rows than the stack holds, no batch
        big = Batch([10, 8])
        assert host.nm_stack_verify(stack, big.ref, 0) == -1 and b"rows" in host.nm_last_error()
        assert host.nm_stack_verify(stack, None, 0) == -1
    finally:
        host.nm_stack_destroy(stack)


def test_stack_verify_rows_of_no_sequence(stack_parts):
    """Rows behind the last sequence take the MoE alone, whatever the batch before had in their places."""
    rng = np.random.default_rng(11)
    host = qg.host()
    cache = Cache(np.random.default_rng(12), [50], [9], typ=F16, layers=LAYERS, kv_heads=HK, page=16, dim=HD)
    stack = make_stack(stack_parts, cache, 9)
    try:
        h0 = rng.standard_normal((9, WIDTH)).astype(np.float32)
        for counts, graph in (([9], 0), ([4], 0), ([9], 1), ([4], 1)):
            batch = Batch(counts, max_rows=9, rows=9)
            call("write", host.nm_stack_hidden(stack), h0.ctypes.data, h0.nbytes)
            say(f"rows {counts} of 9, graph={graph}")
            assert host.nm_stack_verify(stack, batch.ref, graph) == 0, host.nm_last_error()
            call("sync")
            got = np.empty_like(h0)
            call("read", got.ctypes.data, host.nm_stack_hidden(stack), got.nbytes)
            if counts == [4]:
                call("write", host.nm_stack_hidden(stack), h0.ctypes.data, h0.nbytes)
                assert host.nm_stack_forward(stack, 9, 0) == 0, host.nm_last_error()
                call("sync")
                alone = np.empty_like(h0)
                call("read", alone.ctypes.data, host.nm_stack_hidden(stack), alone.nbytes)
                # sums of a few thousand fp32 terms, in an order that other rows may change
                np.testing.assert_allclose(got[4:], alone[4:], rtol=1e-4, atol=1e-4)
                assert np.abs(got[:4] - alone[:4]).max() > 0.01
    finally:
        host.nm_stack_destroy(stack)


@pytest.mark.parametrize("use_graph", [0, 1])
@pytest.mark.parametrize("used", [False, True])
def test_stack_inside_a_callers_capture(stack_parts, use_graph, used):
    """Room for the rows, the stack and the new lengths in one graph of the caller's, replayed on new rows, trees and
    lengths: bit for bit the same calls on a cache of its own.  used: the stack has graphs of its own, for other arrays."""
    host, lib = qg.host(), qg.lib()
    counts = [5, 4]
    make = lambda: Cache(np.random.default_rng(31), [40, 7], [0, 0], typ=F16, layers=LAYERS, kv_heads=HK, page=16, dim=HD, spare=24, table_pages=12)
    caches = [make(), make()]
    stacks = [make_stack(stack_parts, c, 17) for c in caches]
    batches = [Batch(counts, [O.random_tree(np.random.default_rng(32), n) for n in counts]) for _ in caches]
    n = lib.qg_kv_workspace_bytes(caches[0].ref)
    ws, status, path, count = ([f() for _ in caches] for f in (lambda: Device(nbytes=n), lambda: Device(shape=(2,), dtype=np.int32),
                                                              lambda: Device(shape=(2, 5), dtype=np.int32), lambda: Device(shape=(2,), dtype=np.int32)))

    def step(i, graphed):
        c, b = caches[i], batches[i]
        call("kv_reserve", c.ref, b.ref, status[i].p, ws[i].p, n)
        assert host.nm_stack_verify(stacks[i], b.ref, graphed) == 0, host.nm_last_error()
        call("kv_compact", c.ref, b.ref, path[i].p, count[i].p, c.dlength.p)
        assert host.nm_stack_forward(stacks[i], sum(counts), graphed) == 0, host.nm_last_error()

    rng = np.random.default_rng(33)
    graph = C.c_void_p()
    try:
        if used:  # on rows of their own, whose pages are let go again
            other = Batch(counts)
            lengths = Device(np.array([40, 7], np.int32))
            for i in range(2):
                call("kv_reserve", caches[i].ref, other.ref, status[i].p, ws[i].p, n)
                assert host.nm_stack_verify(stacks[i], other.ref, 1) == 0 and host.nm_stack_forward(stacks[i], 3, 1) == 0, host.nm_last_error()
                call("kv_truncate", caches[i].ref, lengths.p)
            call("sync")
        assert lib.qg_graph_recording() == 0
        say(f"capture a stack, use_graph={use_graph} used={used}")
        call("graph_begin", C.byref(graph))
        assert lib.qg_graph_recording() == 1
        step(0, use_graph)
        call("graph_end", graph)
        assert lib.qg_graph_recording() == 0
        for replay in range(4):
            h0 = rng.standard_normal((sum(counts), WIDTH)).astype(np.float32)
            tree = np.concatenate([O.random_tree(rng, k) for k in counts]).astype(np.int32)
            ways = [[0] + sorted(rng.choice(np.arange(1, k), 2, replace=False)) for k in counts]
            for i in range(2):
                call("write", host.nm_stack_hidden(stacks[i]), h0.ctypes.data, h0.nbytes)
                batches[i].dparent.set(tree)
                path[i].set(np.array([w + [-1, -1] for w in ways], np.int32))
                count[i].set(np.array([3, 1 + replay % 3], np.int32))
            say(f"replay {replay}")
            call("graph_launch", graph)
            call("sync")
            step(1, 0)
            call("sync")
            got = [np.empty_like(h0) for _ in range(2)]
            for i in range(2):
                call("read", got[i].ctypes.data, host.nm_stack_hidden(stacks[i]), h0.nbytes)
            np.testing.assert_array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
            for name in ("dk", "dv", "dtable", "drefs", "dlength"):
                np.testing.assert_array_equal(*(getattr(c, name).get().view(np.uint8) for c in caches))
            np.testing.assert_array_equal(caches[0].dlength.get(), [40 + 3 * (replay + 1), 7 + sum(1 + k % 3 for k in range(replay + 1))])
            assert (status[0].get() == 0).all() and np.isfinite(got[0]).all()
    finally:
        if not lib.qg_graph_recording():
            call("sync")
        lib.qg_graph_destroy(graph)
        for stack in stacks:
            host.nm_stack_destroy(stack)


def test_stack_attend_refusals(stack_parts):
    layers, qkv, out, norms, freq = stack_parts
    host = qg.host()
    cache = Cache(np.random.default_rng(1), [5], [5], typ=F16, layers=LAYERS, kv_heads=HK, page=16, dim=HD)
    stack = host.nm_stack_create((qg.MoeLayer * LAYERS)(*[L.desc for L in layers]), LAYERS, 4, 0)
    al = (qg.AttentionLayer * LAYERS)(*[qg.AttentionLayer(qkv=qkv[l].p, out=out[l].p, qkv_type=12, out_type=12) for l in range(LAYERS)])
    good = dict(q_heads=HQ, rope_dims=HD // 2, interleaved=0, freq=freq.p, scale=1.0)
    try:
        batch = Batch([2])
        assert host.nm_stack_verify(stack, batch.ref, 0) == -1  # no attention yet
        for kw in (dict(q_heads=0), dict(rope_dims=12), dict(rope_dims=HD + 8), dict(freq=None)):
            a = qg.Attention(**(good | kw))
            assert host.nm_stack_attend(stack, al, C.byref(a), cache.ref) == -1, kw
        a = qg.Attention(**good)
        one = qg.KvCache.from_buffer_copy(cache.desc)
        one.layers = 1
        assert host.nm_stack_attend(stack, al, C.byref(a), C.byref(one)) == -1
        assert host.nm_stack_attend(stack, None, C.byref(a), cache.ref) == -1
        assert host.nm_stack_attend(stack, al, C.byref(a), cache.ref) == 0
        assert host.nm_stack_attend(stack, al, C.byref(a), cache.ref) == -1  # once
    finally:
        host.nm_stack_destroy(stack)


def test_two_threads_at_once(qgl):
    """Two threads, each with its own cache, workspace and outputs: what each gets alone."""
    import threading
    jobs = []
    for i in range(2):
        rng = np.random.default_rng(70 + i)
        cache = Cache(rng, [900, 10], [0, 0], typ=F16, kv_heads=1, page=16, dim=64, spare=20, table_pages=80)
        s = Step(cache, 18, 9, 4, 3000, True)
        counts, parents = step_inputs(rng, 2, 9, True)
        s.set(rng, counts, parents)
        jobs.append(s)
    alone = []
    for s in jobs:
        s.run()
        alone.append(s.results()[1:8])
        s.c.dlength.set(s.c.length)
    errors = []

    def work(s, want):
        try:
            for _ in range(10):
                s.run()
                for a, b in zip(s.results()[1:8], want):
                    np.testing.assert_array_equal(a.view(np.uint8), b.view(np.uint8))
                s.c.dlength.set(s.c.length)
        except BaseException as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, alone)]
    say("two threads")
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
