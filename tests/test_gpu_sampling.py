"""qg_sample and qg_sampling_softmax against their definition in 64 bits.

Tokens and the set that stays are whole numbers and have to be equal, but for borders that a sum in 64 bits does not decide:
where u or top-p meets a cumulative share closer than BORDER.  (A kernel may add up weights of at most 1 as whole
numbers of 2^-(62 - bits), 2^bits >= cols: off by half of one each, together below 2^(2 bits - 63) <= 2^-27 of a sum
that is at least 1 for the sizes here.)"""
import ctypes as C
import math

import numpy as np
import pytest

from nebula_amd import qg
from nebula_amd.qg import Device

pytestmark = pytest.mark.gpu
BORDER = 2.0 ** -26
# temperature, top-k, top-p, min-p
REQUESTS = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (0.6, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 50, 1.0, 0.0), (1.3, 0, 1.0, 0.05),
            (0.8, 40, 0.95, 0.05), (1.0, 0, 0.9, 0.0), (0.9, 200, 0.99, 0.0), (1.0, 1000, 0.95, 0.02), (1.0, 1, 1.0, 0.0), (2.5, 0, 0.999, 0.0),
            (1.0, 0, 0.0, 0.0), (1.0, 7, 0.5, 0.3), (1.0, 0, 1.0, 1.0), (0.05, 5000, 0.9999, 0.0), (5.0, 30000, 0.7, 0.0), (1.0, 0, 1.0, 1e-30)]


def stays(x, T, k, p, least):
    """The weights that stay in 64 bits (None: nothing can be drawn), and whether a border of top-p was too close to call."""
    x = x.astype(np.float32) + np.float32(0)
    T, p, least = (float(np.float32(v)) for v in (T, p, least))  # as the device holds them
    top = x.max() if len(x) else -np.inf
    if np.isnan(x).any() or not np.isfinite(top):
        return None, False
    order = np.argsort(-x, kind="stable")
    if not T >= 2.0 ** -126:
        w = np.zeros(len(x))
        w[order[0]] = 1
        return w, False
    T = min(T, float(np.finfo(np.float32).max))
    d = (x[order].astype(np.float64) - float(top)) / T
    v, close = np.exp(np.maximum(d, -1e4)), False
    if 0 < k < len(x):
        v[k:] = 0
    if p < 1:
        p = max(p, 0.0)
        upto = np.cumsum(v)
        before = np.concatenate([[0.0], upto[:-1]])
        gone = before >= p * upto[-1]
        gone[0] = False
        close = bool((np.abs(before - p * upto[-1])[(v > 0) & (np.arange(len(v)) > 0)] < BORDER * upto[-1]).any()) and p > 0
        v[gone] = 0
    if least > 0:
        v[v < min(least, 1.0)] = 0
    w = np.zeros(len(x))
    w[order] = v
    return w, close


class Call:
    """Rows, their requests and a workspace on the device."""

    def __init__(self, x, requests, draws=1, u=None, ask=None):
        self.x = np.ascontiguousarray(x, np.float32)
        self.rows, self.cols = self.x.shape
        self.requests = [requests[i % len(requests)] for i in range(self.rows)]
        self.dx = Device(self.x)
        cols = list(zip(*self.requests))
        self.arrays = [Device(np.array(c, t)) for c, t in zip(cols, (np.float32, np.int32, np.float32, np.float32))]
        used = ask or (True,) * 4
        self.sampling = qg.Sampling(*[a.p if on else None for a, on in zip(self.arrays, used)])
        self.ref = C.byref(self.sampling)
        self.draws = draws
        self.u = np.ascontiguousarray(u, np.float32) if u is not None else None
        self.du = Device(self.u) if u is not None else None
        self.token = Device(np.full((self.rows, draws), -7, np.int32))
        self.logprob = Device(np.full((self.rows, draws), 7, np.float32))
        self.bytes = qg.lib().qg_sample_workspace_bytes(self.rows, self.cols)
        self.ws = Device(np.full(self.bytes, 0xA5, np.uint8))

    def sample(self):
        qg.call("sample", self.token.p, self.logprob.p, self.dx.p, self.rows, self.cols, self.draws, self.ref, self.du.p, self.ws.p, self.bytes)

    def check_sample(self):
        token, logprob, unclear = self.token.get(), self.logprob.get(), 0
        for r in range(self.rows):
            w, close = stays(self.x[r], *self.requests[r])
            if w is None:
                assert (token[r] == -1).all() and np.isnan(logprob[r]).all(), r
                continue
            upto = np.cumsum(w)
            for d in range(self.draws):
                got, goal = int(token[r, d]), float(self.u[r, d]) * upto[-1]
                hit = np.nonzero((upto > goal) & (w > 0))[0]
                want = int(hit[0]) if len(hit) else int(np.nonzero(w)[0][-1])
                if close or (np.abs(upto - goal) < BORDER * upto[-1])[w > BORDER / 4].any() or self.u[r, d] == 0 and self.x.shape[1] > 1e5:
                    unclear += got != want
                    assert 0 <= got < self.cols and self.x[r, got] > -np.inf
                    continue
                assert got == want, (r, d, self.requests[r], got, want)
                # the logarithm and its rounding; the sum's part of 2^-40
                want_log = math.log(w[got] / upto[-1])
                assert abs(logprob[r, d] - want_log) <= abs(want_log) * 2.0 ** -23 + 2.0 ** -26, (r, d, logprob[r, d], want_log)
        assert unclear <= 1 + self.rows * self.draws // 50

    def check_probs(self, out):
        unclear = 0
        for r in range(self.rows):
            w, close = stays(self.x[r], *self.requests[r])
            if w is None:
                assert (out[r] == 0).all() if self.x[r].max() == -np.inf else np.isnan(out[r]).all(), r
                continue
            want = w / w.sum()
            if close and ((out[r] > 0) != (want > 1e-46)).any():
                unclear += 1
                continue
            # one rounding of a value with an error below 2^-26 of it (exponents up to 2^10 in 64 bits, the sum)
            bad = np.abs(out[r] - want) > want * (2.0 ** -24 + 2.0 ** -26) + 2.0 ** -149
            assert not bad.any(), (r, self.requests[r], np.nonzero(bad)[0][:5], out[r][bad][:5], want[bad][:5])
            assert (out[r][w == 0] == 0).all(), (r, self.requests[r])
        assert unclear <= 1 + self.rows // 50


def logits(rng, rows, cols, rounded=False, masked=False):
    x = (rng.standard_normal((rows, cols)) * 4).astype(np.float32)
    if masked:
        x[:, rng.random(cols) < 0.4] = -np.inf
        x[:, rng.integers(cols)] = 0.5
    if rounded:  # as a model in bfloat16 has them: many are equal
        x = ((x.view(np.uint32) + 0x8000) & np.uint32(0xffff0000)).view(np.float32)
        x[np.isnan(x)] = -np.inf
    return x


SIZES = [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1025, 4095, 4096, 4097, 8191, 12289, 50000, 131072, 151936]


@pytest.mark.parametrize("rounded,masked", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("cols", SIZES)
def test_sample(qgl, cols, rounded, masked):
    rng = np.random.default_rng(cols * 7 + rounded * 2 + masked)
    rows = len(REQUESTS)
    u = rng.random((rows, 3)).astype(np.float32)
    u[::3, 0] = 0
    u[1::3, 1] = np.float32(1 - 2.0 ** -24)
    c = Call(logits(rng, rows, cols, rounded, masked), REQUESTS, 3, np.minimum(u, np.float32(1 - 2.0 ** -24)))
    c.sample()
    c.check_sample()


@pytest.mark.parametrize("rounded,masked", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("cols", SIZES)
def test_probabilities(qgl, cols, rounded, masked):
    rng = np.random.default_rng(cols * 11 + rounded * 2 + masked)
    c = Call(logits(rng, len(REQUESTS), cols, rounded, masked), REQUESTS)
    out = Device(np.full(c.x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    c.check_probs(out.get())
    qg.call("sampling_softmax", c.dx.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)  # in place
    assert np.array_equal(c.dx.get(), out.get())


def special_rows(rng, cols):
    """Rows as masks, overflows and constant inputs leave them."""
    low, inf, nan = np.finfo(np.float32).min, np.inf, np.nan
    rows = [np.full(cols, -inf), np.full(cols, low), np.full(cols, 0.0), np.full(cols, 3.25), np.full(cols, -1e30), np.full(cols, np.finfo(np.float32).max)]
    for fill in (-inf, low, -1e30, -1e4):
        x = np.full(cols, fill)
        x[rng.integers(cols, size=min(cols, 9))] = rng.standard_normal(min(cols, 9)) * 3
        rows.append(x)
    x = rng.standard_normal(cols) * 1e30
    rows.append(x)
    x = np.where(rng.random(cols) < 0.5, 0.0, -0.0)   # the zeros of both signs are one value
    rows.append(x)
    x = rng.standard_normal(cols)
    x[cols // 2] = nan
    rows.append(x)
    x = rng.standard_normal(cols)
    x[cols - 1] = inf
    rows.append(x)
    x = np.full(cols, -inf)
    x[cols - 1] = nan
    rows.append(x)
    x = rng.standard_normal(cols) * 1e-3              # nearly flat
    rows.append(x)
    x = np.round(rng.standard_normal(cols))           # few values, many ties
    rows.append(x)
    x = -np.arange(cols) * 0.5                        # falls past what 64 bits hold
    rows.append(x)
    x = np.full(cols, -50.0)                          # one token far above equal ones
    x[cols // 3] = 0
    rows.append(x)
    return np.array(rows, np.float32)


@pytest.mark.parametrize("request_", range(len(REQUESTS)))
@pytest.mark.parametrize("cols", [1, 5, 64, 4097, 33000, 140000])
def test_special_rows(qgl, cols, request_):
    rng = np.random.default_rng(cols + request_)
    x = special_rows(rng, cols)
    c = Call(x, [REQUESTS[request_]], 2, (rng.random((len(x), 2)) * 0.999).astype(np.float32))
    c.sample()
    c.check_sample()
    out = Device(np.full(c.x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    c.check_probs(out.get())


@pytest.mark.parametrize("T", [2.0 ** -126, 1e-30, 1e-6, 3e-4, 1e-2, 1e6, 1e30, float(np.finfo(np.float32).max), np.inf, -1.0, np.nan, 1e-40, -0.0])
@pytest.mark.parametrize("scale", [1e-30, 4.0, 1e30])
def test_temperatures(qgl, T, scale):
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((4, 9000)) * scale).astype(np.float32)
    asks = [(T, 0, 1.0, 0.0), (T, 30, 1.0, 0.0), (T, 0, 0.8, 0.0), (T, 0, 1.0, 0.1)]
    c = Call(x, asks, 4, rng.random((4, 4)) * 0.999)
    c.sample()
    c.check_sample()
    out = Device(np.full(x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    c.check_probs(out.get())


def test_requests_that_keep_all(qgl):
    """Values that ask for nothing, whatever they are, and arrays that are not given."""
    rng = np.random.default_rng(6)
    x = logits(rng, 8, 5000)
    off = [(1.0, 0, 1.0, 0.0), (1.0, -5, 2.0, -1.0), (1.0, 5000, np.inf, np.nan), (1.0, 1 << 30, np.nan, -np.inf)]
    u = rng.random((8, 5))
    c = Call(x, off, 5, u)
    c.requests = [off[0]] * 8
    c.sample()
    c.check_sample()
    d = Call(x, [off[0]], 5, u, ask=(False,) * 4)
    d.sample()
    assert np.array_equal(c.token.get(), d.token.get()) and np.array_equal(c.logprob.get(), d.logprob.get())
    # a negative top-p keeps the largest, a min-p above 1 those that equal it
    c = Call(np.round(x), [(1.0, 0, -3.0, 0.0), (1.0, 0, 1.0, 9.0)], 5, u)
    c.sample()
    c.requests = [(1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0)] * 4
    c.check_sample()


@pytest.mark.parametrize("used", [(True, False, False, False), (False, True, False, False), (False, False, True, False), (False, False, False, True)])
def test_one_request_array(qgl, used):
    rng = np.random.default_rng(7)
    ask = tuple(v if on else off for v, on, off in zip((0.7, 33, 0.85, 0.1), used, (1.0, 0, 1.0, 0.0)))
    c = Call(logits(rng, 3, 20000), [ask], 2, rng.random((3, 2)), ask=used)
    c.sample()
    c.check_sample()


def test_rows_that_start_anywhere(qgl):
    """An odd number of columns and a start that is 4-byte aligned only; without log-probabilities."""
    rng = np.random.default_rng(8)
    x = logits(rng, 5, 12347)
    c = Call(x, REQUESTS, 64, rng.random((5, 64)))
    pad = Device(np.concatenate([[np.float32(0)], x.ravel()]).astype(np.float32))
    qg.call("sample", c.token.p, None, pad.p + 4, 5, 12347, 64, c.ref, c.du.p, c.ws.p, c.bytes)
    want = c.token.get().copy()
    c.sample()
    assert np.array_equal(c.token.get(), want)
    c.check_sample()


@pytest.mark.parametrize("rows,cols", [(1, 151936), (17, 32000), (300, 5000)])
def test_replayed(qgl, rows, cols):
    """One captured graph; logits, requests and numbers change between its replays, and other work runs between."""
    rng = np.random.default_rng(9)
    c = Call(logits(rng, rows, cols), REQUESTS, 2, rng.random((rows, 2)))
    out = Device(np.zeros((rows, cols), np.float32))
    graph = C.c_void_p()
    qg.call("graph_begin", C.byref(graph))
    c.sample()
    qg.call("sampling_softmax", out.p, c.dx.p, rows, cols, c.ref, c.ws.p, c.bytes)
    qg.call("graph_end", graph)
    for turn in range(4):
        x, u = logits(rng, rows, cols, rounded=turn % 2 == 1), rng.random((rows, 2)).astype(np.float32)
        c.dx.set(x)
        c.du.set(u)
        c.x, c.u = x, u
        asks = [REQUESTS[(i + turn) % len(REQUESTS)] for i in range(rows)]
        c.requests = asks
        for a, v in zip(c.arrays, zip(*asks)):
            a.set(np.array(v, a.x.dtype))
        qg.call("graph_launch", graph)
        qg.call("sync")
        got, probs, logs = c.token.get().copy(), out.get().copy(), c.logprob.get().copy()
        if rows <= 17:
            c.check_sample()
            c.check_probs(probs)
        c.sample()
        qg.call("sampling_softmax", out.p, c.dx.p, rows, cols, c.ref, c.ws.p, c.bytes)
        assert np.array_equal(c.token.get(), got) and np.array_equal(out.get(), probs) and np.array_equal(c.logprob.get(), logs)
    qgl.qg_graph_destroy(graph)


def test_workspace_of_more_rows(qgl):
    rng = np.random.default_rng(10)
    cols = 30000
    big = Call(logits(rng, 40, cols), REQUESTS, 1, rng.random((40, 1)))
    assert all(0 < qgl.qg_sample_workspace_bytes(r, cols) <= big.bytes for r in range(1, 41))
    big.sample()
    all_tokens = big.token.get().copy()
    for rows in (1, 3, 18, 39):
        qg.call("sample", big.token.p, None, big.dx.p, rows, cols, 1, big.ref, big.du.p, big.ws.p, big.bytes)
        assert np.array_equal(big.token.get()[:rows], all_tokens[:rows]), rows
    big.check_sample()


def test_draws_have_the_probabilities(qgl):
    """4096 draws of a row fall as qg_sampling_softmax says: every share within five standard deviations."""
    rng = np.random.default_rng(11)
    x = np.repeat(logits(rng, 1, 2000), 64, 0)
    for ask in ((0.8, 40, 0.95, 0.0), (1.5, 0, 0.7, 0.01)):
        c = Call(x, [ask], 64, rng.random((64, 64)))
        c.sample()
        out = Device(np.zeros(x.shape, np.float32))
        qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
        p, n = out.get()[0].astype(np.float64), 64 * 64
        share = np.bincount(c.token.get().ravel(), minlength=2000) / n
        assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1 / n).all()
        assert (share[p == 0] == 0).all()


@pytest.mark.parametrize("cols", [262144, 262145, 300001, 600000, 1 << 20])
def test_wide_rows(qgl, cols):
    """Rows of more pieces than waves and lanes hold one each."""
    rng = np.random.default_rng(cols)
    x = logits(rng, 9, cols, rounded=True)
    x[3] = -np.inf
    x[3, [0, 262143, cols - 1]] = [1.0, 2.0, 3.0]
    x[4] = np.sort(x[4])                                    # the largest in the last piece
    x[5] = np.sort(x[5])[::-1]
    asks = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.8, 40, 0.95, 0.05), (1.3, 1000, 0.99, 0.0),
            (1.0, 0, 1.0, 0.02), (0.0, 0, 1.0, 0.0), (1.0, 100000, 1.0, 0.0)]
    c = Call(x, asks, 4, rng.random((9, 4)))
    c.sample()
    c.check_sample()
    out = Device(np.full(x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    c.check_probs(out.get())


@pytest.mark.parametrize("rows,cols", [(256, 12289), (257, 12289), (300, 30000), (1088, 8200)])
def test_many_rows(qgl, rows, cols):
    """Enough rows that each takes half the waves, of several pieces."""
    rng = np.random.default_rng(rows + cols)
    c = Call(logits(rng, rows, cols, rounded=True), REQUESTS, 2, rng.random((rows, 2)))
    c.sample()
    c.check_sample()
    out = Device(np.full(c.x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    c.check_probs(out.get())


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("above", [5.0, 12.0, 40.0, 400.0, 3e4])
def test_peaked_rows(qgl, rows, above):
    """One token far above the others, and cuts that lie deep below it."""
    rng = np.random.default_rng(int(above))
    cols = 20011
    x = logits(rng, rows, cols)
    for r in range(rows):
        x[r, rng.integers(cols)] = x[r].max() + above
    asks = [(1.0, k, p, m) for k in (0, 2, 50, 128, 129, 500, 2000, 9000) for p in (1.0, 0.999999, 0.5) for m in (0.0, 1e-6, 1e-20)]
    c = Call(np.repeat(x, len(asks), 0) if rows == 1 else x, asks, 2, rng.random((len(asks) if rows == 1 else rows, 2)))
    c.sample()
    c.check_sample()
    out = Device(np.full(c.x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    c.check_probs(out.get())


@pytest.mark.parametrize("values", [1, 2, 7, 40, 300])
@pytest.mark.parametrize("cols", [4097, 50021])
def test_ties(qgl, cols, values):
    """Few different values: a cut among equal ones keeps the first of them."""
    rng = np.random.default_rng(values * cols)
    x = (rng.integers(values, size=(24, cols)) * 0.37).astype(np.float32)
    x[8:16] = np.sort(x[8:16], 1)
    x[16:] = -np.sort(-x[16:], 1)
    asks = [(1.0, 100, 1.0, 0.0), (1.0, 128, 1.0, 0.0), (1.0, 129, 0.9, 0.0), (0.5, 2048, 0.95, 0.0), (1.0, 2049, 1.0, 0.0), (2.0, 4000, 0.6, 0.0), (1.0, 0, 0.3, 0.0),
            (1.0, 0, 1.0, 0.5)]
    c = Call(x, asks, 3, rng.random((24, 3)))
    c.sample()
    c.check_sample()
    out = Device(np.full(x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    c.check_probs(out.get())


def test_falling_rows_and_no_chance(qgl):
    """u of 0 and just below 1 meet the first and the last token that stays."""
    rng = np.random.default_rng(14)
    u = np.tile(np.array([0, 1 - 2.0 ** -24], np.float32), (4, 1))
    for cols in (100, 9000, 40000):
        for order in (1, -1):
            x = np.sort(rng.standard_normal((4, cols)) * 3, 1)[:, ::order].astype(np.float32)
            c = Call(x, [(1.0, 30, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 700, 1.0, 0.0), (0.0, 0, 1.0, 0.0)], 2, u)
            c.sample()
            c.check_sample()


def test_two_threads(qgl):
    """Calls and graphs of two threads with workspaces of their own."""
    import threading
    rng = np.random.default_rng(15)
    calls = [Call(logits(rng, rows, cols), REQUESTS, 2, rng.random((rows, 2))) for rows, cols in ((18, 30000), (300, 9000))]
    outs = [Device(np.zeros(c.x.shape, np.float32)) for c in calls]

    def work(c, out):
        def both():
            c.sample()
            qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
        graph = C.c_void_p()
        qg.call("graph_begin", C.byref(graph))
        both()
        qg.call("graph_end", graph)
        for _ in range(5):
            both()
            qg.call("graph_launch", graph)
        qg.call("sync")
        qgl.qg_graph_destroy(graph)

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, outs)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for c, out in zip(calls, outs):
        c.check_sample()
        c.check_probs(out.get())


def test_rows_behind_two_thousand_million_values(qgl):
    """Offsets beyond 32 bits: the last rows of a large array come out as the same rows by themselves."""
    rng = np.random.default_rng(16)
    rows, cols, few = 33000, 65538, 18
    big = Device.__new__(Device)
    big.x, big.p = np.zeros(1, np.uint8), qgl.qg_alloc(rows * cols * 4)
    assert big.p
    c = Call(logits(rng, few, cols), REQUESTS, 1, rng.random((few, 1)))
    c.sample()
    qg.call("sync")
    want, wlog = c.token.get().ravel().copy(), c.logprob.get().ravel().copy()
    probs = Device(np.zeros(c.x.shape, np.float32))
    qg.call("sampling_softmax", probs.p, c.dx.p, few, cols, c.ref, c.ws.p, c.bytes)
    wprobs = probs.get().copy()
    qg.call("zero", big.p, rows * cols * 4)
    for at in (0, rows - few):
        qg.call("write", big.p + at * cols * 4, c.x.ctypes.data, c.x.nbytes)
    arrays = []
    for a in c.arrays:
        v = a.get()
        whole = np.full(rows, v[0], v.dtype)
        whole[:few] = whole[-few:] = v
        arrays.append(Device(whole))
    sampling = qg.Sampling(*[a.p for a in arrays])
    u = np.full(rows, 0.5, np.float32)
    u[:few] = u[-few:] = c.u.ravel()
    du, token, logprob = Device(u), Device(np.full(rows, -7, np.int32)), Device(np.zeros(rows, np.float32))
    n = qgl.qg_sample_workspace_bytes(rows, cols)
    ws = Device.__new__(Device)
    ws.x, ws.p = np.zeros(1, np.uint8), qgl.qg_alloc(n)
    assert ws.p
    qg.call("sample", token.p, logprob.p, big.p, rows, cols, 1, C.byref(sampling), du.p, ws.p, n)
    qg.call("sync")
    for part in (slice(0, few), slice(rows - few, rows)):
        assert np.array_equal(token.get()[part], want) and np.array_equal(logprob.get()[part], wlog)
    qg.call("sampling_softmax", big.p, big.p, rows, cols, C.byref(sampling), ws.p, n)
    got = np.zeros_like(c.x)
    for at in (0, rows - few):
        qg.call("read", got.ctypes.data, big.p + at * cols * 4, got.nbytes)
        assert np.array_equal(got, wprobs)


@pytest.mark.parametrize("value", [0.0, 3.25, -2000.0, 0.7])
@pytest.mark.parametrize("n", [4, 84, 134, 366, 1020, 2044, 4288, 40000, 100000])
def test_shares_that_whole_numbers_meet(qgl, n, value):
    """n equal values, of which top-p keeps an exact part: weights of 1 have sums without a rounding, and no border is unclear."""
    cols = n + n // 3 + 5
    x = np.full((12, cols), -np.inf, np.float32)
    rng = np.random.default_rng(n)
    for row in x:
        row[rng.choice(cols, n, replace=False)] = value
    asks = [(T, k, p, 0.0) for T in (1.0, 0.7, 3.0) for k, p in ((0, 0.5), (0, 0.25), (0, 0.75), (n // 2, 0.5))]
    c = Call(x, asks, 2, np.tile(np.array([0, 1 - 2.0 ** -24], np.float32), (12, 1)))
    c.sample()
    out = Device(np.full(x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    token, probs = c.token.get(), out.get()
    for r, (T, k, p, _) in enumerate(asks):
        kept = np.nonzero(x[r] == np.float32(value))[0][:math.ceil((k or n) * p)]  # the fewest that weigh p of all
        assert np.array_equal(np.nonzero(probs[r])[0], kept), (r, asks[r], np.count_nonzero(probs[r]), len(kept))
        assert (probs[r, kept] == np.float32(1 / len(kept))).all()
        assert token[r].tolist() == [kept[0], kept[-1]], (r, asks[r])
