"""qg_sample and qg_sampling_softmax where a draw or a top-p meets a cumulative share.

What the sums are held to: a weight's exponent x a is a product in 64 bits, below 2^b in size off by 2^(b - 54) at most, and so
is the largest value's; bins hold a weight to 2^-39 of itself, and so the largest's.  Together ln 2 2^(b - 53) + 2^-38 of a
weight: below 2^-35 for exponents below 2^18 (b = 18; |x / T| up to 2^17 and more), below 2^-37 for |x / T| up to 2^14
(b = 15).  A sum S of weights that are off by e of themselves is off by e S, and so is what it is held against: a border
counts as met within 2 e S.  There both sides are accepted, and nothing else: the token before the border or the one
behind it, a nucleus with or without the token at its end."""
import math

import numpy as np
import pytest

from nebula_amd import qg
from nebula_amd.qg import Device
from test_gpu_sampling import Call

pytestmark = pytest.mark.gpu
LD = np.longdouble


def error_of(x, T):
    far = float(np.abs(x[np.isfinite(x)].astype(np.float64)).max()) / T
    assert far * math.log2(math.e) < 2.0 ** 18
    return 2.0 ** -37 if far <= 2.0 ** 14 else 2.0 ** -35


class Exact:
    """A row in 80 bits: its tokens in falling order, their weights, and the numbers of them that may stay."""

    def __init__(self, x, T, k, p, least):
        x, T, p, least = x.astype(np.float32), LD(np.float32(T)), LD(np.float32(p)), LD(np.float32(least))
        self.order = np.argsort(-x, kind="stable")
        self.w = np.exp((x.astype(LD) - LD(x.max())) / T)
        v = self.w[self.order]
        self.e = error_of(x, float(T))
        n = int((v > 0).sum())
        if 0 < k < n:
            n = k
        low = high = n
        if p < 1:
            before = np.concatenate([[LD(0)], np.cumsum(v[:n])[:-1]])
            S = v[:n].sum()
            low = max(1, int((before < (p - 2 * self.e) * S).sum()))
            high = max(1, int((before < (p + 2 * self.e) * S).sum()))
        if least > 0:
            low, high = (min(m, int((v >= least).sum())) for m in (low, high))
        self.low, self.high = low, high
        assert high - low <= 4

    def sets(self):
        for n in range(self.low, self.high + 1):
            kept = np.zeros(len(self.w), bool)
            kept[self.order[:n]] = True
            yield kept

    def check_draw(self, token, logprob, u):
        seen = []
        for kept in self.sets():
            w = np.where(kept, self.w, LD(0))
            upto = np.cumsum(w)
            S, goal = upto[-1], LD(np.float32(u)) * upto[-1]
            may = (w > 0) & (upto > goal - 2 * self.e * S) & (upto - w <= goal + 2 * self.e * S)
            seen += np.nonzero(may)[0].tolist()
            if 0 <= token < len(w) and may[token]:
                want = float(np.log(w[token] / S))
                if abs(logprob - want) <= abs(want) * 2.0 ** -24 + 2.0 ** -34:
                    return
        raise AssertionError((token, logprob, u, sorted(set(seen))))

    def check_probs(self, out):
        for kept in self.sets():
            if np.array_equal(out > 0, kept & (self.w / self.w[kept].sum() > 2.0 ** -150)):
                want = np.where(kept, self.w, 0) / self.w[kept].sum()
                assert (np.abs(out - want) <= want * (2.0 ** -24 + 2.0 ** -34) + 2.0 ** -149).all()
                return
        raise AssertionError((np.count_nonzero(out), self.low, self.high))


def check(x, asks, u):
    """Rows x, their requests and numbers u [rows][draws]: tokens, log-probabilities and probabilities."""
    x, u = np.asarray(x, np.float32), np.asarray(u, np.float32)
    c = Call(x, asks, u.shape[1], u)
    c.sample()
    out = Device(np.full(x.shape, 7, np.float32))
    qg.call("sampling_softmax", out.p, c.dx.p, c.rows, c.cols, c.ref, c.ws.p, c.bytes)
    token, logprob, probs = c.token.get(), c.logprob.get(), out.get()
    for r in range(c.rows):
        exact = Exact(x[r], *c.requests[r])
        for d in range(c.draws):
            exact.check_draw(int(token[r, d]), float(logprob[r, d]), u[r, d])
        exact.check_probs(probs[r])


def around(u):
    """Numbers next to u, u among them, inside [0, 1)."""
    u = np.float32(u)
    near = [np.nextafter(u, np.float32(-1)), u, np.nextafter(u, np.float32(2))]
    return [float(min(max(v, np.float32(0)), np.float32(1 - 2.0 ** -24))) for v in near]


F = float.fromhex
# T, u, the numbers of two values in pieces of their own, the values: what the bins hold of the first reaches past u, what its
# tokens weigh when they are read again does not
BINS = [(1.4138240814208984, 0.3301953673362732, (200, 200), (16.25, 17.25)),
        (F("0x1.d8f3c6p-1"), F("0x1.7a630ep-3"), (496, 572), (F("0x1.bb280ap+2"), F("0x1.053e3ep+3"))),
        (F("0x1.3b9d58p+0"), F("0x1.2f1ad4p-1"), (490, 232), (F("0x1.909d34p+0"), F("0x1.038d28p+1"))),
        (F("0x1.c19ce4p-1"), F("0x1.5b37aap-3"), (769, 654), (F("-0x1.f75316p+1"), F("-0x1.32853cp+1"))),
        (F("0x1.de8206p-1"), F("0x1.9bf60ap-2"), (912, 647), (F("-0x1.72dc98p+1"), F("-0x1.1a702ap+1"))),
        (F("0x1.6e210ep-1"), F("0x1.22af8ap-2"), (417, 199), (F("-0x1.6c5948p-2"), F("0x1.ab78d8p-1")))]


@pytest.mark.parametrize("spread", [1, 3, 4])
@pytest.mark.parametrize("case", range(len(BINS)))
def test_draws_at_the_end_of_a_piece_of_bins(qgl, case, spread):
    """More equal values than lists hold, so that pieces are weighed by their bins: the end of the first piece's share."""
    T, u, counts, values = BINS[case]
    x = np.full(8192, -np.inf, np.float32)
    for i, (n, v) in enumerate(zip(counts, values)):
        x[4096 * i + 7 + spread * np.arange(n) % 4000] = v
    assert (np.isfinite(x).sum(), (x[:4096] > -np.inf).sum()) == (sum(counts), counts[0])
    check([x], [(T, 0, 1.0, 0.01)], [[u] + around(u)])


# T, u, columns, tokens and their values, no filters: weights by powers of x a and of (x - max) a
ALL = [(0.8917738199234009, 0.3943004608154297, 8192, [(5, 104582.859375), (4100, 104583.2421875)]),
       (F("0x1.28fa2ep-1"), F("0x1.ad86d6p-2"), 16384, [(106, F("0x1.3bc91ap+16")), (15370, F("0x1.3bc8fp+16")), (2469, F("0x1.3bc9c2p+16")),
                                                        (5696, F("0x1.3bc9fp+16")), (13845, F("0x1.3bc8e4p+16"))]),
       (F("0x1.38f242p+0"), F("0x1.7d75p-2"), 8192, [(3810, F("0x1.2041ap+16")), (6143, F("0x1.204286p+16")), (7796, F("0x1.204222p+16")),
                                                     (4024, F("0x1.20421ep+16")), (7203, F("0x1.204102p+16"))]),
       (F("0x1.4869a6p+0"), F("0x1.68fadep-3"), 16384, [(1807, F("0x1.93131cp+16")), (7930, F("0x1.93136p+16")), (14967, F("0x1.9313f4p+16")),
                                                        (16233, F("0x1.9313a4p+16"))]),
       (F("0x1.5ac52ep-1"), F("0x1.369746p-1"), 8192, [(8062, F("0x1.d3b784p+16")), (3458, F("0x1.d3b76ep+16")), (2576, F("0x1.d3b6bep+16")),
                                                       (3239, F("0x1.d3b6cap+16"))])]


@pytest.mark.parametrize("case", range(len(ALL)))
def test_draws_at_the_end_of_a_piece_of_all_tokens(qgl, case):
    T, u, cols, values = ALL[case]
    x = np.full(cols, -np.inf, np.float32)
    for i, v in values:
        x[i] = v
    check([x], [(T, 0, 1.0, 0.0)], [[u] + around(u)])
    # among rows enough for workgroups of half the waves
    rows = np.tile(x, (300, 1))
    check(rows[:300], [(T, 0, 1.0, 0.0)], np.tile(np.float32([[u]]), (300, 1)))


# T, top-p, the largest values, how many copies of each lie `off` lower: where the sums of the bins reach top-p is, but for
# the last bits of a sum, the end of the largest; the bin behind them is empty
EMPTY = [(1.051647424697876, 0.5, (-0.15683889389038086, -0.9144611358642578, -1.5316662788391113), 16, 2.915785789489746),
         (F("0x1.19ddeap+0"), 0.5, (F("0x1.a88afp-1"), F("-0x1.7d0cp-4"), F("-0x1.6715ep-1")), 16, F("0x1.86c01cp+1")),
         (F("0x1.5a8006p+0"), 0.25, (F("0x1.2f16p-5"), F("-0x1.48fefp-1"), F("-0x1.b632e8p+0"), F("-0x1.990b2p+1")), 96, F("0x1.2c382ep+2")),
         (F("0x1.26831p-1"), 0.25, (F("0x1.04a64p-2"), F("-0x1.171a4p-3"), F("-0x1.ee166p-2")), 48, F("0x1.9847cp+0")),
         (F("0x1.56d988p+0"), 0.25, (F("0x1.eadcp-1"), F("-0x1.cc6bp-4"), F("-0x1.0b069p+0")), 48, F("0x1.db4a68p+1")),
         (F("0x1.1247ap-1"), 0.5, (F("-0x1.a1ae4p-3"), F("-0x1.479d5p-1"), F("-0x1.298648p+0"), F("-0x1.8aa64p+0")), 32, F("0x1.db4a68p+0")),
         (F("0x1.1247ap+0"), 0.5, (F("-0x1.63c89p-1"), F("-0x1.cfc05p+0"), F("-0x1.2e959cp+1"), F("-0x1.7ec048p+1")), 32, F("0x1.db4a68p+1")),
         (F("0x1.3d8f3cp-1"), 0.25, (F("0x1.69f69p-1"), F("0x1.b84d8p-3"), F("-0x1.5d38cp-3")), 96, F("0x1.1324f4p+1"))]


@pytest.mark.parametrize("cols", [0, 4096, 9000])
@pytest.mark.parametrize("case", range(len(EMPTY)))
def test_top_p_that_ends_before_an_empty_bin(qgl, case, cols):
    T, p, top, copies, off = EMPTY[case]
    top = np.float32(top)
    x = np.concatenate([top, np.repeat(top - np.float32(off), copies)])
    if cols:
        x = np.concatenate([x, np.full(cols - len(x), -np.inf, np.float32)])
    share = np.cumsum(np.exp((top.astype(np.float64) - float(top[0])) / T))
    u = [0.0, 1 - 2.0 ** -24] + [v for s in share for v in around(s / share[-1])]
    check([x], [(T, 0, p, 0.0)], [u])
    check([x, np.roll(x, 3)], [(T, 0, p, 0.0), (T, 0, p, 1e-6)], [u, u])


@pytest.mark.parametrize("ask", [(1.0, 0, 1.0, 0.0), (0.01, 0, 1.0, 0.0), (1e-3, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 0.999, 0.0), (2.0, 0, 1.0, 1e-3), (1.0, 5000, 1.0, 0.0),
                                 (1.0, 3000, 0.9, 1e-3), (1.0, 40, 0.95, 0.0)])
@pytest.mark.parametrize("cols", [4096, 12289, 30000])
def test_draws_at_the_ends_of_pieces_and_chunks(qgl, cols, ask):
    """u next to the shares up to the ends of pieces of 4096 and of the 1024 values that are read at once."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((2, cols)) * ask[0] * 1.5
    x[1] = np.round(x[1] / ask[0] * 8) / 8 * ask[0]  # few different values: longer than any list
    x = (x + {0.01: 100, 1e-3: 90}.get(ask[0], 0)).astype(np.float32)  # |x / T| of 1e4 and 9e4
    asks = [ask] * 2
    u = []
    for row in x:
        e = Exact(row, *ask)
        w = np.where(next(e.sets()), e.w, 0)
        upto = np.cumsum(w) / w.sum()
        ends = np.unique(np.concatenate([np.arange(1024, cols, 1024), [cols]]))[-20:] - 1
        u.append([v for i in ends for v in around(upto[i])])
    n = max(map(len, u))
    check(x, asks, [v + [0.5] * (n - len(v)) for v in u])


@pytest.mark.parametrize("p", [0.3, 0.5, 0.75, 0.9, 0.99])
def test_top_p_next_to_a_sum(qgl, p):
    """Values whose sums come as near to top-p as 32 bits of it let them."""
    rng = np.random.default_rng(int(p * 100))
    x = (rng.standard_normal((12, 3000)) * np.linspace(0.3, 6, 12)[:, None]).astype(np.float32)
    asks, u = [], rng.random((12, 3)).astype(np.float32) * np.float32(0.999)
    for row in x:
        w = np.sort(np.exp(row.astype(LD) - LD(row.max())))[::-1]
        share = np.cumsum(w) / w.sum()
        asks.append((1.0, 0, float(np.float32(share[np.argmin(np.abs(share - LD(p)))])), 0.0))
    check(x, asks, u)
