"""Plain 64-bit statements of the speculative-step operators (include/qwen_gpu.h:
qg_qk_norm_rope, qg_tree_attention, qg_softmax, qg_verify_drafts, qg_kv_*), and the
paged cache that their tests share."""
import ctypes as C
import math

import numpy as np

from nebula_amd import qg
from nebula_amd.qg import Device

F32, F16, BF16 = 0, 1, 30
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # largest relative rounding
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}      # and below the normal numbers
U = 2.0 ** -24


def encode(x, typ):
    """The bytes of float32 values in the cache's type, rounded to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if typ == F32:
        return x
    if typ == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def decode(x, typ):
    if typ == BF16:
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


class Cache:
    """A cache with pages in random order; whatever holds no token is NaN."""

    def __init__(self, rng, lengths, room, *, typ=F16, layers=1, kv_heads=2, page=16, dim=64, spare=2, table_pages=None, fill=True):
        self.typ, self.layers, self.H, self.P, self.D = typ, layers, kv_heads, page, dim
        need = [-(-(l + r) // page) for l, r in zip(lengths, room)]
        self.pages, self.B = sum(need) + spare, len(lengths)
        self.width = table_pages or max(max(need), 1) + 1
        order = rng.permutation(self.pages)
        self.table = np.full((self.B, self.width), -1, np.int32)
        self.refs = np.zeros(self.pages, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.refs[order[:at]] = 1
        self.length = np.array(lengths, np.int32)
        shape = (layers, self.pages, kv_heads, page, dim)
        self.k, self.v = (np.full(shape, np.nan, np.float32) for _ in range(2))
        if fill:
            for b, n in enumerate(lengths):
                for t in range(n):
                    for pool in (self.k, self.v):
                        pool[:, self.table[b, t // page], :, t % page] = rng.standard_normal((layers, kv_heads, dim))
        self.k, self.v = encode(self.k, typ), encode(self.v, typ)
        self.upload()

    def upload(self):
        self.dk, self.dv = Device(self.k), Device(self.v)
        self.dtable, self.dlength, self.drefs = Device(self.table), Device(self.length), Device(self.refs)
        self.desc = qg.KvCache(k=self.dk.p, v=self.dv.p, type=self.typ, layers=self.layers, pages=self.pages, kv_heads=self.H,
                               page_tokens=self.P, head_dim=self.D, refs=self.drefs.p, table=self.dtable.p, length=self.dlength.p,
                               sequences=self.B, table_pages=self.width)
        self.ref = C.byref(self.desc)

    def page_of(self, b, t):
        if not 0 <= t < self.width * self.P:
            return -1
        p = int(self.table[b, t // self.P])
        return p if 0 <= p < self.pages else -1

    def put(self, layer, b, t, k, v):
        """Stores one token's k, v [heads, dim] in the host copy."""
        p = self.page_of(b, t)
        if p >= 0:
            self.k[layer, p, :, t % self.P] = encode(k, self.typ)
            self.v[layer, p, :, t % self.P] = encode(v, self.typ)

    def token(self, pool, layer, b, t):
        return decode(pool[layer, self.page_of(b, t), :, t % self.P], self.typ)


class Batch:
    def __init__(self, counts, parents=None, max_rows=None, rows=None):
        self.start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = rows or int(self.start[-1])
        self.max_rows = max_rows or max(max(counts), 1)
        self.parent = None
        if parents is not None:
            flat = np.array([p for seq in parents for p in seq], np.int32)
            self.parent = np.concatenate([flat, np.full(self.rows - len(flat), -1, np.int32)])
        self.dstart = Device(self.start)
        self.dparent = Device(self.parent) if self.parent is not None else None
        self.desc = qg.KvBatch(rows=self.rows, max_rows=self.max_rows, start=self.dstart.p, parent=self.dparent.p if self.dparent else None)
        self.ref = C.byref(self.desc)

    def places(self):
        """(row, sequence, place) of every row that belongs to a sequence."""
        for s in range(len(self.start) - 1):
            for i in range(min(int(self.start[s + 1] - self.start[s]), self.max_rows)):
                yield int(self.start[s]) + i, s, i

    def line(self, row, place):
        """The places on the row's way to its root, itself first."""
        if self.parent is None:
            return list(range(place, -1, -1))
        out, first = [place], row - place
        while 0 <= self.parent[first + out[-1]] < out[-1]:
            out.append(int(self.parent[first + out[-1]]))
        return out


def random_tree(rng, n, width=3):
    return [-1] + [int(rng.integers(max(0, i - width), i)) for i in range(1, n)]


def norm_rope(x, w, eps, pos, freq, rope, interleaved):
    """One head in 64 bits, and the bound's scale: |a| + |b| of each pair."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / math.sqrt((x * x).mean() + eps) * w.astype(np.float64)
    y, size = x.copy(), np.abs(x)
    half = rope // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = float(pos) * float(freq[i])
        c, s = math.cos(angle), math.sin(angle)
        y[a], y[b] = x[a] * c - x[b] * s, x[b] * c + x[a] * s
        size[a] = size[b] = abs(x[a]) + abs(x[b])
    return y, size


def attention(cache, batch, q, scale, layer=0):
    """Outputs of every row in 64 bits and the error that fp32 scores, weights and sums may leave.  Of the D
    products of a score, and the L of an output, the roundings are taken as independent: their root times four."""
    N, Hq, D = q.shape
    out, tol = np.zeros((N, Hq, D)), np.zeros((N, Hq, D))
    done = np.zeros(N, bool)
    for row, s, place in batch.places():
        L = int(cache.length[s])
        seen = [t for t in range(L) if cache.page_of(s, t) >= 0]
        seen += [L + i for i in sorted(batch.line(row, place)) if cache.page_of(s, L + i) >= 0]
        done[row] = True
        if not seen:
            continue
        K = np.stack([cache.token(cache.k, layer, s, t) for t in seen])
        V = np.stack([cache.token(cache.v, layer, s, t) for t in seen])
        for h in range(Hq):
            kh = h // (Hq // cache.H)
            x = q[row, h].astype(np.float64)
            z = K[:, kh] @ x * scale
            top = z.max()
            if top == -np.inf:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                p = np.exp(z - top)
                out[row, h] = (p[:, None] * V[:, kh]).sum(0) / p.sum()
                size = (np.abs(K[:, kh]) @ np.abs(x)).max() * abs(scale) / math.sqrt(D)
                ds = 4 * U * (math.sqrt(D) * size + 4 + 2 * np.abs(z).max())
                tol[row, h] = np.abs(V[:, kh]).max(0) * (2 * ds + 4 * U * (4 + math.sqrt(len(seen))))
    return out, tol, done


def verify(p, q, token, u, u_last, batch):
    """tokens_out, path, count by the definition, one distribution at a time."""
    B, n = len(u_last), batch.max_rows
    tokens, path, count = np.full((B, n), -1, np.int32), np.full((B, n), -1, np.int32), np.zeros(B, np.int32)
    for s in range(B):
        first, rows = int(batch.start[s]), min(int(batch.start[s + 1] - batch.start[s]), n)
        if rows <= 0:
            continue
        node, way, said = 0, [0], []
        while True:
            P = p[first + node].astype(np.float64)
            a, mass, gone, found = 0.0, 1.0, [], None
            for i in range(1, rows):
                up = i - 1 if batch.parent is None else int(batch.parent[first + i])
                x = int(token[first + i])
                if up != node or not 0 <= x < p.shape[1]:
                    continue
                if q is not None:
                    Q = q[first + node].astype(np.float64)
                    if float(u[first + i]) * Q[x] * mass < P[x] - a * Q[x]:
                        found = i
                        break
                    a += mass
                    mass = float(np.clip(P - a * Q, 0, None).sum())
                else:
                    px = 0.0 if x in gone else P[x]
                    if float(u[first + i]) * mass < px:
                        found = i
                        break
                    mass -= max(px, 0.0)
                    gone.append(x)
            if found is None:
                break
            said.append(int(token[first + found]))
            way.append(found)
            node = found
        w = P - a * q[first + node].astype(np.float64) if q is not None else P.copy()
        w[gone] = 0
        w = np.where(w > 0, w, 0)
        if not w.sum() > 0:
            w = np.where(P > 0, P, 0)
        c = np.cumsum(w)
        hit = np.nonzero((c > float(u_last[s]) * c[-1]) & (w > 0))[0]
        said.append(int(hit[0]) if len(hit) else int(np.nonzero(w > 0)[0][-1]) if (w > 0).any() else -1)
        tokens[s, :len(said)], path[s, :len(way)], count[s] = said, way, len(way)
    return tokens, path, count
