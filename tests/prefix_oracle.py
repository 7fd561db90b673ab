"""Caches whose sequences share pages, for the tests of qg_kv_prefixes and
qg_prefix_attention, and what the first of them finds, stated plainly."""
import numpy as np

from nebula_amd.qg import Device
from spec_oracle import F16, Cache, encode


class Forked(Cache):
    """Sequences given as (from, common, own): the first `common` tokens are those of sequence `from` (whole pages of
    them held together, the rest copied), `own` more follow; -1 for a sequence of its own."""

    def __init__(self, rng, family, room, *, typ=F16, layers=1, kv_heads=2, page=16, dim=64, spare=2, extra=1):
        tables, lengths, n = [], [], 0
        for (up, common, own), r in zip(family, room):
            common = min(common, lengths[up]) if up >= 0 else 0
            length = common + own
            held = tables[up][:common // page] if up >= 0 else []
            more = -(-(length + r) // page) - len(held)
            tables.append(held + list(range(n, n + more)))
            lengths.append(length)
            n += more
        super().__init__(rng, [0] * len(family), [0] * len(family), typ=typ, layers=layers, kv_heads=kv_heads, page=page, dim=dim,
                         spare=n + spare, table_pages=max(map(len, tables)) + extra)
        order = rng.permutation(self.pages)
        for b, t in enumerate(tables):
            self.table[b, :len(t)] = order[t]
        self.refs = np.bincount(self.table[self.table >= 0], minlength=self.pages).astype(np.int32)
        self.length = np.array(lengths, np.int32)
        k, v = (np.full((layers, self.pages, kv_heads, page, dim), np.nan, np.float32) for _ in range(2))
        for b, length in enumerate(lengths):
            for j in range(-(-length // page)):
                p, m = self.table[b, j], min(page, length - j * page)
                for pool in (k, v):
                    new = np.isnan(pool[0, p, 0, :m, 0])  # tokens that no earlier sequence brought
                    pool[:, p, :, :m][:, :, new] = rng.standard_normal((layers, kv_heads, int(new.sum()), dim))
        self.k, self.v = encode(k, typ), encode(v, typ)
        self.upload()


def prefixes(table, pages, page_tokens, length, counts):
    """link, shared of every sequence, pair by pair."""
    S, W = table.shape
    link, shared = np.full(S, -1, np.int32), np.zeros(S, np.int32)
    whole = [min(max(int(n), 0), W * page_tokens) // page_tokens for n in length]
    for s in range(S):
        for t in range(s):
            if counts[s] <= 0 or counts[t] <= 0:
                continue
            n = 0
            while n < min(whole[s], whole[t]) and table[s, n] == table[t, n] and 0 <= table[s, n] < pages:
                n += 1
            if n * page_tokens > shared[s]:
                link[s], shared[s] = t, n * page_tokens
    return link, shared
