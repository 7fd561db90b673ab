// Shared by the kernels of a speculative step: host checks, the sequence and
// the ancestors of a row, values of the cache's types.
#pragma once
#include "qg_internal.h"
#include "qg_kv_index.h"

enum { QG_MAX_SEQUENCES = 1024, QG_MAX_TREE = 64, QG_MAX_ROWS = 65536 };

// Host checks of what can be seen without the device; 0 or an invalid-value code.
int qg_kv_check(const qg_kv_cache *c, bool pages, KvView *v);
int qg_batch_check(const qg_kv_batch *b, bool tree, BatchView *v);
// n bytes at a and m bytes at b share an address
static inline bool qg_overlap(const void *a, size_t n, const void *b, size_t m) {
    return a && b && (uintptr_t)a < (uintptr_t)b + m && (uintptr_t)b < (uintptr_t)a + n;
}
struct QgSpan { const void *at; size_t bytes; };
// Whether a span of the first list shares an address with one of the second.
template <int N, int M>
static inline bool qg_any_overlap(const QgSpan (&a)[N], const QgSpan (&b)[M]) {
    for (const QgSpan &x : a)
        for (const QgSpan &y : b)
            if (qg_overlap(x.at, x.bytes, y.at, y.bytes)) return true;
    return false;
}
static inline size_t qg_ints(size_t n) { return 4 * n; }
static inline size_t qg_table_bytes(const KvView &c) { return qg_ints((size_t)c.sequences * c.table_pages); }

// The sequence of a row (a wave's lanes together), or -1: the last one whose
// first row is not behind it, if its rows reach that far.
QG_DEV int batch_sequence(const BatchView &b, int sequences, int row, int lane, int &first, int &n) {
    int before = 0;
    for (int s0 = 0; s0 < sequences; s0 += 64) {
        const int s = s0 + lane;
        before += __popcll(__ballot(s < sequences && b.start[s] <= row));
    }
    const int s = before - 1;
    if (s < 0) return -1;
    batch_rows(b, s, first, n);
    return row >= first && row - first < n ? s : -1;
}

// Lane i < n of a wave: the set of rows that row i of a tree descends from,
// itself included, as a bit mask; its size less one is the row's depth.  A
// parent must be an earlier row.  Pointer doubling: six steps for 64 rows.
QG_DEV unsigned long long tree_ancestors(const int *parent, int n, int lane) {
    unsigned long long m = lane < n ? 1ULL << lane : 0;
    int up = lane < n ? tree_parent(parent[lane], lane) : -1;
#pragma unroll
    for (int step = 0; step < 6; step++) {
        const int from = up < 0 ? lane : up;
        const unsigned long long a = __shfl(m, from);
        const int b = __shfl(up, from);
        if (up >= 0) { m |= a; up = b; }
    }
    return m;
}

// One value of the cache, and its store (one rounding to nearest).
template <int TYPE>
QG_DEV float kv_load(const uint8_t *p, size_t i) {
    if (TYPE == QT_F32) return ((const float *)p)[i];
    if (TYPE == QT_F16) return (float)((const _Float16 *)p)[i];
    return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
}
QG_DEV uint32_t kv_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x ? (u >> 16) | 0x40u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
QG_DEV uint32_t kv_f16(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
