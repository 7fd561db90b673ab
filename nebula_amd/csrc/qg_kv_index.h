// The paged cache and its batches as kernels see them (qg_kv_cache, qg_kv_batch
// of include/qwen_gpu.h), and the reads that keep every index inside them
// whatever tables, lengths, row starts and parents hold.  Plain C++ for the
// device and the host: the same functions are tested without a GPU.
#pragma once
#include <stddef.h>
#include <stdint.h>
#ifdef __HIPCC__
#define KV_FN static __device__ __host__ __forceinline__
#else
#define KV_FN static inline
#endif

struct KvView {
    uint8_t *k, *v;
    int *refs, *table, *length;
    int type, layers, pages, heads, shift, dim, sequences, table_pages;  // page_tokens == 1 << shift
};
struct BatchView {
    const int *start, *parent;
    int rows, max_rows;
};

KV_FN int kv_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
KV_FN int kv_capacity(const KvView &c) { return c.table_pages << c.shift; }
KV_FN int kv_length(const KvView &c, int s) { return kv_clamp(c.length[s], 0, kv_capacity(c)); }
// The rows of sequence s: first and number, inside the batch whatever start holds.
KV_FN void batch_rows(const BatchView &b, int s, int &first, int &n) {
    first = kv_clamp(b.start[s], 0, b.rows);
    n = kv_clamp(b.start[s + 1], first, b.rows) - first;
    n = n < b.max_rows ? n : b.max_rows;
}
// The page of position t (any int) of sequence s, or -1.
KV_FN int kv_page(const KvView &c, int s, int t) {
    if (t < 0 || t >= kv_capacity(c)) return -1;
    const int p = c.table[(size_t)s * c.table_pages + (t >> c.shift)];
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}
// Whether tokens of a page (or -1) belong to more than one table entry, as far as the
// cache says (refs may be NULL): then they may not be written.
KV_FN bool kv_shared(const KvView &c, int page) { return page >= 0 && c.refs && c.refs[page] > 1; }
// Element offset of token `slot` (0..page_tokens-1) of a page.
KV_FN size_t kv_at(const KvView &c, int layer, int page, int head, int slot) {
    return ((((size_t)layer * c.pages + page) * c.heads + head) << c.shift | (unsigned)slot) * c.dim;
}
// The row that row i of a tree continues, or -1: it must come earlier.
KV_FN int tree_parent(int parent, int i) { return parent >= 0 && parent < i ? parent : -1; }
