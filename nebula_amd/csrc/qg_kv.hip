// Pages of the cache (qg_kv_* of include/qwen_gpu.h): reserve with copy on
// write, fork, truncate, the move of accepted rows, page copies.  All counts
// live on the device and every call is a fixed number of kernels without a
// host read, so a step that forks, reserves and compacts can be captured.
// Which page is taken never depends on the order in which workgroups run: free
// pages are those with no holder, taken in ascending order.
#include "qg_kv.h"

int qg_kv_check(const qg_kv_cache *c, bool pages, KvView *v) {
    if (!c || !c->k || !c->v || !c->table || !c->length || (pages && !c->refs)) return hipErrorInvalidValue;
    if ((((uintptr_t)c->k | (uintptr_t)c->v) & 15) || (((uintptr_t)c->table | (uintptr_t)c->length | (uintptr_t)c->refs) & 3))
        return hipErrorInvalidValue;
    if (c->type != QT_F32 && c->type != QT_F16 && c->type != QT_BF16) return hipErrorInvalidValue;
    if (c->layers < 1 || c->layers > 65536 || c->pages < 1 || c->pages > 1 << 30 || c->kv_heads < 1 || c->kv_heads > 128) return hipErrorInvalidValue;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return hipErrorInvalidValue;
    if (c->page_tokens < 8 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1))) return hipErrorInvalidValue;
    if (c->sequences < 1 || c->sequences > QG_MAX_SEQUENCES || c->table_pages < 1) return hipErrorInvalidValue;
    if ((int64_t)c->table_pages * c->page_tokens > 1LL << 28) return hipErrorInvalidValue;
    const size_t size = (size_t)c->kv_heads * c->page_tokens * c->head_dim * (c->type == QT_F32 ? 4 : 2);
    if ((size_t)c->layers > (((size_t)1 << 46) / size) / (size_t)c->pages) return hipErrorInvalidValue;
    if (v) {
        int shift = 0;
        while (1 << shift < c->page_tokens) shift++;
        *v = KvView{(uint8_t *)c->k, (uint8_t *)c->v, c->refs, c->table, c->length, c->type, c->layers, c->pages, c->kv_heads, shift,
                    c->head_dim, c->sequences, c->table_pages};
    }
    return hipSuccess;
}

int qg_batch_check(const qg_kv_batch *b, bool tree, BatchView *v) {
    if (!b || !b->start || ((uintptr_t)b->start & 3) || ((uintptr_t)b->parent & 3)) return hipErrorInvalidValue;
    if (b->rows < 1 || b->rows > QG_MAX_ROWS || b->max_rows < 1 || b->max_rows > b->rows) return hipErrorInvalidValue;
    if ((tree || b->parent) && b->max_rows > QG_MAX_TREE) return hipErrorInvalidValue;
    if (v) *v = BatchView{b->start, b->parent, b->rows, b->max_rows};
    return hipSuccess;
}

namespace {

QG_DEV void let_go(const KvView &c, int page) {
    if ((unsigned)page < (unsigned)c.pages) atomicSub(&c.refs[page], 1);
}

__global__ __launch_bounds__(256) void kv_truncate_kernel(KvView c, const int *new_length) {
    const int s = blockIdx.x;
    int n = kv_length(c, s);
    if (new_length) n = min(n, max(new_length[s], 0));
    const int keep = (n + (1 << c.shift) - 1) >> c.shift;
    int *row = c.table + (size_t)s * c.table_pages;
    for (int j = keep + threadIdx.x; j < c.table_pages; j += 256) {
        const int page = row[j];
        if (page != -1) { let_go(c, page); row[j] = -1; }
    }
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0) c.length[s] = n;
}

// Fork in two kernels, first half: pair i's source row as it is before the call, and one more
// holder for each of its pages.  ws: [n][table_pages + 2] (use, length, pages).
__global__ __launch_bounds__(256) void kv_fork_stage_kernel(KvView c, const int *dst, const int *src, int n, int *ws) {
    const int i = blockIdx.x, d = dst[i], from = src[i];
    int *at = ws + (size_t)i * (c.table_pages + 2);
    bool bad = (unsigned)d >= (unsigned)c.sequences || (unsigned)from >= (unsigned)c.sequences || d == from;
    for (int j = i + 1 + threadIdx.x; j < n; j += 256)
        bad |= dst[j] == d && (unsigned)src[j] < (unsigned)c.sequences && src[j] != d;
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) at[0] = !bad;
    if (bad) return;
    const int len = kv_length(c, from), keep = (len + (1 << c.shift) - 1) >> c.shift;
    if (threadIdx.x == 0) at[1] = len;
    for (int j = threadIdx.x; j < c.table_pages; j += 256) {
        int page = j < keep ? c.table[(size_t)from * c.table_pages + j] : -1;
        if ((unsigned)page >= (unsigned)c.pages) page = -1;
        if (page >= 0) atomicAdd(&c.refs[page], 1);
        at[2 + j] = page;
    }
}
// Second half: the destination lets go of its own pages and takes the staged ones.
__global__ __launch_bounds__(256) void kv_fork_kernel(KvView c, const int *dst, const int *ws) {
    const int *at = ws + (size_t)blockIdx.x * (c.table_pages + 2);
    if (!at[0]) return;
    const int d = dst[blockIdx.x];
    int *row = c.table + (size_t)d * c.table_pages;
    for (int j = threadIdx.x; j < c.table_pages; j += 256) {
        let_go(c, row[j]);
        row[j] = at[2 + j];
    }
    if (threadIdx.x == 0) c.length[d] = at[1];
}

// Both halves for few pairs and entries, by one workgroup that holds them in registers
// between; its holder counts pass through one CU.  One / two kernels: 1 pair x 64 pages
// 3.7 / 6.3 us, 8 x 512 5.2 / 7.1, 32 x 64 5.9 / 7.0, but 64 x 16 7.6 / 7.0, 16 x 512 8.5 / 6.2.
constexpr int FORK_PAIRS = 32, FORK_HELD = 4;
__global__ __launch_bounds__(1024) void kv_fork_small_kernel(KvView c, const int *dst, const int *src, int n) {
    __shared__ int s_dst[FORK_PAIRS], s_src[FORK_PAIRS], s_len[FORK_PAIRS];
    const int tid = threadIdx.x, all = n * c.table_pages;
    if (tid < n) { s_dst[tid] = dst[tid]; s_src[tid] = src[tid]; }
    __syncthreads();
    int len = -1;  // -1: the pair is left out
    if (tid < n) {
        const int d = s_dst[tid], from = s_src[tid];
        bool bad = (unsigned)d >= (unsigned)c.sequences || (unsigned)from >= (unsigned)c.sequences || d == from;
        for (int j = tid + 1; j < n; j++) bad |= s_dst[j] == d && (unsigned)s_src[j] < (unsigned)c.sequences && s_src[j] != d;
        if (!bad) len = kv_length(c, from);
        s_len[tid] = len;
    }
    __syncthreads();
    int page[FORK_HELD], old[FORK_HELD], at[FORK_HELD];
#pragma unroll
    for (int k = 0; k < FORK_HELD; k++) {
        const int e = k * 1024 + tid;
        page[k] = old[k] = at[k] = -1;
        if (e >= all) continue;
        const int i = e / c.table_pages, j = e - i * c.table_pages, tokens = s_len[i];
        if (tokens < 0) continue;
        at[k] = s_dst[i] * c.table_pages + j;
        old[k] = c.table[at[k]];
        if (j < (tokens + (1 << c.shift) - 1) >> c.shift) page[k] = c.table[s_src[i] * c.table_pages + j];
    }
    __syncthreads();  // tables and lengths are read, in every wave
#pragma unroll
    for (int k = 0; k < FORK_HELD; k++) {
        if (at[k] < 0) continue;
        const bool held = (unsigned)page[k] < (unsigned)c.pages;
        if (held) atomicAdd(&c.refs[page[k]], 1);
        let_go(c, old[k]);
        c.table[at[k]] = held ? page[k] : -1;
    }
    if (len >= 0) c.length[s_dst[tid]] = len;
}

// Inclusive sum over the 1024 threads of a workgroup; s_sum[16] is scratch.
QG_DEV int block_scan(int v, int *s_sum, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    __syncthreads();
    if (lane == 63) s_sum[wave] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        const int x = s_sum[w];
        if (w < wave) before += x;
        total += x;
    }
    return v + before;
}

// Reserve, one workgroup (its sums run over all sequences and over the free
// pages in order); 16 lanes look at a sequence's entries.  An entry needs a
// page if it is empty, or if its page is held elsewhere too.  The second kind
// is marked in the table as -2 - page while the sequences are counted, so that
// every sequence judges by the holders before the call.  Pages are taken for
// the whole batch or not at all: a sequence may keep a shared page only because
// the others get copies of theirs.
// Eight dependent reads in a row bound it: 9 us for 64 sequences (12.5 with a wave
// per sequence).
// ws: the copies for kv_cow_kernel, number and (source, destination) pairs, then
// the free pages found.
__global__ __launch_bounds__(1024) void kv_reserve_kernel(KvView c, BatchView b, int *status, int *ws) {
    __shared__ int s_len[QG_MAX_SEQUENCES], s_rows[QG_MAX_SEQUENCES], s_page[QG_MAX_SEQUENCES], s_need[QG_MAX_SEQUENCES], s_sum[16];
    __shared__ int s_rank[QG_MAX_SEQUENCES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = 1 << c.shift;
    int *copies = ws + 2, *free_pages = copies + 2 * c.sequences;
    // each sequence's rows, and the page with room behind its tokens
    int st = 0, mine = -1;
    if (tid < c.sequences) {
        int first, rows;
        batch_rows(b, tid, first, rows);
        const int len = kv_length(c, tid);
        if (rows > kv_capacity(c) - len) { st = 2; rows = 0; }
        if (rows && (len & (P - 1))) mine = kv_page(c, tid, len);
        s_len[tid] = len;
        s_rows[tid] = rows;
        s_page[tid] = mine;
    }
    __syncthreads();
    // of the batch's sequences that share a page no other holds, the first keeps it
    bool copied = false;
    if (mine >= 0) {
        const int held = c.refs[mine];
        if (held > 1) {
            int same = 0;
            bool before = false;
            for (int j = 0; j < c.sequences; j++)
                if (s_page[j] == mine) { same++; before |= j < tid; }
            copied = before || same < held;
        }
    }
    __syncthreads();
    if (tid < c.sequences) s_page[tid] = copied;
    __syncthreads();
    // 16 lanes per sequence, four sequences per wave: what one waits for, all wait for
    const int part = lane >> 4, l16 = lane & 15;
    auto ours = [&](bool x) { return (unsigned)(__ballot(x) >> (16 * part)) & 0xffffu; };  // of the sequence's 16 lanes
    for (int s0 = 0; s0 < c.sequences; s0 += 64) {
        const int s = s0 + wave * 4 + part;
        const bool live = s < c.sequences;
        const int len = live ? s_len[s] : 0, rows = live ? s_rows[s] : 0, here = len >> c.shift;
        const int end = rows ? (len + rows + P - 1) >> c.shift : here;
        int need = 0;
        for (int j = here + l16; __any(j < end); j += 16) {
            bool take = false;
            if (j < end) {
                int *entry = c.table + (size_t)s * c.table_pages + j;
                const int page = *entry;
                const bool none = (unsigned)page >= (unsigned)c.pages;
                take = none || (j == here && (len & (P - 1)) ? s_page[s] != 0 : c.refs[page] > 1);
                if (take) *entry = none ? -1 : -2 - page;
            }
            need += __popc(ours(take));
        }
        if (live && l16 == 0) s_need[s] = need;
    }
    __syncthreads();
    int total;
    const int need = tid < c.sequences ? s_need[tid] : 0;
    const int upto = block_scan(need, s_sum, total);
    // the first `total` free pages in ascending order, 16 of the pool per thread and round
    int found = 0;
    for (int p0 = 0; p0 < c.pages && found < total; p0 += 16384) {
        unsigned mask = 0;
        int held[16];
#pragma unroll
        for (int i = 0; i < 16; i++) held[i] = c.refs[min(p0 + tid * 16 + i, c.pages - 1)];
#pragma unroll
        for (int i = 0; i < 16; i++) mask |= p0 + tid * 16 + i < c.pages && held[i] == 0 ? 1u << i : 0u;
        int sum;
        int at = found + block_scan(__popc(mask), s_sum, sum) - __popc(mask);
        for (; mask && at < total; mask &= mask - 1) free_pages[at++] = p0 + tid * 16 + __ffs(mask) - 1;
        found += sum;
    }
    if (tid < c.sequences) {
        if (s_rows[tid] && total > found) st = 1;
        status[tid] = st;
        s_page[tid] = upto - need;  // the sequence's first page in the list
    }
    // a copied page is its sequence's first
    int n_copies;
    const int rank = block_scan(copied, s_sum, n_copies);
    if (tid < c.sequences) s_rank[tid] = rank - 1;
    if (tid == 0) ws[0] = total <= found ? n_copies : 0;
    __syncthreads();  // free_pages and copies written above are read or written by other waves below
    const bool served = total <= found;
    for (int s0 = 0; s0 < c.sequences; s0 += 64) {
        const int s = s0 + wave * 4 + part;
        const bool live = s < c.sequences && s_need[s];
        const int len = live ? s_len[s] : 0, here = len >> c.shift, end = live ? (len + s_rows[s] + P - 1) >> c.shift : here;
        int from = live ? s_page[s] : 0;
        for (int j = here + l16; __any(j < end); j += 16) {
            int *entry = c.table + (size_t)s * c.table_pages + j;
            const int mark = j < end ? *entry : 0;
            const bool take = mark < 0;
            const unsigned all = ours(take);
            if (take && served) {
                const int page = free_pages[from + __popc(all & ((1u << l16) - 1))];
                *entry = page;
                c.refs[page] = 1;
                if (mark < -1) {
                    atomicSub(&c.refs[-2 - mark], 1);
                    if (j == here && (len & (P - 1))) { copies[2 * s_rank[s]] = -2 - mark; copies[2 * s_rank[s] + 1] = page; }
                }
            } else if (take && mark < -1) {
                *entry = -2 - mark;
            }
            from += __popc(all);
        }
    }
}

// One layer's page, k (blockIdx.z even) or v, in 16-byte pieces.
QG_DEV void copy_page(const KvView &c, int dst, int src, int layer, bool v, int part, int parts) {
    const size_t bytes = ((size_t)c.heads << c.shift) * c.dim * (c.type == QT_F32 ? 4 : 2);
    uint8_t *base = (v ? c.v : c.k) + (size_t)layer * c.pages * bytes;
    const uint4 *from = (const uint4 *)(base + src * bytes);
    uint4 *to = (uint4 *)(base + dst * bytes);
    for (size_t i = (size_t)part * 256 + threadIdx.x; i < bytes / 16; i += (size_t)parts * 256) to[i] = from[i];
}
// The copies that reserve listed: 56 pages of 1 MB over 8 layers in 11 to 13 us (117 MB read
// and written; forks of one page read it from the caches).
__global__ __launch_bounds__(256) void kv_cow_kernel(KvView c, const int *ws, int parts) {
    const int per = 2 * c.layers * parts;  // of one page: layers, k and v, parts
    const long all = (long)ws[0] * per;
    for (long i = blockIdx.x; i < all; i += gridDim.x) {
        const int copy = (int)(i / per), x = (int)(i % per);
        copy_page(c, ws[3 + 2 * copy], ws[2 + 2 * copy], x / parts >> 1, x / parts & 1, x % parts, parts);
    }
}
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(KvView c, const int *dst, const int *src, int n) {
    const int i = blockIdx.x, d = dst[i], s = src[i];
    bool bad = (unsigned)d >= (unsigned)c.pages || (unsigned)s >= (unsigned)c.pages;
    for (int j = threadIdx.x; j < n; j += 256) bad |= src[j] == d || (j > i && dst[j] == d);
    if (__syncthreads_or(bad)) return;
    for (int k = blockIdx.z; k < 2 * c.layers; k += gridDim.z) copy_page(c, d, s, k >> 1, k & 1, blockIdx.y, gridDim.y);
}

// The accepted rows of a sequence move to the front of its new rows.  A thread
// owns one 16-byte column of one head, layer and side and carries it through
// all moves, so no two threads meet; a path ascends, so row i never lands
// where a later one starts, and eight rows may be read before the first is written.
// Moves are few: 16 sequences x 48 layers take 4.8 us, a launch and four reads.
// new_length NULL: written by kv_length_kernel, where the workgroups of a
// sequence read the lengths that it replaces.
// The rows of a sequence's path that are followed; lane i's row p, and the pages that it
// comes from and goes to.  A path ends where it does not ascend, and at a page that others
// hold: reserve found no room for a copy, and the row was not stored.  Nor do rows count
// behind the last one that has pages: without room there are none from some row on.
QG_DEV int path_rows(const KvView &c, const BatchView &b, const int *path, const int *count, int s, int len, int lane, int &p, int &from, int &to) {
    int first, n;
    batch_rows(b, s, first, n);
    const int keep = min(max(count[s], 0), n);
    p = lane < keep ? path[(size_t)s * b.max_rows + lane] : -1;
    const int before = __shfl_up(p, 1);
    const bool ok = lane < keep && p < n && p > (lane ? before : -1);
    from = ok ? kv_page(c, s, len + p) : -1;
    to = ok ? kv_page(c, s, len + lane) : -1;
    const bool shared = kv_shared(c, from) || kv_shared(c, to);
    const unsigned long long fault = ~__ballot(ok && !shared);
    const unsigned long long held = __ballot(from >= 0 && to >= 0) & (fault ? (fault & -fault) - 1 : ~0ULL);
    return held ? 64 - __clzll(held) : 0;
}
__global__ __launch_bounds__(64) void kv_length_kernel(KvView c, BatchView b, const int *path, const int *count, int *new_length) {
    int p, from, to;
    const int len = kv_length(c, blockIdx.x), upto = path_rows(c, b, path, count, blockIdx.x, len, threadIdx.x, p, from, to);
    if (threadIdx.x == 0) new_length[blockIdx.x] = len + upto;
}
__global__ __launch_bounds__(256) void kv_compact_kernel(KvView c, BatchView b, const int *path, const int *count, int *new_length) {
    __shared__ size_t s_from[QG_MAX_TREE], s_to[QG_MAX_TREE];
    __shared__ int s_moves;
    const int s = blockIdx.y, lane = threadIdx.x & 63, es = c.type == QT_F32 ? 4 : 2;
    if (threadIdx.x < 64) {
        const int len = kv_length(c, s);
        int p, from, to;
        const int upto = path_rows(c, b, path, count, s, len, lane, p, from, to);
        const int slot = (1 << c.shift) - 1;
        const bool both = lane < upto && p != lane && from >= 0 && to >= 0;
        const unsigned long long all = __ballot(both);
        if (both) {
            const int at = __popcll(all & ((1ULL << lane) - 1));
            s_from[at] = kv_at(c, 0, from, 0, (len + p) & slot) * es;
            s_to[at] = kv_at(c, 0, to, 0, (len + lane) & slot) * es;
        }
        if (lane == 0) {
            s_moves = __popcll(all);
            if (blockIdx.x == 0 && new_length) new_length[s] = len + upto;
        }
    }
    __syncthreads();
    const int moves = s_moves;
    if (!moves) return;
    const int pieces = c.dim * es / 16;
    const size_t layer = (((size_t)c.pages * c.heads) << c.shift) * c.dim * es, head = ((size_t)c.dim << c.shift) * es;
    const int all = 2 * c.layers * c.heads * pieces;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256) {
        const int piece = i % pieces, h = i / pieces % c.heads, l = i / pieces / c.heads;
        uint8_t *base = (l & 1 ? c.v : c.k) + (l >> 1) * layer + h * head + piece * 16;
        for (int m0 = 0; m0 < moves; m0 += 8) {
            uint4 x[8];
#pragma unroll
            for (int m = 0; m < 8; m++) x[m] = *(const uint4 *)(base + s_from[min(m0 + m, moves - 1)]);
#pragma unroll
            for (int m = 0; m < 8; m++)
                if (m0 + m < moves) *(uint4 *)(base + s_to[m0 + m]) = x[m];
        }
    }
}

size_t page_parts(const KvView &c) {  // workgroups per page, layer and side: 16 pieces of 16 bytes per thread
    const size_t bytes = ((size_t)c.heads << c.shift) * c.dim * (c.type == QT_F32 ? 4 : 2);
    const size_t n = (bytes / 16 + 4095) / 4096;
    return n < 64 ? n : 64;
}
unsigned layer_parts(const KvView &c) { return 2 * c.layers < 4096 ? 2 * c.layers : 4096; }
}  // namespace

extern "C" {

size_t qg_kv_workspace_bytes(const qg_kv_cache *cache) {
    if (qg_kv_check(cache, false, nullptr)) return 0;
    const size_t fork = (size_t)cache->sequences * (cache->table_pages + 2), reserve = 2 + 2 * (size_t)cache->sequences + cache->pages;
    return 4 * (fork > reserve ? fork : reserve);
}

int qg_kv_reserve(const qg_kv_cache *cache, const qg_kv_batch *batch, int *status, void *ws, size_t ws_bytes) {
    KvView c;
    BatchView b;
    if (qg_kv_check(cache, true, &c) || qg_batch_check(batch, false, &b)) return hipErrorInvalidValue;
    if (!status || !ws || (((uintptr_t)status | (uintptr_t)ws) & 3) || ws_bytes < qg_kv_workspace_bytes(cache)) return hipErrorInvalidValue;
    const size_t S = c.sequences;
    const QgSpan cached[3] = {{c.table, qg_table_bytes(c)}, {c.length, qg_ints(S)}, {c.refs, qg_ints(c.pages)}}, starts[1] = {{b.start, qg_ints(S + 1)}},
                 said[1] = {{status, qg_ints(S)}}, space[1] = {{ws, qg_kv_workspace_bytes(cache)}};
    if (qg_any_overlap(said, cached) || qg_any_overlap(said, starts) || qg_any_overlap(said, space) || qg_any_overlap(space, cached) ||
        qg_any_overlap(space, starts) || qg_any_overlap(starts, cached))
        return hipErrorInvalidValue;
    kv_reserve_kernel<<<1, 1024, 0, qg_stream()>>>(c, b, status, (int *)ws);
    const long work = 2L * c.layers * page_parts(c) * c.sequences;
    kv_cow_kernel<<<(unsigned)(work < 8192 ? work : 8192), 256, 0, qg_stream()>>>(c, (const int *)ws, (int)page_parts(c));
    return hipGetLastError();
}

int qg_kv_fork(const qg_kv_cache *cache, const int *dst, const int *src, int n, void *ws, size_t ws_bytes) {
    KvView c;
    if (qg_kv_check(cache, true, &c)) return hipErrorInvalidValue;
    if (!dst || !src || n < 1 || n > c.sequences || !ws || ws_bytes < qg_kv_workspace_bytes(cache) ||
        (((uintptr_t)dst | (uintptr_t)src | (uintptr_t)ws) & 3))
        return hipErrorInvalidValue;
    const QgSpan pairs[2] = {{dst, qg_ints(n)}, {src, qg_ints(n)}}, space[1] = {{ws, qg_kv_workspace_bytes(cache)}},
                 cached[3] = {{c.table, qg_table_bytes(c)}, {c.length, qg_ints(c.sequences)}, {c.refs, qg_ints(c.pages)}};
    if (qg_any_overlap(pairs, cached) || qg_any_overlap(pairs, space) || qg_any_overlap(space, cached)) return hipErrorInvalidValue;
    if (n <= FORK_PAIRS && (long)n * c.table_pages <= FORK_HELD * 1024) {
        kv_fork_small_kernel<<<1, 1024, 0, qg_stream()>>>(c, dst, src, n);
        return hipGetLastError();
    }
    kv_fork_stage_kernel<<<n, 256, 0, qg_stream()>>>(c, dst, src, n, (int *)ws);
    kv_fork_kernel<<<n, 256, 0, qg_stream()>>>(c, dst, (const int *)ws);
    return hipGetLastError();
}

int qg_kv_truncate(const qg_kv_cache *cache, const int *new_length) {
    KvView c;
    if (qg_kv_check(cache, true, &c) || ((uintptr_t)new_length & 3)) return hipErrorInvalidValue;
    const QgSpan given[1] = {{new_length, qg_ints(c.sequences)}}, lengths[1] = {{c.length, qg_ints(c.sequences)}},
                 others[2] = {{c.table, qg_table_bytes(c)}, {c.refs, qg_ints(c.pages)}};
    if ((new_length != c.length && qg_any_overlap(given, lengths)) || qg_any_overlap(given, others)) return hipErrorInvalidValue;
    kv_truncate_kernel<<<c.sequences, 256, 0, qg_stream()>>>(c, new_length);
    return hipGetLastError();
}

int qg_kv_compact(const qg_kv_cache *cache, const qg_kv_batch *batch, const int *path, const int *count, int *new_length) {
    KvView c;
    BatchView b;
    if (qg_kv_check(cache, false, &c) || qg_batch_check(batch, true, &b)) return hipErrorInvalidValue;
    if (!path || !count || !new_length || (((uintptr_t)path | (uintptr_t)count | (uintptr_t)new_length) & 3)) return hipErrorInvalidValue;
    const bool own = new_length == cache->length;
    // a sequence's first workgroup writes its new length while the others read what the path is made of
    const size_t S = c.sequences;
    const QgSpan written[1] = {{new_length, qg_ints(S)}}, lengths[1] = {{c.length, qg_ints(S)}},
                 read[5] = {{path, qg_ints(S * b.max_rows)}, {count, qg_ints(S)}, {b.start, qg_ints(S + 1)}, {c.table, qg_table_bytes(c)}, {c.refs, qg_ints(c.pages)}};
    if ((!own && qg_any_overlap(written, lengths)) || qg_any_overlap(written, read)) return hipErrorInvalidValue;
    const long all = 2L * c.layers * c.heads * (c.dim * (c.type == QT_F32 ? 4 : 2) / 16), blocks = (all + 255) / 256;
    kv_compact_kernel<<<dim3((unsigned)(blocks < 1024 ? blocks : 1024), c.sequences), 256, 0, qg_stream()>>>(c, b, path, count,
                                                                                                          own ? nullptr : new_length);
    if (own) kv_length_kernel<<<c.sequences, 64, 0, qg_stream()>>>(c, b, path, count, new_length);
    return hipGetLastError();
}

int qg_kv_copy_pages(const qg_kv_cache *cache, const int *dst, const int *src, int n) {
    KvView c;
    if (qg_kv_check(cache, false, &c)) return hipErrorInvalidValue;
    if (!dst || !src || n < 1 || n > 4096 || (((uintptr_t)dst | (uintptr_t)src) & 3)) return hipErrorInvalidValue;
    kv_copy_pages_kernel<<<dim3(n, (unsigned)page_parts(c), layer_parts(c)), 256, 0, qg_stream()>>>(c, dst, src, n);
    return hipGetLastError();
}

}  // extern "C"
