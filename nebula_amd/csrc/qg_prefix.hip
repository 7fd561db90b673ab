// Attention of a batch whose sequences begin with the same pages
// (qg_kv_prefixes, qg_prefix_attention of include/qwen_gpu.h).
//
// Forked sequences hold one page of a common prompt in several tables.  Each
// sequence hangs on the earlier one that it has the most leading pages in common
// with, which makes a tree of sequences, and the places where sequences leave one
// another cut their tokens into segments: a run of keys that the same sequences
// see.  A segment's rows, of all its sequences, share one read of its keys; what
// a row sees is the segments on its way to the root, whose partial results are
// joined as the parts of one sequence are (o = sum p v, l = sum p, m = max per part).
// In the order in which the tree is walked, longest common part first, a segment's
// sequences lie next to each other, so that its rows are a range.
#include "qg_attention.h"
#include "qg_lanes.h"
#include "qg_prefix_index.h"

namespace {

// ------------------------------------------------------------------------
// Which sequences begin with the same pages: a wave per sequence.  Bound by dependent
// reads (a length, an entry of every earlier sequence, the pages in common): 1024
// sequences of up to 80 pages 13 us, 64 of 98304 tokens 6.  Each earlier sequence that has more in common than those
// before it is one more such round: where every sequence branches from the one before it at a later page, this and the plan
// take 51 us for 64 sequences, 233 for 256 and 1360 for 1024 (from one text, at one place, 9, 19 and 27).
// ------------------------------------------------------------------------
QG_DEV int whole_pages(const KvView &c, int s) { return kv_length(c, s) >> c.shift; }
QG_DEV int table_page(const KvView &c, int s, int j) {
    const int p = c.table[(size_t)s * c.table_pages + j];
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}
// Leading pages that sequences s and t have in common, of `most`.
QG_DEV int common_pages(const KvView &c, int s, int t, int most, int lane) {
    constexpr int EACH = 8;  // of a lane at once
    for (int j0 = 0; j0 < most; j0 += 64 * EACH) {
        int x[EACH], y[EACH];
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            const int j = min(j0 + 64 * k + lane, most - 1);
            x[k] = c.table[(size_t)s * c.table_pages + j];
            y[k] = c.table[(size_t)t * c.table_pages + j];
        }
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            const int j = j0 + 64 * k + lane;
            const unsigned long long not_same = __ballot(j >= most || x[k] != y[k] || (unsigned)x[k] >= (unsigned)c.pages);
            if (not_same) return min(j0 + 64 * k + (int)__builtin_ctzll(not_same), most);
        }
    }
    return most;
}
// Sequence s by a wave.
QG_DEV void link_sequence(const KvView &c, const BatchView &b, const PrefixView &v, int *link, int *shared, int s, int lane) {
    int first, n, best = 0, with = -1;
    batch_rows(b, s, first, n);
    const int whole = whole_pages(c, s);
    // an earlier sequence has more in common than the best so far only if its page there is the same
    for (int t0 = 0; n > 0 && t0 < s && best < whole;) {
        const int t = min(t0 + lane, s - 1);
        int f, m;
        batch_rows(b, t, f, m);
        const int p = table_page(c, s, best), length = whole_pages(c, t), q = table_page(c, t, best);
        const unsigned long long all = __ballot(t0 + lane < s && m > 0 && length > best && p >= 0 && q == p);
        if (!all) { t0 += 64; continue; }
        const int l = __builtin_ctzll(all), u = t0 + l, x = common_pages(c, s, u, min(whole, __builtin_amdgcn_readlane(length, l)), lane);
        if (x > best) { best = x; with = u; }
        t0 = u + 1;
    }
    if (lane == 0) {
        const int tokens = best << c.shift;
        v.link[s] = with;
        v.shared[s] = tokens;
        if (link) link[s] = with;
        if (shared) shared[s] = tokens;
    }
}
__global__ __launch_bounds__(256) void prefix_link_kernel(KvView c, BatchView b, PrefixView v, int *link, int *shared) {
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (s < c.sequences) link_sequence(c, b, v, link, shared, s, threadIdx.x & 63);
}

// ------------------------------------------------------------------------
// Segments, by one workgroup or wave, a thread per sequence.  Sorted by the sequence that they hang on, and by
// falling common part there, the ones that leave it behind some token are a run, and what a segment needs of
// its siblings are sums over runs.
// ------------------------------------------------------------------------
// Common parts count in steps of a quantum: shorter segments would cost more than
// they save (8 sequences of 2048 tokens, 8 layers: 128 and 256 196 and 198 us, 1024 218;
// two levels of 8 x 8: 69 and 69, 77).  It is doubled until the rows of all shared segments together are few
// enough for the partial results that a workspace holds.
//
// Nothing is shared where all of it together saves less than `least` bytes of reads.  One row a sequence, us of a layer, the pages
// shared / each sequence by itself / in qg_tree_attention (heads, cache, sequences, MiB saved):
//   2 x 128 fp16 8, 10: 17.2 / 14.5 / 13.3    8, 23: 17.7 / 17.8 / 15.6    8, 47: 19.1 / 20.6 / 19.2    8, 95: 24.2 / 27.8 / 28.8
//   2 x 128 fp16 2, 48: 24.5 / 28.2 / 29.2    32, 47: 21.5 / 21.2 / 17.3   32, 93: 25.8 / 26.2 / 23.0   32, 155: 26.0 / 31.0 / 27.1
//   4 x 256 fp16 8, 42: 23.5 / 25.6 / 20.3    8, 91: 24.5 / 33.9 / 27.5    1 x 64 fp16 8, 96: 30.0 / 29.1 / 28.7, 160: 30.7 / 39.0 / 38.5
//   8 x 128 F32 8, 42: 22.1 / 23.3 / 20.2     32 (of 256 tokens), 62: 31.3 / 25.1 / 23.8
// the two sides cross between 20 and 95; the limit costs at most 2.5 us in what was timed but for the last, 6.
// What a prompt chunk's rows (more than a tree has) share does not count: their products take longer than their reads, and the row
// groups fill the registers with one sequence's rows as well.  8 chunks of 128 rows over 8000 common tokens: 2 x 128 fp16 229 / 212
// / 212, 4 x 128 with groups of five 330 / 219 / 253, 8 x 128 466 / 371 / 365; of 30 such batches of 96 and 128 rows one gained.
// Of 17 rows most gain (8 x 128 bf16 85 / 109 / 88), of 33 and 64 some lose.
constexpr int QUANTUM = 256;
constexpr int64_t LEAST_SAVING = 48 << 20;
thread_local int64_t tl_least_saving = LEAST_SAVING;
__host__ __device__ inline long shared_rows_most(long rows) {
    const long most = 16 * rows < 16384 ? 16 * rows : 16384;
    return most > 3 * rows ? most : 3 * rows;
}
template <int THREADS>
struct PlanShared {
    unsigned long long key[THREADS];
    int link[THREADS], cut[THREADS], n[THREADS], size[THREADS], off[THREADS], rep[THREADS], next[THREADS], sees[THREADS], top[THREADS], upto[THREADS + 1],
        run[THREADS + 1], first[THREADS + 1], wave[THREADS / 64 + 1];
    unsigned long long sum, saved;
};
template <int THREADS>
QG_DEV void plan_sync() {
    if (THREADS > 64) __syncthreads();
    else { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }
}
// Sum over the threads before this one; all: over all.
template <int THREADS>
QG_DEV int plan_before(PlanShared<THREADS> &s, int x, int t, int &all) {
    const int upto = wave_upto(x);
    if (THREADS == 64) { all = of_lane(upto, 63); return upto - x; }
    plan_sync<THREADS>();
    if ((t & 63) == 63) s.wave[t >> 6] = upto;
    plan_sync<THREADS>();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) {
        const int y = s.wave[w];
        if (w < t >> 6) before += y;
        all += y;
    }
    return before + upto - x;
}
// Sorts a key of each thread: exchanges at a distance of 64 and more through shared memory.
template <int THREADS>
QG_DEV unsigned long long plan_sort(PlanShared<THREADS> &s, unsigned long long key, int t) {
#pragma unroll 1
    for (int k = 2; k <= THREADS; k *= 2)
#pragma unroll 1
        for (int j = k / 2; j >= 1; j /= 2) {
            unsigned long long other;
            if (j >= 64) {
                plan_sync<THREADS>();
                s.key[t] = key;
                plan_sync<THREADS>();
                other = s.key[t ^ j];
            } else {
                other = __shfl_xor(key, j);
            }
            const bool low = (t & j) == 0, up = (t & k) == 0;
            key = (key < other) == (low == up) ? key : other;
        }
    plan_sync<THREADS>();
    s.key[t] = key;
    plan_sync<THREADS>();
    return key;
}
template <int THREADS>
QG_DEV void plan_segments(const KvView &c, const BatchView &b, const PrefixView &v, PlanShared<THREADS> &s, int64_t least_tokens, int t) {
    const int S = c.sequences;
    int first = 0, n = 0, len = 0, link0 = -1, shared0 = 0;
    if (t < S) {
        batch_rows(b, t, first, n);
        len = kv_length(c, t);
        if (n > 0) { link0 = v.link[t]; shared0 = v.shared[t]; }
    }
    s.n[t] = n;
    int link = -1, cut = 0;
    for (int quantum = QUANTUM > 1 << c.shift ? QUANTUM : 1 << c.shift;; quantum *= 2) {
        // the nearest on the way up that has less in common with the one above it
        cut = shared0 / quantum * quantum;
        plan_sync<THREADS>();
        s.link[t] = link0;
        s.cut[t] = cut;
        s.size[t] = 0;
        s.top[t] = -1;
        if (t == 0) { s.sum = 0; s.saved = 0; }
        plan_sync<THREADS>();
        const unsigned long long saved = wave_all_add((unsigned long long)(n > QG_MAX_TREE ? 0 : cut));
        if ((t & 63) == 0) atomicAdd(&s.saved, saved);
        link = cut ? link0 : -1;
        while (link >= 0 && s.cut[link] >= cut) link = s.link[link];
        plan_sync<THREADS>();
        if ((int64_t)s.saved < least_tokens) link = -1;  // a sequence does not read again what it shares
        if (link < 0) cut = 0;
        s.link[t] = link;
        s.cut[t] = cut;
        plan_sync<THREADS>();
        // rows of a sequence and those that hang on it
        if (n > 0)
            for (int u = t; u >= 0; u = s.link[u]) atomicAdd(&s.size[u], n);
        const unsigned long long own = n > 0 ? (unsigned long long)(link + 1) << 40 | (unsigned long long)((1 << 29) - cut) << 10 | (unsigned)t : ~0ULL;
        const unsigned long long key = plan_sort(s, own, t);
        // thread t now stands for the t-th in order, sequence u
        const bool is = key != ~0ULL;
        const int u = (int)(key & 1023);
        const unsigned long long before = t ? s.key[t - 1] : ~0ULL;
        const bool group = is && (t == 0 || before >> 40 != key >> 40), run = is && (t == 0 || before >> 10 != key >> 10);
        int rows, runs;
        const int upto = plan_before(s, is ? s.size[u] : 0, t, rows), mine = plan_before(s, (int)run, t, runs) + run - 1;
        s.upto[t] = upto;
        if (run) s.run[mine] = t;
        if (t == 0) {
            s.upto[THREADS] = rows;
            s.run[runs] = THREADS;
        }
        const int on = (int)(key >> 40) - 1;  // what u hangs on
        if (group) {
            s.first[on + 1] = upto;
            if (on >= 0) s.top[on] = u;
        }
        plan_sync<THREADS>();
        if (is) {
            const int start = s.run[mine], behind = s.run[mine + 1];
            s.off[u] = upto - s.first[on + 1];
            s.rep[u] = (int)(s.key[start] & 1023);
            s.next[u] = behind < THREADS && s.key[behind] >> 40 == key >> 40 ? (int)(s.key[behind] & 1023) : -1;
            s.sees[u] = s.upto[behind] - s.first[on + 1];
            if (run && on >= 0) atomicAdd(&s.sum, (unsigned long long)(s.sees[u] + s.n[on]));
        }
        plan_sync<THREADS>();
        if ((long)s.sum <= shared_rows_most(b.rows)) break;
    }
    // first rows in walking order
    int pos = 0;
    if (n > 0) {
        pos = s.off[t];
        for (int u = link; u >= 0; u = s.link[u]) pos += s.n[u] + s.off[u];
    }
    // the segments' numbers: the shared ones first
    const bool shares = n > 0 && link >= 0 && s.rep[t] == t;
    int heads, tails;
    const int head_id = plan_before(s, (int)shares, t, heads), tail_id = heads + plan_before(s, (int)(n > 0), t, tails);
    plan_sync<THREADS>();
    int *id = s.run, *at = s.first;  // done with
    id[t] = shares ? head_id : -1;
    at[t] = pos;
    plan_sync<THREADS>();
    if (t == 0) { v.head[0] = heads + tails; v.head[1] = heads; }
    // rows of no sequence: before the first, behind the last, and what one has too many
    int2 *of_row = (int2 *)v.of_row;
    for (int r = t, upto = kv_clamp(b.start[0], 0, b.rows); r < upto; r += THREADS) of_row[r] = make_int2(-1, 0);
    for (int r = kv_clamp(b.start[S], 0, b.rows) + t; r < b.rows; r += THREADS) of_row[r] = make_int2(-1, 0);
    if (t < S)
        for (int r = first + n, upto = kv_clamp(b.start[t + 1], 0, b.rows); r < upto; r++) of_row[r] = make_int2(-1, 0);
    auto put = [&](int i, const Segment &x) {
        int4 *to = (int4 *)(v.segments + (size_t)i * SEG_INTS);
        to[0] = make_int4(x.owner, x.begin, x.end, x.row0);
        to[1] = make_int4(x.rows, x.up, x.tail, 0);
    };
    // the segment that ends where sequence u leaves the one that it hangs on
    auto above = [&](int u) { return s.link[u] >= 0 ? id[s.rep[u]] : -1; };
    if (n > 0) {
        const int top = s.top[t];  // the first of those that leave it last
        put(tail_id, Segment{t, top >= 0 ? s.cut[top] : cut, len + n, pos, n, top >= 0 ? id[top] : above(t), 1, 0});
        for (int i = 0; i < n; i++) {
            if (pos + i < b.rows) v.row_of[pos + i] = first + i;
            of_row[first + i] = make_int2(tail_id, pos + i);
        }
    }
    if (shares) {
        const int next = s.next[t], up = next >= 0 ? id[s.rep[next]] : above(link);
        put(head_id, Segment{link, next >= 0 ? s.cut[next] : s.cut[link], cut, at[link], s.sees[t] + s.n[link], up, 0, 0});
    }
}
template <int THREADS>
__global__ __launch_bounds__(THREADS) void prefix_plan_kernel(KvView c, BatchView b, PrefixView v, int64_t least_tokens) {
    __shared__ PlanShared<THREADS> s;
    plan_segments<THREADS>(c, b, v, s, least_tokens, threadIdx.x);
}
// Both for few sequences, a wave each: 8 sequences 6.3 us, as two kernels 8.5; with more the waves of one
// workgroup would take several sequences each.
constexpr int SMALL = 16;
__global__ __launch_bounds__(64 * SMALL) void prefix_small_kernel(KvView c, BatchView b, PrefixView v, int64_t least_tokens, int *link, int *shared) {
    __shared__ PlanShared<64> s;
    const int wave = threadIdx.x >> 6;
    if (wave < c.sequences) link_sequence(c, b, v, link, shared, wave, threadIdx.x & 63);
    __syncthreads();
    if (wave == 0) plan_segments<64>(c, b, v, s, least_tokens, threadIdx.x);
}

// ------------------------------------------------------------------------
// Attention: one pass over a segment's keys with the running maximum and sum of a softmax, S^T = K Q^T and O^T = V^T P^T
// on the 16-bit matrix cores, q and p in two fp16 or three bf16 planes, tiles and planes as qg_tree_attention has them.
// A unit is a part of a segment's keys for a group of up to 16 MOST of its rows x heads, so that a key that is read
// serves as many rows as the registers hold.  64 sequences of one row over 98304 tokens in common (heads 16 over 2 of
// 128, fp16): 155 us where the products alone take 94, the matrix cores busy for a quarter of the cycles and the waves
// waiting for keys from L2 and behind it for half of theirs; qg_tree_attention takes 507.  16 trees of 17 rows over
// 24576 tokens (bf16) 153 us, 107 and 198.  8 sequences over 2048 tokens 17 us, of which the way to a unit's first key
// (plan 2.9, pages 2.2, queries 2.5) and the end are more than half.
// ------------------------------------------------------------------------
struct PrefixArgs : AttnRows {
    float *part_o;    // [tiles][16][D]
    float2 *part_ml;  // [tiles][16]
    int4 *joins;      // [2 sequences] SegmentParts
    int *odd;         // [rows][q_heads]: results that are no numbers, where they are written at once
    int resident, tiles;
};

QG_DEV Segment read_segment(const KvView &c, const BatchView &b, const PrefixView &v, int i) {
    const int4 *p = (const int4 *)(v.segments + (size_t)i * SEG_INTS);
    const int4 x = p[0], y = p[1];
    return segment_inside(c, b, Segment{x.x, x.y, x.z, x.w, y.x, y.y, y.z, 0});
}

// A unit of work: a part of a segment's keys, a head, a group of its rows.
struct Unit {
    Segment s;
    int id, groups, tiles, chunk, parts, part, z, h, tile;  // tiles: of a group; tile: the first of the segment's
};
constexpr int CHUNK = 128;  // keys per unit, at least and in steps of
// What a unit costs, in key x weight: a key weighs 1 more than its row tiles (its reads, and the products and
// weights of each tile), and to begin and to end takes as long as 1000 do (two levels of
// 8 x 8: 69 us, with 100 78 and with 4000 76; 8 x 2048 tokens 198, 200 and 230).
constexpr float UNIT_COST = 1000.0f;
__host__ __device__ constexpr int key_weight(int tiles) { return 1 + tiles; }

// A segment's row groups of equal size and as few as the registers allow.
struct UnitLane { int keys, groups, tiles; };
template <int MOST>
QG_DEV UnitLane unit_lane(const PrefixArgs &A, const Segment &s) {
    const int rows = s.rows * A.group, keys = s.end - s.begin;
    if (rows <= 0 || keys <= 0) return UnitLane{0, 0, 1};
    const int groups = (rows + 16 * MOST - 1) / (16 * MOST);
    int tiles = 1;
#pragma unroll
    for (int k = 1; k < MOST; k++) tiles += rows > 16 * k * groups;
    return UnitLane{keys, groups, tiles};
}
// The keys of a segment's part where a unit's keys cost `even`, and the parts.
QG_DEV int part_keys(float even, int tiles) {
    return ((int)fminf(even * __builtin_amdgcn_rcpf((float)key_weight(tiles)), (float)(1 << 28)) / CHUNK + 1) * CHUNK;
}
QG_DEV int part_count(float even, const UnitLane &x) {
    const int chunk = part_keys(even, x.tiles), n = (int)(((float)x.keys - 0.5f) * __builtin_amdgcn_rcpf((float)chunk)) + 1;
    return x.groups ? n + (n * chunk < x.keys) : 0;  // the product may be off in its last bits: never a key too few
}
// Every workgroup finds its unit by itself: in one round of resident workgroups (two, where the row groups alone come to
// half of one) units that cost about the same, of the shared segments first, and of both an eighth to each XCD, in whose
// L2 the row groups with the same keys meet.  False if there is none.  A thread per segment; a part's size is formed anew
// where it is needed, since an array that is picked from by a variable would be moved to shared memory under a size that
// is read from the launch's packet in the host's memory (8 us; this takes 2.9).
template <int NW>
struct FindShared { float f[2][2][NW]; int i[2][2][NW], found[8]; };
template <int MOST, int NW>
QG_DEV bool find_unit(const KvView &c, const BatchView &b, const PrefixArgs &A, const PrefixView &v, int block, FindShared<NW> &s, Unit &p) {
    constexpr int THREADS = 64 * NW;
    const int tid = threadIdx.x, wave = tid >> 6, most = 2 * c.sequences;
    const Segment own = read_segment(c, b, v, min(tid, most - 1));
    const int count = segment_count(c, v), shared = kv_clamp(v.head[1], 0, count);
    if (tid == 0) s.found[0] = -1;
    auto lane_of = [&](const Segment &x, int i) { return i < count ? unit_lane<MOST>(A, x) : UnitLane{0, 0, 1}; };
    const UnitLane mine = lane_of(own, tid);
    // f(a thread's segment, its number) for all
    auto each = [&](auto f) {
#pragma unroll 1
        for (int i = tid; i - tid < count; i += THREADS) f(i < THREADS ? mine : lane_of(read_segment(c, b, v, min(i, most - 1)), i), i);
    };
    // sums of two values over the workgroup; the places alternate, so that one barrier does
    int turn = 0;
    auto sum2 = [&](auto (&at)[2][2][NW], auto &x, auto &y) {
        turn ^= 1;
        x = wave_all_add(x);
        y = wave_all_add(y);
        if ((tid & 63) == 0) { at[turn][0][wave] = x; at[turn][1][wave] = y; }
        __syncthreads();
        x = at[turn][0][0];
        y = at[turn][1][0];
#pragma unroll
        for (int w = 1; w < NW; w++) { x += at[turn][0][w]; y += at[turn][1][w]; }
    };
    float groups = 0.0f, cost = 0.0f;
    each([&](const UnitLane &x, int) {
        groups += (float)x.groups;
        cost += (float)x.groups * ((float)x.keys * (float)key_weight(x.tiles) + UNIT_COST);
    });
    sum2(s.f, groups, cost);
    groups *= (float)c.heads;
    cost *= (float)c.heads;
    const float room = (2.0f * groups <= (float)A.resident ? 1.0f : 2.0f) * (float)A.resident;
    // 1.0001: above the sum whatever its roundings, so that the tiles suffice.  Groups that are cut round up by a part at
    // most: with that much less room what the units cost together fits.
    float even = 1.0001f * cost / room, cut = 0.0f, none = 0.0f;
    each([&](const UnitLane &x, int) { cut += (float)(x.keys * key_weight(x.tiles)) > even ? (float)x.groups : 0.0f; });
    sum2(s.f, cut, none);
    cut *= (float)c.heads;
    if (groups <= room) even = 1.0001f * cost / (room - fminf(cut, 0.5f * room));
    int of_shared = 0, units = 0;
    each([&](const UnitLane &x, int i) {
        const int n = part_count(even, x) * x.groups * c.heads;
        units += n;
        of_shared += i < shared ? n : 0;
    });
    sum2(s.i, units, of_shared);
    // blocks go round the XCDs
    const int run = (of_shared + 7) / 8, tail_run = (units - of_shared + 7) / 8, x = block & 7, k = block >> 3;
    const int unit = k < run ? x * run + k : of_shared + x * tail_run + (k - run);
    if (unit < 0 || unit >= (k < run ? of_shared : units) || k - run >= tail_run) return false;  // below 0: row starts that overlap, past 2^31 units
    int before = 0, tiles = 0;
    each([&](const UnitLane &x, int i) {
        const int parts = part_count(even, x), own = parts * x.groups * c.heads;
        const int upto = wave_upto(own), upto_tiles = wave_upto(own * x.tiles);
        turn ^= 1;
        if ((tid & 63) == 63) { s.i[turn][0][wave] = upto; s.i[turn][1][wave] = upto_tiles; }
        __syncthreads();
        int first = before + upto - own, tile = tiles + upto_tiles - own * x.tiles;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const int n = s.i[turn][0][w], m = s.i[turn][1][w];
            if (w < wave) { first += n; tile += m; }
            before += n;
            tiles += m;
        }
        if (unit >= first && unit < first + own) {
            s.found[0] = i; s.found[1] = x.groups; s.found[2] = x.tiles; s.found[3] = parts; s.found[4] = tile; s.found[5] = unit - first;
        }
    });
    __syncthreads();
    p.id = __builtin_amdgcn_readfirstlane(s.found[0]);
    if (p.id < 0) return false;
    p.s = read_segment(c, b, v, p.id);
    p.groups = __builtin_amdgcn_readfirstlane(s.found[1]);
    p.tiles = __builtin_amdgcn_readfirstlane(s.found[2]);
    p.parts = __builtin_amdgcn_readfirstlane(s.found[3]);
    p.tile = __builtin_amdgcn_readfirstlane(s.found[4]);
    const int rest = __builtin_amdgcn_readfirstlane(s.found[5]), of_head = rest / p.groups;
    p.z = rest - of_head * p.groups;
    p.part = of_head / c.heads;
    p.h = of_head - p.part * c.heads;
    p.chunk = part_keys(even, p.tiles);
    return true;
}

template <int TYPE, int D, int MOST, int NW>
struct PrefixShared {
    typedef Tile<TYPE, D> T;
    static constexpr int JOIN = NW * 16 * (D + 4) * 4, Q = MOST * T::Q_BYTES;  // of one row tile; two are used in turn
    __attribute__((aligned(16))) uint8_t mem[Q > 2 * JOIN ? Q : 2 * JOIN];
    float m[NW][16 * MOST], l[NW][16 * MOST], back[16 * MOST];
    unsigned long long seen[QG_MAX_TREE];
    FindShared<NW> find;
};

// One unit, as qg_tree_attention takes a part of a sequence: each wave walks tiles of
// keys of its own, for RT row tiles, and the waves' sums are joined in shared memory.
template <int TYPE, int D, int RT, bool TAIL, int NW, typename SHARED>
QG_DEV void unit_attention(const PrefixArgs &A, const KvView &c, const BatchView &b, const PrefixView &v, const Unit &p, SHARED &s) {
    typedef Tile<TYPE, D> T;
    constexpr int RG = 16 * RT, E = T::E, DL = T::DL, KEYS = T::KEYS;
    constexpr bool FIRST = D > 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int row0 = p.z * RG, rows = p.s.rows * A.group, owner = p.s.owner;
    int first = 0, count = 0, len = p.s.end;
    if (TAIL) {
        batch_rows(b, owner, first, count);
        len = kv_length(c, owner);
    }
    // the unit's keys, and the first one that some row may not see
    const int begin = p.s.begin + p.part * p.chunk;
    int keys = p.s.end, open = p.s.end;
    if (TAIL) {
        if (!b.parent) keys = min(keys, len + by_group(A, min(row0 + RG, rows) - 1) + 1);
        open = len + (b.parent ? 0 : by_group(A, row0) + 1);
    }
    const int end = min(begin + p.chunk, keys);
    const bool direct = TAIL && p.parts == 1 && p.s.begin == 0;
    const int tile0 = p.tile + ((p.part * c.heads + p.h) * p.groups + p.z) * RT;
    const bool fits = tile0 >= 0 && tile0 + RT <= A.tiles;
    if (tid == 0 && p.part == 0 && p.h == 0 && p.z == 0) A.joins[p.id] = make_int4(p.tile, p.parts, p.groups, RT);
    if (begin >= end) {  // rows that come before the sequence's last keys
        if (fits && tid < RG) A.part_ml[(size_t)tile0 * 16 + tid] = make_float2(-__builtin_inff(), 0.0f);
        return;
    }
    const size_t page_bytes = ((size_t)c.heads << c.shift) * D * T::ES;
    const uint8_t *kbase = c.k + (((size_t)A.layer * c.pages * c.heads + p.h) << c.shift) * D * T::ES;
    const uint8_t *vbase = c.v + (((size_t)A.layer * c.pages * c.heads + p.h) << c.shift) * D * T::ES;
    const int slot_mask = (1 << c.shift) - 1;
    // a run of E keys from position pos, aligned to E: inside one page
    auto run = [&](const uint8_t *base, int page, int pos) { return base + (size_t)max(page, 0) * page_bytes + (size_t)((pos & slot_mask) * (D * T::ES)); };
    // the pages and the places of the rows first, then what lies there: two round trips before the first product
    T tile;
    int t0 = begin + wave * KEYS, kpos = t0 + E * (n >> 2), vpos = t0 + E * g;
    int kpage = kv_page(c, owner, kpos), vpage = kv_page(c, owner, vpos);
    int kpage1 = kv_page(c, owner, kpos + NW * KEYS), vpage1 = kv_page(c, owner, vpos + NW * KEYS);
    int rows_at[RG / (4 * NW)];
#pragma unroll
    for (int i = 0; i < RG / (4 * NW); i++) {
        const int at = row0 + (i * NW + wave) * 4 + g, t = by_group(A, at);
        rows_at[i] = -1;
        if (at < rows) rows_at[i] = TAIL ? (t < count ? first + t : -1) : kv_clamp(v.row_of[p.s.row0 + t], 0, b.rows - 1);
    }
    if (t0 < end) {
        tile.load_k(run(kbase, kpage, kpos), n, g);
        tile.load_v(run(vbase, vpage, vpos), n);
    }
    float x[RG / (4 * NW)][DL];
    size_t at_q[RG / (4 * NW)];  // the row and head, or -1
#pragma unroll
    for (int i = 0; i < RG / (4 * NW); i++) {
        const int at = row0 + (i * NW + wave) * 4 + g, row = rows_at[i];
        at_q[i] = row >= 0 ? (size_t)row * A.q_heads + p.h * A.group + (at - by_group(A, at) * A.group) : (size_t)-1;
#pragma unroll
        for (int d = 0; d < DL; d += 4) {
            const float4 y = row >= 0 ? *(const float4 *)(A.q + at_q[i] * D + n * DL + d) : make_float4(0, 0, 0, 0);
            x[i][d] = y.x; x[i][d + 1] = y.y; x[i][d + 2] = y.z; x[i][d + 3] = y.w;
        }
    }
#pragma unroll
    for (int i = 0; i < RG / (4 * NW); i++) {
        const int r = (i * NW + wave) * 4 + g;
#pragma unroll
        for (int d = 0; d < DL; d++) x[i][d] *= A.scale;
        float back = 1.0f;
        if constexpr (TYPE == QT_F16) {
            float top = 0.0f;
#pragma unroll
            for (int d = 0; d < DL; d++) top = fmaxf(top, fabsf(x[i][d]));
            top = qg_row_max(top);
            // 2^e with top 2^e in [2^13, 2^14): fp16's whole precision for what matters of the row
            const int e = min(max(127 + 13 - (int)(__float_as_uint(top) >> 23), -126), 126);
            if (top > 0.0f && top < __builtin_inff()) {
                const float f = __uint_as_float((uint32_t)(e + 127) << 23);
                back = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int d = 0; d < DL; d++) x[i][d] *= f;
            }
        }
        if (n == 0) s.back[r] = back;
        if (n == 0 && TAIL && p.part == 0 && at_q[i] != (size_t)-1) A.odd[at_q[i]] = 0;
        uint8_t *frag = s.mem + (r >> 4) * T::Q_BYTES;
#pragma unroll
        for (int d = 0; d < DL; d += 8) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = d + j < DL ? x[i][(d + j) % DL] : 0.0f;
            T::put_q(frag, r & 15, n * DL + d, y, DL - d);
        }
    }
    if (TAIL && b.parent && wave == 0) s.seen[lane] = tree_ancestors(b.parent + first, count, lane);
    __syncthreads();

    qg_f4 o[RT][DL];
    float m[RT], l[RT], back[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
        back[r] = TYPE == QT_F16 ? s.back[16 * r + n] : 1.0f;
        m[r] = -__builtin_inff();
        l[r] = 0.0f;
#pragma unroll
        for (int t = 0; t < DL; t++) o[r][t] = qg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (; t0 < end; t0 += NW * KEYS) {
        float z[RT][E];
        if (FIRST) __builtin_amdgcn_s_setprio(1);
        tile.template scores<RT>(s.mem, lane, z);
        if (FIRST) __builtin_amdgcn_s_setprio(0);
        // the next tile's keys, whose pages are known, and the pages of the one after it
        const int here = vpage, here_pos = vpos;
        const bool more = t0 + NW * KEYS < end;
        kpos += NW * KEYS;
        vpos += NW * KEYS;
        vpage = vpage1;
        if (more) {
            tile.load_k(run(kbase, kpage1, kpos), n, g);
            kpage1 = kv_page(c, owner, kpos + NW * KEYS);
            vpage1 = kv_page(c, owner, vpos + NW * KEYS);
        }
        if (t0 + KEYS > open || !__all(here >= 0)) {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (here < 0 || here_pos + e >= end) tile.drop_v(e);
#pragma unroll
            for (int r = 0; r < RT; r++) {
                // bit e: key here_pos + e, below the row's prefix or among the rows that it descends from
                unsigned seen = first_bits(end - here_pos, E);
                if (TAIL) {
                    const int t = by_group(A, row0 + 16 * r + n), prefix = b.parent ? len : len + t + 1, k = here_pos - len;
                    unsigned mine = first_bits(prefix - here_pos, E);
                    if (b.parent && t < count && k < 64 && k > -E) mine |= (unsigned)(k < 0 ? s.seen[t] << -k : s.seen[t] >> k);
                    seen &= mine;
                }
                if (here < 0) seen = 0;
#pragma unroll
                for (int e = 0; e < E; e++) z[r][e] = seen >> e & 1 ? z[r][e] : -__builtin_inff();
            }
        }
        // scores to weights: the maximum is renewed only where it moves by more than the lag
#pragma unroll
        for (int r = 0; r < RT; r++) {
            float top = z[r][0];
#pragma unroll
            for (int e = 1; e < E; e++) top = fmaxf(top, z[r][e]);
            top *= back[r];
            if (__any(top > m[r] + m_lag(TYPE))) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float next = fmaxf(m[r], top);
                const float a = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m[r] - next);
                m[r] = next;
                l[r] *= a;
#pragma unroll
                for (int t = 0; t < DL; t++) o[r][t] *= a;
            }
            const float base = m[r] == -__builtin_inff() ? 0.0f : m[r] - p_base(TYPE);
#pragma unroll
            for (int e = 0; e < E; e++) {
                z[r][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[r][e], back[r], -base));
                l[r] += z[r][e];
            }
        }
        if (FIRST) __builtin_amdgcn_s_setprio(1);
        tile.template outputs<RT>(z, o);
        if (FIRST) __builtin_amdgcn_s_setprio(0);
        if (more) tile.load_v(run(vbase, vpage, vpos), n);
    }

    // the waves' sums are joined row tile by row tile: their weights first
#pragma unroll
    for (int r = 0; r < RT; r++) {
        l[r] += __shfl_xor(l[r], 16);
        l[r] += __shfl_xor(l[r], 32);
        if (g == 0) { s.m[wave][16 * r + n] = m[r]; s.l[wave][16 * r + n] = l[r]; }
    }
    __syncthreads();  // the queries' fragments are done with, too
    if (tid < RG) {
        float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) top = fmaxf(top, s.m[w][tid]);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float lw = s.l[w][tid], f = part_weight(s.m[w][tid], lw, top);
            if (f >= 0.0f) sum = __builtin_fmaf(f, lw, sum);
            s.m[w][tid] = f;
        }
        s.l[0][tid] = sum;
        if (!direct && fits) A.part_ml[(size_t)tile0 * 16 + tid] = make_float2(top, sum);
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
        float *join = (float *)(s.mem + (r & 1) * SHARED::JOIN);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < DL; t += 4)
                *(float4 *)(join + (wave * 16 + n) * (D + 4) + DL * (4 * g + i) + t) =
                    make_float4(o[r][t][i], o[r][t + 1][i], o[r][t + 2][i], o[r][t + 3][i]);
        __syncthreads();
#pragma unroll
        for (int x0 = 0; x0 < 16 * D / 4; x0 += 64 * NW) {
            const int at4 = x0 + tid, row = at4 / (D / 4), d = at4 % (D / 4) * 4, at = row0 + 16 * r + row;
            float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float f = s.m[w][16 * r + row];
                const float4 u = *(const float4 *)(join + (w * 16 + row) * (D + 4) + d);
                y.x = f < 0.0f ? y.x : __builtin_fmaf(f, u.x, y.x);
                y.y = f < 0.0f ? y.y : __builtin_fmaf(f, u.y, y.y);
                y.z = f < 0.0f ? y.z : __builtin_fmaf(f, u.z, y.z);
                y.w = f < 0.0f ? y.w : __builtin_fmaf(f, u.w, y.w);
            }
            if (at >= rows) continue;
            if (direct) {
                const float sum = s.l[0][16 * r + row], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int t = by_group(A, at);
                if (t >= count) continue;
                const size_t to = (size_t)(first + t) * A.q_heads + p.h * A.group + (at - t * A.group);
                *(float4 *)(A.out + to * D + d) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
                if (odd_sums(y.x, y.y, sum) || odd_sums(y.z, y.w, sum)) A.odd[to] = 1;
            } else if (fits) {
                *(float4 *)(A.part_o + ((size_t)(tile0 + r) * 16 + row) * D + d) = y;
            }
        }
    }
}

template <int TYPE, int D, int MOST, bool TAIL, int NW, int RT, typename SHARED>
QG_DEV void unit_of_tiles(const PrefixArgs &A, const KvView &c, const BatchView &b, const PrefixView &v, const Unit &p, SHARED &s) {
    if (p.tiles == RT) unit_attention<TYPE, D, RT, TAIL, NW>(A, c, b, v, p, s);
    else if constexpr (RT < MOST) unit_of_tiles<TYPE, D, MOST, TAIL, NW, RT + 1>(A, c, b, v, p, s);
}
template <int TYPE, int D, int MOST, int NW>
__global__ __launch_bounds__(64 * NW, (D / 64) * MOST <= 6 ? 2 : 1) void prefix_attention_kernel(PrefixArgs A, KvView c, BatchView b, PrefixView v) {
    __shared__ PrefixShared<TYPE, D, MOST, NW> s;
    Unit p;
    if (!find_unit<MOST, NW>(c, b, A, v, blockIdx.x, s.find, p)) return;
    if (p.s.tail) unit_of_tiles<TYPE, D, MOST, true, NW, 1>(A, c, b, v, p, s);
    else unit_of_tiles<TYPE, D, MOST, false, NW, 1>(A, c, b, v, p, s);
}

// Joins a row's segments.  Few rows and heads: a workgroup each, whose four waves
// share the parts (8 rows, 8 layers: 198 us, by a wave each 203); many: a wave each
// (272 rows of 20 heads 156 us, by workgroups 164).  Bound by four dependent reads: 6 to 11 us.
constexpr int JOIN_WAVES = 4;
constexpr size_t JOIN_FEW = 1024;

// Parts i0, i0 + by, .. of a row, `step` rows of partial results apart from `slot` on:
// added to the sums y under the largest m so far.  A lane holds the weight of one part.
template <int D>
QG_DEV void join_parts(const PrefixArgs &A, long slot, long step, int parts, int i0, int by, int lane, float &top, float &sum, float (&y)[D / 64]) {
    constexpr int V = D / 64;
    const float2 *ml = A.part_ml + slot;
    const float *po = A.part_o + slot * D + lane * V;
    for (; i0 < parts; i0 += 64 * by) {
        const int mine = i0 + lane * by, count = min((parts - i0 + by - 1) / by, 64);
        const float2 x = mine < parts ? ml[mine * step] : make_float2(-__builtin_inff(), 0.0f);
        const float next = fmaxf(top, qg_wave_max(x.x));
        const float old = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - next);
        const float f = part_weight(x.x, x.y, next);
        top = next;
        sum = sum * old + qg_sum_lanes<64>(f < 0.0f ? 0.0f : f * x.y);
#pragma unroll
        for (int w = 0; w < V; w++) y[w] *= old;
        for (int i = 0; i < count; i += 8) {
            float u[8][V];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float *from = po + (i0 + min(i + k, count - 1) * by) * step * D;
#pragma unroll
                for (int w = 0; w < V; w++) u[k][w] = from[w];
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float q = i + k < count ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), (i + k) & 63)) : -1.0f;
#pragma unroll
                for (int w = 0; w < V; w++) y[w] = q < 0.0f ? y[w] : __builtin_fmaf(q, u[k][w], y[w]);
            }
        }
    }
}
template <int TYPE, int D, int EACH>
__global__ __launch_bounds__(64 * JOIN_WAVES) void prefix_join_kernel(PrefixArgs A, KvView c, BatchView b, PrefixView v) {
    constexpr int V = D / 64;
    __shared__ float s_y[JOIN_WAVES][D];
    __shared__ float2 s_w[JOIN_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t at = EACH == 1 ? blockIdx.x : (size_t)blockIdx.x * EACH + wave;
    if (at >= (size_t)b.rows * A.q_heads) return;
    const int row = (int)(at / A.q_heads), head = (int)(at % A.q_heads), h = by_group(A, head);
    const int2 place = ((const int2 *)v.of_row)[row];
    const int count = segment_count(c, v), pos = __builtin_amdgcn_readfirstlane(place.y);
    int id = __builtin_amdgcn_readfirstlane(place.x);
    if (id < 0 || id >= count) return;  // nothing was written for it
    bool odd = false;
    Segment g = read_segment(c, b, v, id);
    int4 j = A.joins[id];
    if (g.begin == 0 && j.y == 1) {
        odd = A.odd[at] == 1;
    } else {
        float top = -__builtin_inff(), sum = 0.0f, y[V];
#pragma unroll
        for (int w = 0; w < V; w++) y[w] = 0.0f;
        for (int k = 0; k < count; k++) {
            const int x = (pos - g.row0) * A.group + (head - h * A.group);
            long slot, step;
            if (pos >= g.row0 && pos < g.row0 + g.rows && segment_place(SegmentParts{j.x, j.y, j.z, j.w}, c.heads, h, x, A.tiles, slot, step)) {
                if (EACH > 1) join_parts<D>(A, slot, step, j.y, 0, 1, lane, top, sum, y);
                else join_parts<D>(A, slot, step, j.y, (wave + k) & (JOIN_WAVES - 1), JOIN_WAVES, lane, top, sum, y);
            }
            id = g.up;
            if (id < 0 || id >= count) break;
            g = read_segment(c, b, v, id);
            j = A.joins[id];
        }
        if (EACH == 1) {
#pragma unroll
            for (int w = 0; w < V; w++) s_y[wave][lane * V + w] = y[w];
            if (lane == 0) s_w[wave] = make_float2(top, sum);
            __syncthreads();
            if (wave) return;
            const float most = fmaxf(fmaxf(s_w[0].x, s_w[1].x), fmaxf(s_w[2].x, s_w[3].x));
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < V; w++) y[w] = 0.0f;
#pragma unroll
            for (int w = 0; w < JOIN_WAVES; w++) {
                const float2 u = s_w[w];
                const float f = part_weight(u.x, u.y, most);
                if (f < 0.0f) continue;
                sum = __builtin_fmaf(f, u.y, sum);
#pragma unroll
                for (int i = 0; i < V; i++) y[i] = __builtin_fmaf(f, s_y[w][lane * V + i], y[i]);
            }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int w = 0; w < V; w++) {
            odd |= odd_sums(y[w], 0.0f, sum);
            A.out[at * D + lane * V + w] = y[w] * inv;
        }
        odd = __any(odd);
    }
    if (!odd || (EACH == 1 && wave)) return;
    int first, n;
    const int s = batch_sequence(b, c.sequences, row, lane, first, n);
    if (s >= 0) attend_row<TYPE, D>(A, c, b, s, first, n, row, head, lane, s_y[wave]);
}

// Row groups of all segments, at most (each rounds up), and their row tiles: groups of t tiles have more than t - 1 tiles' rows each.
long groups_most(const BatchView &b, int S, int group, int dim) {
    return (shared_rows_most(b.rows) + b.rows) * group / (16 * most_tiles(dim)) + 2L * S;
}
// Tiles of partial results that the units can ask for: parts of a segment are at most its share of a round + 1.
long tiles_most(const BatchView &b, int S, int heads, int group, int dim) {
    return 2L * resident(dim, most_tiles(dim)) * most_tiles(dim) +
           heads * ((shared_rows_most(b.rows) + b.rows) * group / 16 + groups_most(b, S, group, dim) + 2L * S);
}
template <int TYPE, int D>
void launch(const PrefixArgs &A, const KvView &c, const BatchView &b, const PrefixView &v, hipStream_t s) {
    const long units = 2 * A.resident + groups_most(b, c.sequences, A.group, D) * c.heads + 16;
    prefix_attention_kernel<TYPE, D, most_tiles(D), WAVES><<<(unsigned)((units + 7) / 8 * 8), 64 * WAVES, 0, s>>>(A, c, b, v);
    const size_t jobs = (size_t)b.rows * A.q_heads;
    if (jobs > JOIN_FEW) prefix_join_kernel<TYPE, D, 4><<<(unsigned)((jobs + 3) / 4), 256, 0, s>>>(A, c, b, v);
    else prefix_join_kernel<TYPE, D, 1><<<(unsigned)jobs, 256, 0, s>>>(A, c, b, v);
}
template <int TYPE>
void launch_dim(const PrefixArgs &A, const KvView &c, const BatchView &b, const PrefixView &v, hipStream_t s) {
    if (c.dim == 64) launch<TYPE, 64>(A, c, b, v, s);
    else if (c.dim == 128) launch<TYPE, 128>(A, c, b, v, s);
    else launch<TYPE, 256>(A, c, b, v, s);
}
constexpr long JOBS = 1L << 25;  // rows x heads: of the join kernel, a wave each, within 2^32 threads
constexpr long TILES = 1L << 27; // of partial results, within an int of rows
}  // namespace

extern "C" {

int64_t qg_prefix_least_saving(int64_t bytes) {
    const int64_t before = tl_least_saving;
    tl_least_saving = bytes < 0 ? LEAST_SAVING : bytes < (int64_t)1 << 60 ? bytes : (int64_t)1 << 60;
    return before;
}

size_t qg_kv_prefixes_bytes(const qg_kv_cache *cache, const qg_kv_batch *batch) {
    if (qg_kv_check(cache, false, nullptr) || qg_batch_check(batch, false, nullptr)) return 0;
    return prefix_bytes(cache->sequences, batch->rows);
}

int qg_kv_prefixes(int *link, int *shared, const qg_kv_cache *cache, const qg_kv_batch *batch, void *prefixes, size_t prefixes_bytes) {
    KvView c;
    BatchView b;
    const size_t need = qg_kv_prefixes_bytes(cache, batch);
    if (!need || qg_kv_check(cache, false, &c) || qg_batch_check(batch, false, &b)) return hipErrorInvalidValue;
    if (!prefixes || prefixes_bytes < need || ((uintptr_t)prefixes & 15) || (((uintptr_t)link | (uintptr_t)shared) & 3)) return hipErrorInvalidValue;
    const size_t each = qg_ints(c.sequences);
    const QgSpan out[3] = {{link, each}, {shared, each}, {prefixes, need}},
                 in[3] = {{c.table, qg_table_bytes(c)}, {c.length, each}, {b.start, each + 4}};
    if (qg_any_overlap(out, in) || qg_overlap(link, each, shared, each) || qg_overlap(prefixes, need, link, each) || qg_overlap(prefixes, need, shared, each))
        return hipErrorInvalidValue;
    const PrefixView v = prefix_view(prefixes, c.sequences, b.rows);
    const int64_t token = 2LL * c.heads * c.dim * (c.type == QT_F32 ? 4 : 2), least = (tl_least_saving + token - 1) / token;
    if (c.sequences <= SMALL) {
        prefix_small_kernel<<<1, 64 * SMALL, 0, qg_stream()>>>(c, b, v, least, link, shared);
        return hipGetLastError();
    }
    prefix_link_kernel<<<(c.sequences + 3) / 4, 256, 0, qg_stream()>>>(c, b, v, link, shared);
    if (c.sequences <= 64) prefix_plan_kernel<64><<<1, 64, 0, qg_stream()>>>(c, b, v, least);
    else prefix_plan_kernel<QG_MAX_SEQUENCES><<<1, QG_MAX_SEQUENCES, 0, qg_stream()>>>(c, b, v, least);
    return hipGetLastError();
}

size_t qg_prefix_attention_workspace_bytes(const qg_kv_cache *cache, const qg_kv_batch *batch, int q_heads) {
    BatchView b;
    if (qg_kv_check(cache, false, nullptr) || qg_batch_check(batch, false, &b)) return 0;
    if (q_heads < 1 || q_heads % cache->kv_heads || q_heads / cache->kv_heads > 128) return 0;
    if ((long)batch->rows * q_heads > JOBS) return 0;
    const long tiles = tiles_most(b, cache->sequences, cache->kv_heads, q_heads / cache->kv_heads, cache->head_dim);
    if (tiles > TILES) return 0;
    return (size_t)tiles * 16 * (4 * (size_t)cache->head_dim + sizeof(float2)) + sizeof(int4) * 2 * (size_t)cache->sequences +
           4 * (size_t)batch->rows * q_heads;
}

int qg_prefix_attention(float *out, const float *q, int q_heads, float scale, const qg_kv_cache *cache, int layer, const qg_kv_batch *batch,
                        const void *prefixes, size_t prefixes_bytes, void *ws, size_t ws_bytes) {
    KvView c;
    BatchView b;
    const size_t need = qg_prefix_attention_workspace_bytes(cache, batch, q_heads), plan = qg_kv_prefixes_bytes(cache, batch);
    if (!need || !plan || qg_kv_check(cache, false, &c) || qg_batch_check(batch, false, &b)) return hipErrorInvalidValue;
    if (!out || !q || !ws || ws_bytes < need || (((uintptr_t)out | (uintptr_t)q | (uintptr_t)ws) & 15)) return hipErrorInvalidValue;
    if (!prefixes || prefixes_bytes < plan || ((uintptr_t)prefixes & 15)) return hipErrorInvalidValue;
    if (layer < 0 || layer >= c.layers || !__builtin_isfinite(scale * 1.44269504088896341f)) return hipErrorInvalidValue;
    const size_t bytes = 4 * (size_t)b.rows * q_heads * c.dim;
    const QgSpan written[2] = {{out, bytes}, {ws, need}}, read[2] = {{q, bytes}, {prefixes, plan}};
    if (qg_any_overlap(written, read) || qg_overlap(out, bytes, ws, need)) return hipErrorInvalidValue;
    const int group = q_heads / c.heads;
    const long tiles = tiles_most(b, c.sequences, c.heads, group, c.dim);
    float *part_o = (float *)ws;
    float2 *part_ml = (float2 *)(part_o + (size_t)tiles * 16 * c.dim);
    int4 *joins = (int4 *)(part_ml + (size_t)tiles * 16);
    const PrefixArgs A{attn_rows(out, q, q_heads, group, layer, scale), part_o, part_ml, joins, (int *)(joins + 2 * (size_t)c.sequences),
                       resident(c.dim, most_tiles(c.dim)), (int)tiles};
    const PrefixView v = prefix_view(const_cast<void *>(prefixes), c.sequences, b.rows);
    if (c.type == QT_F32) launch_dim<QT_F32>(A, c, b, v, qg_stream());
    else if (c.type == QT_F16) launch_dim<QT_F16>(A, c, b, v, qg_stream());
    else launch_dim<QT_BF16>(A, c, b, v, qg_stream());
    return hipGetLastError();
}

}  // extern "C"
