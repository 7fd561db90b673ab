// The buffer of qg_kv_prefixes (include/qwen_gpu.h) as kernels see it, and the reads
// that keep every index inside the batch and the cache whatever it holds (a buffer of
// an earlier batch, say).  Plain C++ for the device and the host: the same functions are tested
// without a GPU.
#pragma once
#include "qg_kv_index.h"

// A run of keys, begin..end-1 of sequence owner, and the rows that see all of it, in
// walking order; of the last segment of a sequence (tail) its own rows, by the batch's
// tree or chain.  up: the segment in front of it, -1 for none.
struct Segment { int owner, begin, end, row0, rows, up, tail, pad; };
enum { SEG_INTS = 8, PREFIX_HEAD = 16 };

struct PrefixView {
    int *head;           // [0] number of segments, [1] of the shared ones, which come first
    int *segments;       // [2 S] Segment
    int *link, *shared;  // [S] as found, see qg_kv_prefixes
    int *row_of;         // [rows] in walking order
    int *of_row;         // [rows][2] the last segment of a row's sequence, -1 for none, and the row's place in walking order
};
KV_FN PrefixView prefix_view(void *at, int S, int rows) {
    int *p = (int *)at, *seg = p + PREFIX_HEAD, *link = seg + 2 * (size_t)S * SEG_INTS, *row_of = link + 2 * (size_t)S;
    return PrefixView{p, seg, link, link + S, row_of + 2 * (size_t)rows, row_of};
}
KV_FN size_t prefix_bytes(int S, int rows) { return 4 * ((size_t)PREFIX_HEAD + 2 * (size_t)S * SEG_INTS + 2 * (size_t)S + 3 * (size_t)rows); }

KV_FN int segment_count(const KvView &c, const PrefixView &v) { return kv_clamp(v.head[0], 0, 2 * c.sequences); }
KV_FN Segment segment_inside(const KvView &c, const BatchView &b, Segment s) {
    s.owner = kv_clamp(s.owner, 0, c.sequences - 1);
    s.begin = kv_clamp(s.begin, 0, kv_capacity(c)) & ~31;  // runs of keys are aligned
    s.end = kv_clamp(s.end, s.begin, kv_capacity(c) + b.max_rows);
    s.row0 = kv_clamp(s.row0, 0, b.rows);
    s.rows = kv_clamp(s.rows, 0, b.rows - s.row0);
    s.up = s.up >= 0 && s.up < 2 * c.sequences ? s.up : -1;
    return s;
}

// Where a segment's partial results lie, in tiles of 16 rows: the first, parts, row
// groups, tiles of a group.
struct SegmentParts { int tile, parts, groups, tiles; };
// Row x (of rows x heads of a group) of head h in them: the first part's place, and the step
// to the next; false if any part is outside `all` tiles, whatever p holds.
KV_FN bool segment_place(const SegmentParts &p, int heads, int h, int x, int all, long &slot, long &step) {
    if (p.tile < 0 || p.tile >= all || p.parts < 1 || p.parts > all || p.groups < 1 || p.groups > all || p.tiles < 1 || p.tiles > 4) return false;
    const int z = x / (16 * p.tiles);
    if (x < 0 || z >= p.groups) return false;
    step = (long)heads * p.groups * p.tiles * 16;
    slot = ((long)p.tile + ((long)h * p.groups + z) * p.tiles) * 16 + x % (16 * p.tiles);
    const long end = (long)all * 16;
    return step <= end && slot < end && (p.parts - 1) <= (end - 1 - slot) / step;
}
