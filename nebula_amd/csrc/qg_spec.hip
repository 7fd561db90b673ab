// Operators of a speculative step that work on rows: per-head norms and
// rotation of queries and keys with the store into the cache, softmax of
// logits, verification of drafts (include/qwen_gpu.h).
#include "qg_kv.h"

namespace {

// ------------------------------------------------------------------------
// Norm + rotation.  y = x / sqrt(mean(x^2) + eps) * w per head, then pairs
// (a, b) -> (a cos t - b sin t, b cos t + a sin t), t = position * freq.
// t grows with the position, so it is formed in 64 bits and reduced to a
// fraction of a turn before the fp32 sine (a position of 90000 in fp32 would
// be off by 4e-3 rad).  Four dimensions per lane; a head takes D/4 lanes.
// ------------------------------------------------------------------------
struct RopeArgs {
    float *q_out, *k_out;
    const float *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    const float *q_norm, *k_norm;
    const double *freq;
    const int *position;
    float eps;
    int rows, q_heads, kv_heads, rope, interleaved, cached;
};

QG_DEV void turn_of(double angle, float &s, float &c) {
    double r = angle * 0.15915494309189533577;  // turns
    r -= __builtin_rint(r);
    sincospif((float)(2.0 * r), &s, &c);
}

// A wave takes U heads-per-wave of one row: the row's place, its angles' sines and
// the loads of all its heads once.  Bound by memory where rows are many (8192 rows
// of 16 + 2 + 2 heads of 128: 35 us, 4.5 TB/s; with one head per wave 59), by the
// launch and three dependent reads where they are few (one row 3.7 us).
template <int D, int U>
__global__ __launch_bounds__(256) void qk_rope_kernel(RopeArgs A, KvView c, BatchView b, int layer, int parts) {
    constexpr int LPH = D / 4, HPW = 64 / LPH;  // lanes per head, heads per wave
    const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6), row = id / parts;
    if (row >= A.rows) return;
    const int d = (lane % LPH) * 4, h0 = id % parts * (U * HPW) + lane / LPH, heads = A.q_heads + A.kv_heads * (A.cached ? 2 : 1);
    // where head h of the row is read; 0, 1, 2: q, k, v
    auto kind = [&](int h) { return h < A.q_heads ? 0 : h < A.q_heads + A.kv_heads ? 1 : 2; };
    auto nth = [&](int h) { return h < A.q_heads ? h : h < A.q_heads + A.kv_heads ? h - A.q_heads : h - A.q_heads - A.kv_heads; };
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW, k = kind(h), i = nth(h);
        const float *src = k == 0 ? A.q + row * A.q_row + i * A.q_head : k == 1 ? A.k + row * A.k_row + i * A.k_head
                                                                              : A.v + row * A.v_row + i * A.v_head;
        const float4 y = h < heads ? *(const float4 *)(src + d) : make_float4(0, 0, 0, 0);
        x[u][0] = y.x; x[u][1] = y.y; x[u][2] = y.z; x[u][3] = y.w;
    }
    int pos = 0, slot = -1, page = -1;
    if (A.cached) {
        int first, n;
        const int s = batch_sequence(b, c.sequences, row, lane, first, n);
        if (s < 0) return;
        const int place = row - first;
        int depth = place;
        if (b.parent) depth = __popcll(__shfl(tree_ancestors(b.parent + first, n, lane), place)) - 1;
        const int len = kv_length(c, s);
        pos = len + depth;
        page = kv_page(c, s, len + place);
        slot = (len + place) & ((1 << c.shift) - 1);
    }
    if (A.position) pos = A.position[row];
    // of a lane's four dimensions: their pairs' angles, and the lane that holds the other halves
    const int half = A.rope / 2;
    const bool low = d < half, turned = d < A.rope;
    float sn[4], cs[4];
    if (turned) {
        const int f = A.interleaved ? d / 2 : low ? d : d - half;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (A.interleaved && i >= 2) { sn[i] = cs[i] = 0.0f; continue; }
            turn_of((double)pos * A.freq[f + i], sn[i], cs[i]);
        }
    }
    if (A.cached && kv_shared(c, page)) page = -1;  // behind the angles, which do not wait for it
    const int other = (lane + (low ? half / 4 : -(half / 4))) & 63;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW, k = kind(h), i = nth(h);
        const float *w = k == 0 ? A.q_norm : A.k_norm;
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) ss = __builtin_fmaf(x[u][j], x[u][j], ss);
        ss = qg_row_sum(ss);
        if (LPH >= 32) ss += __shfl_xor(ss, 16);
        if (LPH >= 64) ss += __shfl_xor(ss, 32);
        if (k < 2 && w) {
            const float scale = 1.0f / __builtin_sqrtf(ss / (float)D + A.eps);
            const float4 w4 = *(const float4 *)(w + d);
            x[u][0] = x[u][0] * scale * w4.x;
            x[u][1] = x[u][1] * scale * w4.y;
            x[u][2] = x[u][2] * scale * w4.z;
            x[u][3] = x[u][3] * scale * w4.w;
        }
        if (A.rope) {
            float y[4];
            if (A.interleaved) {
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    y[j] = x[u][j] * cs[j / 2] - x[u][j + 1] * sn[j / 2];
                    y[j + 1] = x[u][j + 1] * cs[j / 2] + x[u][j] * sn[j / 2];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float p = __shfl(x[u][j], other);
                    y[j] = low ? x[u][j] * cs[j] - p * sn[j] : x[u][j] * cs[j] + p * sn[j];
                }
            }
            if (k < 2 && turned) {
#pragma unroll
                for (int j = 0; j < 4; j++) x[u][j] = y[j];
            }
        }
        if (h >= heads) continue;
        const float4 y = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
        if (k == 0) *(float4 *)(A.q_out + ((size_t)row * A.q_heads + i) * D + d) = y;
        if (k == 1 && A.k_out) *(float4 *)(A.k_out + ((size_t)row * A.kv_heads + i) * D + d) = y;
        if (k == 0 || page < 0) continue;
        uint8_t *pool = k == 1 ? c.k : c.v;
        const size_t at = kv_at(c, layer, page, i, slot) + d;
        if (c.type == QT_F32) {
            *(float4 *)((float *)pool + at) = y;
        } else {
            uint32_t r[4];
#pragma unroll
            for (int j = 0; j < 4; j++) r[j] = c.type == QT_F16 ? kv_f16(x[u][j]) : kv_bf16(x[u][j]);
            *(uint2 *)((uint16_t *)pool + at) = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
        }
    }
}
template <int D>
void launch_rope(const RopeArgs &A, const KvView &c, const BatchView &b, int layer, hipStream_t s) {
    const int units = (A.q_heads + A.kv_heads * (A.cached ? 2 : 1) + 256 / D - 1) / (256 / D);  // wavefuls of heads per row
    const bool wide = (long)A.rows * units > 8192;  // more waves than the card holds: five times the work for each
    const int parts = wide ? (units + 4) / 5 : units;
    const unsigned blocks = (unsigned)(((long)A.rows * parts + 3) / 4);
    if (wide) qk_rope_kernel<D, 5><<<blocks, 256, 0, s>>>(A, c, b, layer, parts);
    else qk_rope_kernel<D, 1><<<blocks, 256, 0, s>>>(A, c, b, layer, parts);
}

// ------------------------------------------------------------------------
// Softmax of a row: e_i = 2^((x_i - m) log2 e / T), out = e_i / sum e.  A NaN, or
// an infinite m, makes the sum NaN and with it the row.  Loads and stores are
// one float per lane, so that a row may start anywhere.
// ------------------------------------------------------------------------

// 1 / T as the kernels use it: exponents are (x a - m a) b, in one fused step and a
// product.  a is 1, or 2^-64 for temperatures from 2^64 on, where x - m may be past the
// range although its share of T is not.  b 0 stands for temperature 0.
struct SoftScale {
    float a, b;
    __device__ __forceinline__ float power(float x, float ma) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, a, -ma) * b); }
};

// A workgroup's value by `op`, in every thread; s holds one per wave.
template <int THREADS, typename T, typename F>
QG_DEV T block_all(T v, T *s, F op) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = op(v, __shfl_xor(v, d));
    if (THREADS == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) v = op(v, s[w]);
    return v;
}
struct Larger { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Added {
    template <typename T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct Lower { __device__ __forceinline__ int operator()(int a, int b) const { return min(a, b); } };
constexpr int SM_NAN = -1;  // in place of the index of a row's largest value
// Where a thread's values THREADS apart hold the row's largest m first: the number
// of the value (an index each would cost a register each), -1 without one.
struct FirstOf {
    int k = -1;
    bool nan = false;
    __device__ __forceinline__ void see(int i, float x, float m) {  // from the last one down
        if (x == m) k = i;
        nan |= x != x;
    }
    template <int THREADS> __device__ __forceinline__ int index() const { return nan ? SM_NAN : k < 0 ? 0x7fffffff : k * THREADS + (int)threadIdx.x; }
};

// N values of a thread, THREADS apart, from x[0..n) on: whole groups of G without
// a bound per value, which would cost an address each.
template <int THREADS, int N, int G, typename F>
QG_DEV void read_spread(const float *x, int n, F put) {
    const float *at = x + threadIdx.x;
#pragma unroll
    for (int k0 = 0; k0 < N; k0 += G) {
        if ((k0 + G) * THREADS <= n) {
#pragma unroll
            for (int k = k0; k < k0 + G; k++) put(k, at[k * THREADS]);
        } else {
#pragma unroll
            for (int k = k0; k < k0 + G; k++) put(k, k * THREADS + (int)threadIdx.x < n ? at[k * THREADS] : -__builtin_inff());
        }
    }
}
template <int THREADS, int N, int G, typename F>
QG_DEV void write_spread(float *x, int n, F get) {
    float *at = x + threadIdx.x;
#pragma unroll
    for (int k0 = 0; k0 < N; k0 += G) {
        if ((k0 + G) * THREADS <= n) {
#pragma unroll
            for (int k = k0; k < k0 + G; k++) at[k * THREADS] = get(k);
        } else {
#pragma unroll
            for (int k = k0; k < k0 + G; k++)
                if (k * THREADS + (int)threadIdx.x < n) at[k * THREADS] = get(k);
        }
    }
}

// A workgroup per row of up to (REGS + KEPT) THREADS values: REGS values of a thread
// stay in registers and KEPT in shared memory between the three passes (largest
// value, sum, output).  96 + 36 values of 1024 threads are a CU's whole store: a row
// of 135168 is read once and written once (1088 x 131072: 255 us, 4.5 TB/s; read
// twice, with one value per thread and pass, 631).  BEST: temperature 0, in a kernel
// of its own, since the registers hold one of the two (250 us; both in one kernel 350).
template <int THREADS, int REGS, int KEPT, bool BEST>
__global__ __launch_bounds__(THREADS) void softmax_row_kernel(float *out, const float *x, int cols, SoftScale scale) {
    __shared__ float s_x[KEPT ? KEPT * THREADS : 1], s_f[THREADS / 64];
    __shared__ int s_i[BEST ? THREADS / 64 : 1];
    const int tid = threadIdx.x;
    const float *row = x + (size_t)blockIdx.x * cols;
    float *to = out + (size_t)blockIdx.x * cols;
    const float none = -__builtin_inff();
    float r[REGS], m = none;
    read_spread<THREADS, REGS, 8>(row, cols, [&](int k, float v) { r[k] = v; });
    if constexpr (KEPT > 0)
        read_spread<THREADS, KEPT, 4>(row + REGS * THREADS, cols - REGS * THREADS, [&](int k, float v) {
            s_x[k * THREADS + tid] = v;
            m = fmaxf(m, v);
        });
#pragma unroll
    for (int k = 0; k < REGS; k++) m = fmaxf(m, r[k]);
    m = block_all<THREADS>(m, s_f, Larger());
    if constexpr (BEST) {
        FirstOf first;
#pragma unroll 4
        for (int k = KEPT - 1; k >= 0; k--) first.see(REGS + k, s_x[k * THREADS + tid], m);
#pragma unroll
        for (int k = REGS - 1; k >= 0; k--) first.see(k, r[k], m);
        const int at = block_all<THREADS>(first.index<THREADS>(), s_i, Lower());
        const float rest = at == SM_NAN || m == __builtin_inff() ? __builtin_nanf("") : 0.0f;
        const int one = rest == 0.0f && m != none && at % THREADS == tid ? at / THREADS : -1;
        write_spread<THREADS, REGS, 8>(to, cols, [&](int k) { return k == one ? 1.0f : rest; });
        if constexpr (KEPT > 0)
            write_spread<THREADS, KEPT, 4>(to + REGS * THREADS, cols - REGS * THREADS, [&](int k) { return REGS + k == one ? 1.0f : rest; });
        return;
    }
    if (m == none) m = 0.0f;  // nothing but -infinity, or NaN: a sum of 0, or NaN
    const float ma = m * scale.a;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < REGS; k++) { r[k] = scale.power(r[k], ma); sum += r[k]; }
#pragma unroll 8
    for (int k = 0; k < KEPT; k++) {
        const float e = scale.power(s_x[k * THREADS + tid], ma);
        s_x[k * THREADS + tid] = e;
        sum += e;
    }
    sum = block_all<THREADS>(sum, s_f, Added());
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    write_spread<THREADS, REGS, 8>(to, cols, [&](int k) { return r[k] * inv; });
    if constexpr (KEPT > 0)
        write_spread<THREADS, KEPT, 4>(to + REGS * THREADS, cols - REGS * THREADS, [&](int k) { return s_x[k * THREADS + tid] * inv; });
}

// Few rows: pieces of SM_PIECE values, a workgroup each; first every piece's
// largest value, its index and the sum, then every piece's outputs from the row's
// (the second read is served by the caches).  17 x 151936: 3.7 + 6.1 us for 4.3 us of
// memory traffic, each kernel a launch and two or three dependent reads.
constexpr int SM_THREADS = 256, SM_REGS = 16, SM_PIECE = SM_THREADS * SM_REGS;
struct SoftPart { float m, sum; int at, pad; };

template <bool LAST>
__global__ __launch_bounds__(SM_THREADS) void softmax_piece_kernel(float *out, const float *x, int cols, SoftScale scale, SoftPart *parts) {
    __shared__ float s_f[4];
    __shared__ int s_i[4];
    const int pieces = (cols + SM_PIECE - 1) / SM_PIECE, which = blockIdx.x / pieces, piece = blockIdx.x % pieces;
    const int tid = threadIdx.x, c0 = piece * SM_PIECE, n = min(SM_PIECE, cols - c0);
    const float *row = x + (size_t)which * cols + c0, none = -__builtin_inff();
    parts += (size_t)which * pieces;
    float r[SM_REGS], m = none, sum = 0.0f;
    read_spread<SM_THREADS, SM_REGS, SM_REGS>(row, n, [&](int k, float v) { r[k] = v; });
    if (!LAST) {
#pragma unroll
        for (int k = 0; k < SM_REGS; k++) m = fmaxf(m, r[k]);
        m = block_all<SM_THREADS>(m, s_f, Larger());
        int at = 0;
        if (scale.b == 0.0f || m == none) {
            FirstOf first;
#pragma unroll
            for (int k = SM_REGS - 1; k >= 0; k--) first.see(k, r[k], m);
            at = block_all<SM_THREADS>(first.index<SM_THREADS>(), s_i, Lower());
        } else {
#pragma unroll
            for (int k = 0; k < SM_REGS; k++) sum += scale.power(r[k], m * scale.a);
            sum = block_all<SM_THREADS>(sum, s_f, Added());
        }
        if (tid == 0) parts[piece] = SoftPart{m, sum, at == SM_NAN ? SM_NAN : c0 + at, 0};
        return;
    }
    float *to = out + (size_t)which * cols + c0;
    for (int i = tid; i < pieces; i += SM_THREADS) m = fmaxf(m, parts[i].m);
    m = block_all<SM_THREADS>(m, s_f, Larger());
    const float ma = m * scale.a;
    int at = 0x7fffffff;
    for (int i = tid; i < pieces; i += SM_THREADS) {
        const SoftPart p = parts[i];
        if (p.at == SM_NAN) at = SM_NAN;
        else if (p.m == m) at = min(at, p.at);
        if (p.m != none) sum += p.sum * scale.power(p.m, ma);
    }
    sum = block_all<SM_THREADS>(sum, s_f, Added());
    at = block_all<SM_THREADS>(at, s_i, Lower());
    const bool nan = at == SM_NAN || m == __builtin_inff();
    const float inv = 1.0f / sum;
    const bool one = scale.b == 0.0f || m == none;
    write_spread<SM_THREADS, SM_REGS, SM_REGS>(to, n, [&](int k) {
        float y = scale.power(r[k], ma) * inv;
        if (one) y = m != none && c0 + k * SM_THREADS + tid == at ? 1.0f : 0.0f;
        return nan ? __builtin_nanf("") : y;
    });
}
// Pieces for long rows: always where a row is longer than a workgroup holds (96 rows of
// 200000: 38 us in pieces, 77 by rows; 512: 242 / 286), else while the rows are too
// few to fill the card (131072 columns: 64 rows 16.9 / 24.8, 96 26.9 / 27.8, 128 33.5 /
// 29.1; 70000: 64 11.3 / 20.3, 256 35.6 / 32.7).  Rows of up to 40960 are faster by
// rows however few (1 row of 32000: 8.0 / 6.8; 8192: 7.9 / 5.1).
constexpr int SM_SHORT = 40 * 1024, SM_HELD = (96 + 36) * 1024;
// The rows up to which rows of `cols` values go in pieces.
int softmax_piece_rows(int cols) { return cols > SM_HELD ? 0x7fffffff : cols > SM_SHORT ? 12999999 / cols : 0; }
bool softmax_pieces(int rows, int cols) { return rows <= softmax_piece_rows(cols); }
template <bool BEST>
void softmax_rows(float *out, const float *x, int rows, int cols, SoftScale scale, hipStream_t s) {
    if (cols <= 4096) softmax_row_kernel<256, 16, 0, BEST><<<rows, 256, 0, s>>>(out, x, cols, scale);
    else if (cols <= 16384) softmax_row_kernel<1024, 16, 0, BEST><<<rows, 1024, 0, s>>>(out, x, cols, scale);
    else if (cols <= SM_SHORT) softmax_row_kernel<1024, 40, 0, BEST><<<rows, 1024, 0, s>>>(out, x, cols, scale);
    else softmax_row_kernel<1024, 96, 36, BEST><<<rows, 1024, 0, s>>>(out, x, cols, scale);
}

// ------------------------------------------------------------------------
// Verification.  After j rejections at a row the target's distribution without
// the drafts' share is max(p_{j-1} - q, 0) / Z; written out from the first, that
// is max(p - a q, 0) / B with a += B at each rejection.  So a sum over the
// vocabulary depends on (row, a) alone, and the walk is a sequence of such sums
// with a little arithmetic between.  A sum is a launch over pieces of the
// vocabulary, whose workgroups all take the walk to the next sum by themselves;
// the last kernel draws the token.  A chain has one sum: it ends at its first
// rejection.
// ------------------------------------------------------------------------
constexpr int VF_THREADS = 256, VF_BLOCK = 4096, VF_LAST = 1024;

// A draft, in the lane of its place: its token and parent, its number, and its
// probabilities at the row that it continues.  Every wave holds them all.
struct Draft { float p, q, u; int token, up; };
struct Walk;
struct VerifyArgs {
    int *tokens_out, *path, *count;
    const float *p, *q, *u, *u_last;
    const int *token;
    int cols, piece, pieces; // a piece: whole blocks of VF_BLOCK tokens
    double *sums;            // [2][sequences][pieces], likewise
    Walk *walks;             // [sequences][2], the last round's and this one's
    Draft *drafts;           // [sequences][QG_MAX_TREE], as the first round read them
};
// Where a sequence's walk stands: the accepted rows, the rejected drafts of the
// current row, and what is left of its distribution.
struct Walk {
    unsigned long long taken, gone;
    double a, mass;
    int node, next, half, state;  // half: of sums, the one that holds this (row, a)'s
};
enum { WALK_SUM = 0, WALK_DRAW_SUM = 1, WALK_DRAW = 2 };  // needs a sum; needs one and then draws; draws

QG_DEV Draft read_draft(const VerifyArgs &A, const BatchView &b, int first, int n, int lane) {
    Draft d{0.0f, 0.0f, 0.0f, 0, -1};
    if (lane < n) {
        const int r = first + lane;
        d.token = A.token[r];
        d.up = b.parent ? tree_parent(b.parent[r], lane) : lane - 1;
        d.u = A.u[r];
        if ((unsigned)d.token >= (unsigned)A.cols) d.up = -1;
        if (d.up >= 0) {
            const size_t at = (size_t)(first + d.up) * A.cols + d.token;
            d.p = A.p[at];
            if (A.q) d.q = A.q[at];
        }
    }
    return d;
}
QG_DEV float lane_f(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }
QG_DEV unsigned long long same_u64(unsigned long long x) {  // of a value that all lanes share: in scalar registers
    return (unsigned long long)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)x);
}
// Takes the walk on until a sum is needed or a token can be drawn, by a whole wave.
// summed: mass is the sum of what is left at (node, a).
QG_DEV void walk_on(Walk &w, const Draft &d, bool sampled, bool summed) {
    for (;;) {
        // the row's drafts that are still to be tried, in order
        unsigned long long drafts = __ballot(d.up == w.node && (int)(threadIdx.x & 63) >= w.next);
        bool moved = false;
        for (; drafts && !moved; drafts &= drafts - 1) {
            const int i = __builtin_ctzll(drafts);
            const double u = (double)lane_f(d.u, i);
            double p = (double)lane_f(d.p, i);
            summed = false;
            if (sampled) {
                const double q = (double)lane_f(d.q, i);
                p -= w.a * q;
                moved = u * q * w.mass < p;
            } else {
                const int x = __builtin_amdgcn_readlane(d.token, i);
                if (__ballot(d.token == x) & w.gone) p = 0.0;
                moved = u * w.mass < p;
            }
            w.next = i + 1;
            if (moved) {
                w.taken |= 1ULL << i;
                w.node = i;
                w.a = 0.0; w.mass = 1.0; w.gone = 0;
            } else if (sampled) {
                w.a += w.mass;
                w.state = WALK_SUM;
                return;
            } else {
                w.mass -= p > 0.0 ? p : 0.0;
                w.gone |= 1ULL << i;
            }
        }
        if (!moved) break;
    }
    w.state = summed ? WALK_DRAW : WALK_DRAW_SUM;
}
// What is left of token i at a row: max(p - a q, 0), or p without the rejected tokens.
struct Left {
    const float *p, *q;
    double a;
    unsigned long long gone;
    int token;  // the lane's draft
    __device__ __forceinline__ double of(float pi, float qi, int i) const {
        double w = (double)pi;
        if (q) w -= a * (double)qi;
        else for (unsigned long long g = gone; g; g &= g - 1) w = __builtin_amdgcn_readlane(token, __builtin_ctzll(g)) == i ? 0.0 : w;
        return w > 0.0 ? w : 0.0;
    }
    __device__ __forceinline__ double at(int i) const { return of(p[i], q ? q[i] : 0.0f, i); }
};
QG_DEV Left left_of(const VerifyArgs &A, const Walk &w, const Draft &d, int first) {
    const size_t at = (size_t)(first + w.node) * A.cols;
    return Left{A.p + at, A.q ? A.q + at : nullptr, w.a, same_u64(w.gone), d.token};
}
// The sum over tokens c0 .. end - 1, in every thread of THREADS.
template <int THREADS>
QG_DEV double piece_sum(const Left &l, int c0, int end, double *s) {
    constexpr int R = VF_BLOCK / THREADS;
    double v = 0.0;
    for (; c0 + VF_BLOCK <= end; c0 += VF_BLOCK) {
        const float *at = l.p + c0 + threadIdx.x, *by = (l.q ? l.q : l.p) + c0 + threadIdx.x;
        float p[R], q[R];
#pragma unroll
        for (int k = 0; k < R; k++) p[k] = at[k * THREADS];
        if (l.q) {
#pragma unroll
            for (int k = 0; k < R; k++) q[k] = by[k * THREADS];
        }
#pragma unroll
        for (int k = 0; k < R; k++) v += l.of(p[k], q[k], c0 + k * THREADS + threadIdx.x);
    }
    for (int i = c0 + threadIdx.x; i < end; i += THREADS) v += l.at(i);
    return block_all<THREADS>(v, s, Added());
}
// The pieces' sums of the half that holds them, in order, 64 to a wave's lanes;
// both halves are read before it is known which (the first 64 of each, `ahead`).
struct Ahead { double v[2]; };
QG_DEV Ahead pieces_ahead(const VerifyArgs &A, int sequences, int s, int lane) {
    Ahead x;
#pragma unroll
    for (int h = 0; h < 2; h++) x.v[h] = lane < A.pieces ? A.sums[((size_t)h * sequences + s) * A.pieces + lane] : 0.0;
    return x;
}
QG_DEV double wave_upto(double v, int lane) {  // inclusive sums over the lanes
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const double y = __shfl_up(v, x);
        if (lane >= x) v += y;
    }
    return v;
}
// Their sum, in every lane of every wave.
QG_DEV double all_pieces(const double *sums, int pieces, double ahead, int lane) {
    double total = 0.0;
    for (int k0 = 0; k0 < pieces; k0 += 64)
        total += __shfl(wave_upto(k0 == 0 ? ahead : k0 + lane < pieces ? sums[k0 + lane] : 0.0, lane), 63);
    return total;
}

// One sum: workgroup x of sequence y takes the walk to its next sum and adds its
// piece of it.  round 0 starts the walk.  64 sequences x 131072 tokens: 14 us for the
// first sum (67 MB, 4.7 TB/s), then 4 to 6 for what few sequences still need; one
// sequence x 151936: 4 us, four dependent reads.
__global__ __launch_bounds__(VF_THREADS) void verify_sum_kernel(VerifyArgs A, BatchView b, int round) {
    __shared__ double s_red[4];
    const int s = blockIdx.y, lane = threadIdx.x & 63;
    int first, n;
    batch_rows(b, s, first, n);
    if (n == 0) return;
    Walk w{1, 0, 0.0, 1.0, 0, 1, 0, WALK_SUM};
    Draft d;
    if (round) {
        w = A.walks[s * 2 + ((round - 1) & 1)];
        if (w.state != WALK_SUM) {  // decided: the next kernel finds it where it looks
            if (blockIdx.x == 0 && threadIdx.x == 0) A.walks[s * 2 + (round & 1)] = w;
            return;
        }
        const Ahead x = pieces_ahead(A, gridDim.y, s, lane);
        d = A.drafts[s * QG_MAX_TREE + lane];
        w.mass = all_pieces(A.sums + ((size_t)w.half * gridDim.y + s) * A.pieces, A.pieces, w.half ? x.v[1] : x.v[0], lane);
    } else {
        d = read_draft(A, b, first, n, lane);
        if (blockIdx.x == 0 && threadIdx.x < QG_MAX_TREE) A.drafts[s * QG_MAX_TREE + lane] = d;
    }
    walk_on(w, d, A.q != nullptr, round > 0);
    if (w.state != WALK_DRAW) {
        w.half = round & 1;
        const int c0 = blockIdx.x * A.piece;
        const double v = piece_sum<VF_THREADS>(left_of(A, w, d, first), c0, min(c0 + A.piece, A.cols), s_red);
        if (threadIdx.x == 0) A.sums[((size_t)w.half * gridDim.y + s) * A.pieces + blockIdx.x] = v;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) A.walks[s * 2 + (round & 1)] = w;
}

// The rest of the walk and the last token, a workgroup per sequence.
__global__ __launch_bounds__(VF_LAST) void verify_draw_kernel(VerifyArgs A, BatchView b, int rounds) {
    __shared__ double s_red[16];
    __shared__ int2 s_got[VF_LAST / 64];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int first, n;
    batch_rows(b, s, first, n);
    int *tokens = A.tokens_out + (size_t)s * b.max_rows, *path = A.path + (size_t)s * b.max_rows;
    if (n == 0) {
        if (tid < b.max_rows) tokens[tid] = path[tid] = -1;
        if (tid == 0) A.count[s] = 0;
        return;
    }
    const Ahead x = pieces_ahead(A, gridDim.x, s, lane);
    Walk w = A.walks[s * 2 + ((rounds - 1) & 1)];
    const Draft d = A.drafts[s * QG_MAX_TREE + lane];
    double *sums = A.sums + ((size_t)w.half * gridDim.x + s) * A.pieces, ahead = (w.half ? x.v[1] : x.v[0]);
    auto sum_of = [&](const Left &l) {  // by this workgroup alone
        __syncthreads();
        for (int k = 0; k < A.pieces; k++) {
            const double v = piece_sum<VF_LAST>(l, k * A.piece, min((k + 1) * A.piece, A.cols), s_red);
            if (tid == 0) sums[k] = v;
        }
        __threadfence_block();
        __syncthreads();
        ahead = lane < A.pieces ? sums[lane] : 0.0;
        return all_pieces(sums, A.pieces, ahead, lane);
    };
    double total = all_pieces(sums, A.pieces, ahead, lane);
    while (w.state == WALK_SUM) {
        w.mass = total;
        walk_on(w, d, A.q != nullptr, true);
        if (w.state != WALK_DRAW) total = sum_of(left_of(A, w, d, first));
    }
    Left l = left_of(A, w, d, first);
    if (!(total > 0.0)) {  // nothing is left: the row's own distribution
        l = Left{l.p, nullptr, 0.0, 0, 0};
        total = sum_of(l);
    }
    // The piece in which the running sum passes the goal (the last one with something in it, should rounding keep it
    // below), then the token there.  Only tokens with something left are taken, so that the two steps' roundings
    // cannot pick another.
    const double goal = (double)A.u_last[s] * total;
    int pick = -1, piece = -1;
    double at = 0.0, before = 0.0;
    for (int k0 = 0; k0 < A.pieces; k0 += 64) {  // the same in every wave
        const double v = k0 == 0 ? ahead : k0 + lane < A.pieces ? sums[k0 + lane] : 0.0, upto = wave_upto(v, lane);
        const unsigned long long some = __ballot(v > 0.0), pass = __ballot(v > 0.0 && before + upto > goal);
        if (pass || some) {
            const int k = pass ? __builtin_ctzll(pass) : 63 - __builtin_clzll(some);
            piece = k0 + k;
            at = before + __shfl(upto, k) - __shfl(v, k);
        }
        if (pass) break;
        before += __shfl(upto, 63);
    }
    bool found = false;
    for (int c0 = piece * A.piece; piece >= 0 && !found && c0 < min((piece + 1) * A.piece, A.cols); c0 += VF_BLOCK) {
        double v[4], mine = 0.0;
        const int i0 = c0 + 4 * tid;  // four tokens in a row per thread
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = i0 + j < A.cols ? l.at(i0 + j) : 0.0;
            mine += v[j];
        }
        const double upto = wave_upto(mine, lane);
        __syncthreads();
        if (lane == 63) s_red[wave] = upto;
        __syncthreads();
        // each wave's first token past the goal, or its last one with something left
        double sum = at + (upto - mine), block = 0.0;
#pragma unroll
        for (int k = 0; k < VF_LAST / 64; k++) {
            const double x = s_red[k];
            block += x;
            if (k < wave) sum += x;
        }
        at += block;
        int past = -1, last = -1;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            sum += v[j];
            if (v[j] > 0.0) {
                last = i0 + j;
                if (sum > goal && past < 0) past = i0 + j;
            }
        }
        const unsigned long long passes = __ballot(past >= 0), some = __ballot(last >= 0);
        const int got = passes ? __shfl(past, __builtin_ctzll(passes)) : some ? __shfl(last, 63 - __builtin_clzll(some)) : -1;
        if (lane == 0) s_got[wave] = make_int2(got, passes != 0);
        __syncthreads();
        for (int k = 0; k < VF_LAST / 64 && !found; k++) {  // the first that passes, else the last one
            const int2 x = s_got[k];
            if (x.x >= 0) pick = x.x;
            found = x.y;
        }
    }
    // the accepted rows are an ascending path
    const int kept = __popcll(w.taken);
    if (tid >= kept && tid < b.max_rows) path[tid] = tokens[tid] = -1;
    if (tid < n && w.taken >> tid & 1) {
        const int k = __popcll(w.taken & ((1ULL << tid) - 1));
        path[k] = tid;
        if (k) tokens[k - 1] = d.token;
    }
    if (tid == 0) {
        tokens[kept - 1] = pick;
        A.count[s] = kept;
    }
}
// The tokens of a piece and their number: pieces of a block for few sequences, of
// more for many, whose workgroups are enough and whose walks then cost less.
struct Pieces { size_t x, y; };
Pieces verify_pieces(int sequences, int cols) {
    const size_t blocks = ((size_t)cols + VF_BLOCK - 1) / VF_BLOCK, per = (blocks * sequences + 2047) / 2048;
    return Pieces{per * VF_BLOCK, (blocks + per - 1) / per};
}
// No number of sequences up to this one has more pieces together: each has at most
// blocks / per + 1, and blocks * sequences / per is at most 2048.
size_t verify_sums(int sequences, int cols) {
    const size_t each = (((size_t)cols + VF_BLOCK - 1) / VF_BLOCK) * sequences, all = 2048 + (size_t)sequences;
    return each < all ? each : all;
}
// Sums by launches over the whole card; a tree's later ones (each takes another
// rejection with drafts left to try) are few and fall to the drawing workgroup.
// With 2 / 4 / 7: 64 trees of 17 rows x 131072 tokens 75 / 38 / 46 us, 16 of 33 x
// 50000 40 / 31 / 39, one of 17 x 151936 15 / 19 / 26.
int verify_rounds(const BatchView &b, bool sampled) { return b.parent && sampled ? 4 : 1; }

}  // namespace

extern "C" {

int qg_qk_norm_rope(float *q_out, float *k_out, const qg_qk_rows *in, const qg_kv_cache *cache, int layer, const qg_kv_batch *batch) {
    if (!in || !q_out || !in->q || !in->k || in->rows < 1 || in->rows > QG_MAX_ROWS) return hipErrorInvalidValue;
    const int D = in->head_dim;
    if ((D != 64 && D != 128 && D != 256) || in->q_heads < 1 || in->q_heads > 1024 || in->kv_heads < 1 || in->kv_heads > 1024)
        return hipErrorInvalidValue;
    if (in->rope_dims < 0 || in->rope_dims > D || in->rope_dims % 8 || (in->rope_dims && !in->freq)) return hipErrorInvalidValue;
    if (in->eps < 0.0f || in->eps != in->eps) return hipErrorInvalidValue;
    KvView c{};
    BatchView b{};
    if (cache) {
        if (qg_kv_check(cache, false, &c) || qg_batch_check(batch, false, &b)) return hipErrorInvalidValue;
        if (b.rows != in->rows || c.heads != in->kv_heads || c.dim != D || layer < 0 || layer >= c.layers || !in->v) return hipErrorInvalidValue;
    } else if (batch || (in->rope_dims && !in->position)) {
        return hipErrorInvalidValue;
    }
    const int64_t strides = in->q_row | in->q_head | in->k_row | in->k_head | (cache ? in->v_row | in->v_head : 0);
    const uintptr_t at = (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)in->q | (uintptr_t)in->k | (cache ? (uintptr_t)in->v : 0) |
                         (uintptr_t)in->q_norm | (uintptr_t)in->k_norm;
    if ((strides & 3) || (at & 15) || ((uintptr_t)in->freq & 7) || ((uintptr_t)in->position & 3)) return hipErrorInvalidValue;
    // the floats that each input spans; a stride may be 0 or larger than needed, never negative
    auto span = [&](int64_t row, int64_t head, int heads) { return 4 * (size_t)((in->rows - 1) * row + (heads - 1) * head + D); };
    const int64_t most = (int64_t)1 << 40;
    for (int64_t x : {in->q_row, in->q_head, in->k_row, in->k_head, cache ? in->v_row : 0, cache ? in->v_head : 0})
        if (x < 0 || x > most) return hipErrorInvalidValue;
    const size_t qn = 4 * (size_t)in->rows * in->q_heads * D, kn = 4 * (size_t)in->rows * in->kv_heads * D;
    const size_t qs = span(in->q_row, in->q_head, in->q_heads), ks = span(in->k_row, in->k_head, in->kv_heads);
    const bool q_own = q_out == in->q && in->q_head == D && in->q_row == (int64_t)in->q_heads * D;
    const bool k_own = k_out == in->k && in->k_head == D && in->k_row == (int64_t)in->kv_heads * D;
    if ((!q_own && qg_overlap(q_out, qn, in->q, qs)) || qg_overlap(q_out, qn, in->k, ks) || qg_overlap(q_out, qn, k_out, kn) ||
        (k_out && ((!k_own && qg_overlap(k_out, kn, in->k, ks)) || qg_overlap(k_out, kn, in->q, qs))))
        return hipErrorInvalidValue;
    if (cache) {
        const size_t vs = span(in->v_row, in->v_head, in->kv_heads);
        if (qg_overlap(q_out, qn, in->v, vs) || qg_overlap(k_out, kn, in->v, vs)) return hipErrorInvalidValue;
    }
    const RopeArgs A{q_out, k_out, in->q, in->k, in->v, in->q_row, in->q_head, in->k_row, in->k_head, in->v_row, in->v_head,
                     in->q_norm, in->k_norm, in->freq, in->position, in->eps, in->rows, in->q_heads, in->kv_heads, in->rope_dims,
                     in->interleaved != 0, cache != nullptr};
    if (D == 64) launch_rope<64>(A, c, b, layer, qg_stream());
    else if (D == 128) launch_rope<128>(A, c, b, layer, qg_stream());
    else launch_rope<256>(A, c, b, layer, qg_stream());
    return hipGetLastError();
}

size_t qg_softmax_workspace_bytes(int rows, int cols) {
    if (rows < 1 || rows > QG_MAX_ROWS || cols < 1 || cols > 1 << 24 || (long)rows * cols > 1L << 35) return 0;
    // of every number of rows up to this one, the largest that goes in pieces
    const int most = rows < softmax_piece_rows(cols) ? rows : softmax_piece_rows(cols);
    return most ? (size_t)most * ((cols + SM_PIECE - 1) / SM_PIECE) * sizeof(SoftPart) : sizeof(SoftPart);
}

int qg_softmax(float *out, const float *x, int rows, int cols, float temperature, void *ws, size_t ws_bytes) {
    const size_t need = qg_softmax_workspace_bytes(rows, cols);
    if (!need || !out || !x || !ws || ws_bytes < need || (((uintptr_t)out | (uintptr_t)x) & 3) || ((uintptr_t)ws & 15)) return hipErrorInvalidValue;
    if (!(temperature == 0.0f || temperature >= 0x1p-126f) || !__builtin_isfinite(temperature)) return hipErrorInvalidValue;
    const size_t bytes = 4 * (size_t)rows * cols;
    if ((out != x && qg_overlap(out, bytes, x, bytes)) || qg_overlap(ws, need, x, bytes) || qg_overlap(ws, need, out, bytes)) return hipErrorInvalidValue;
    const float a = temperature >= 0x1p64f ? 0x1p-64f : 1.0f;
    const SoftScale scale{a, temperature > 0.0f ? 1.44269504088896341f / (temperature * a) : 0.0f};
    if (softmax_pieces(rows, cols)) {
        const unsigned grid = (unsigned)((cols + SM_PIECE - 1) / SM_PIECE * rows);
        softmax_piece_kernel<false><<<grid, SM_THREADS, 0, qg_stream()>>>(out, x, cols, scale, (SoftPart *)ws);
        softmax_piece_kernel<true><<<grid, SM_THREADS, 0, qg_stream()>>>(out, x, cols, scale, (SoftPart *)ws);
    } else if (scale.b > 0.0f) {
        softmax_rows<false>(out, x, rows, cols, scale, qg_stream());
    } else {
        softmax_rows<true>(out, x, rows, cols, scale, qg_stream());
    }
    return hipGetLastError();
}

size_t qg_verify_workspace_bytes(int sequences, int cols) {
    if (sequences < 1 || sequences > QG_MAX_SEQUENCES || cols < 1 || cols > 1 << 24) return 0;
    return 2 * (verify_sums(sequences, cols) * sizeof(double) + (size_t)sequences * sizeof(Walk)) + (size_t)sequences * QG_MAX_TREE * sizeof(Draft);
}

int qg_verify_drafts(int *tokens_out, int *path, int *count, const float *p, const float *q, const int *token, const float *u,
                     const float *u_last, int cols, int sequences, const qg_kv_batch *batch, void *ws, size_t ws_bytes) {
    BatchView b;
    const size_t need = qg_verify_workspace_bytes(sequences, cols);
    if (!need || qg_batch_check(batch, true, &b)) return hipErrorInvalidValue;
    if (!tokens_out || !path || !count || !p || !token || !u || !u_last || !ws || ws_bytes < need || ((uintptr_t)ws & 15)) return hipErrorInvalidValue;
    if (((uintptr_t)tokens_out | (uintptr_t)path | (uintptr_t)count | (uintptr_t)p | (uintptr_t)q | (uintptr_t)token | (uintptr_t)u |
         (uintptr_t)u_last) & 3)
        return hipErrorInvalidValue;
    const size_t vb = 4 * (size_t)b.rows * cols, ob = 4 * (size_t)sequences * b.max_rows, cb = 4 * (size_t)sequences;
    // the last kernel writes the outputs where its other workgroups read; the first ones read every input and write the workspace
    const QgSpan out[3] = {{tokens_out, ob}, {path, ob}, {count, cb}}, space[1] = {{ws, need}},
                 all_along[4] = {{p, vb}, {q, vb}, {u_last, cb}, {b.start, qg_ints((size_t)sequences + 1)}},
                 first[3] = {{token, qg_ints(b.rows)}, {u, qg_ints(b.rows)}, {b.parent, qg_ints(b.rows)}};
    if (qg_any_overlap(out, space) || qg_any_overlap(out, all_along) || qg_any_overlap(space, all_along) || qg_any_overlap(space, first) ||
        qg_overlap(tokens_out, ob, path, ob) || qg_overlap(tokens_out, ob, count, cb) || qg_overlap(path, ob, count, cb))
        return hipErrorInvalidValue;
    const Pieces pieces = verify_pieces(sequences, cols);
    const int rounds = verify_rounds(b, q != nullptr);
    Walk *walks = (Walk *)ws;
    const VerifyArgs A{tokens_out, path, count, p, q, u, u_last, token, cols, (int)pieces.x, (int)pieces.y, (double *)(walks + 2 * sequences), walks,
                       (Draft *)((double *)(walks + 2 * sequences) + 2 * (size_t)sequences * pieces.y)};
    for (int r = 0; r < rounds; r++) verify_sum_kernel<<<dim3((unsigned)pieces.y, sequences), VF_THREADS, 0, qg_stream()>>>(A, b, r);
    verify_draw_kernel<<<sequences, VF_LAST, 0, qg_stream()>>>(A, b, rounds);
    return hipGetLastError();
}

}  // extern "C"
