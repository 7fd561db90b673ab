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

template <int D>
__global__ __launch_bounds__(256) void qk_rope_kernel(RopeArgs A, KvView c, BatchView b, int layer) {
    constexpr int LPH = D / 4, HPW = 64 / LPH;  // lanes per head, heads per wave
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x;
    const int d = (lane % LPH) * 4, h = (blockIdx.y * 4 + wave) * HPW + lane / LPH;
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
    const int kind = h < A.q_heads ? 0 : h < A.q_heads + A.kv_heads ? 1 : 2;
    const int head = kind == 0 ? h : h - A.q_heads - (kind == 2 ? A.kv_heads : 0);
    const bool live = h < A.q_heads + A.kv_heads * (A.cached ? 2 : 1);
    const float *src = kind == 0 ? A.q + row * A.q_row + head * A.q_head : kind == 1 ? A.k + row * A.k_row + head * A.k_head
                                                                                 : A.v + row * A.v_row + head * A.v_head;
    float4 x4 = live ? *(const float4 *)(src + d) : make_float4(0, 0, 0, 0);
    float x[4] = {x4.x, x4.y, x4.z, x4.w};
    const float *w = kind == 0 ? A.q_norm : A.k_norm;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) ss = __builtin_fmaf(x[i], x[i], ss);
    ss = qg_row_sum(ss);
    if (LPH >= 32) ss += __shfl_xor(ss, 16);
    if (LPH >= 64) ss += __shfl_xor(ss, 32);
    if (kind < 2 && w) {
        const float scale = 1.0f / __builtin_sqrtf(ss / (float)D + A.eps);
        const float4 w4 = *(const float4 *)(w + d);
        x[0] = x[0] * scale * w4.x;
        x[1] = x[1] * scale * w4.y;
        x[2] = x[2] * scale * w4.z;
        x[3] = x[3] * scale * w4.w;
    }
    if (A.rope) {
        const int half = A.rope / 2;
        float y[4];
        if (A.interleaved) {
            const int f = min(d, A.rope - 4) / 2;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float sn, cs;
                turn_of((double)pos * A.freq[f + i], sn, cs);
                y[2 * i] = x[2 * i] * cs - x[2 * i + 1] * sn;
                y[2 * i + 1] = x[2 * i + 1] * cs + x[2 * i] * sn;
            }
        } else {
            const bool low = d < half;
            const int other = lane + (low ? half / 4 : -(half / 4)), f = d < A.rope ? (low ? d : d - half) : 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __shfl(x[i], other & 63);
                float sn, cs;
                turn_of((double)pos * A.freq[f + i], sn, cs);
                y[i] = low ? x[i] * cs - p * sn : x[i] * cs + p * sn;
            }
        }
        if (kind < 2 && d < A.rope) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = y[i];
        }
    }
    if (!live) return;
    if (kind == 0) {
        *(float4 *)(A.q_out + ((size_t)row * A.q_heads + head) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
        return;
    }
    if (kind == 1 && A.k_out) *(float4 *)(A.k_out + ((size_t)row * A.kv_heads + head) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
    if (page < 0) return;
    uint8_t *pool = kind == 1 ? c.k : c.v;
    const size_t at = kv_at(c, layer, page, head, slot) + d;
    if (c.type == QT_F32) {
        *(float4 *)((float *)pool + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = c.type == QT_F16 ? kv_f16(x[i]) : kv_bf16(x[i]);
        *(uint2 *)((uint16_t *)pool + at) = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
    }
}

// ------------------------------------------------------------------------
// Softmax of a row: e_i = exp((x_i - m) / T), out = e_i / sum e.
// ------------------------------------------------------------------------
constexpr int SM_THREADS = 1024;

// The largest of two values; NaN if either is.
QG_DEV float max_nan(float a, float b) { return a != a || a > b ? a : b; }

// A workgroup's value by `op`, in every thread; s[16] is scratch.
template <typename T, typename F>
QG_DEV T block_all(T v, T *s, F op) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = op(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int w = 1; w < SM_THREADS / 64; w++) v = op(v, s[w]);
    return v;
}

__global__ __launch_bounds__(SM_THREADS) void softmax_row_kernel(float *out, const float *x, int cols, float inv) {
    __shared__ float s_f[16];
    __shared__ int s_i[16];
    const float *row = x + (size_t)blockIdx.x * cols;
    float *to = out + (size_t)blockIdx.x * cols;
    float m = -__builtin_inff();
    for (int i = threadIdx.x; i < cols; i += SM_THREADS) m = max_nan(row[i], m);
    m = block_all(m, s_f, max_nan);
    if (m == -__builtin_inff()) {
        for (int i = threadIdx.x; i < cols; i += SM_THREADS) to[i] = 0.0f;
        return;
    }
    if (!__builtin_isfinite(m)) {
        for (int i = threadIdx.x; i < cols; i += SM_THREADS) to[i] = __builtin_nanf("");
        return;
    }
    if (inv == 0.0f) {  // temperature 0
        int at = cols;
        for (int i = cols - 1 - threadIdx.x; i >= 0; i -= SM_THREADS) if (row[i] == m) at = i;
        at = block_all(at, s_i, [](int a, int b) { return min(a, b); });
        for (int i = threadIdx.x; i < cols; i += SM_THREADS) to[i] = i == at ? 1.0f : 0.0f;
        return;
    }
    float sum = 0.0f;
    for (int i = threadIdx.x; i < cols; i += SM_THREADS) sum += expf((row[i] - m) * inv);
    sum = block_all(sum, s_f, [](float a, float b) { return a + b; });
    for (int i = threadIdx.x; i < cols; i += SM_THREADS) to[i] = expf((row[i] - m) * inv) / sum;
}

// ------------------------------------------------------------------------
// Verification.  A workgroup per sequence.  After j rejections at a row the
// target's distribution without the drafts' share is max(p_{j-1} - q, 0) / Z;
// written out from the first that is max(p - a q, 0) / B with a += B at each
// rejection, so every pass reads p and q alone and nothing is kept per token.
// ------------------------------------------------------------------------
constexpr int VF_TILE = 4 * SM_THREADS, VF_TILES = (1 << 24) / VF_TILE;

struct VerifyArgs {
    int *tokens_out, *path, *count;
    const float *p, *q, *u, *u_last;
    const int *token;
    int cols;
};
// What is left of token i at a row: w = max(p - a q, 0), or p without the
// rejected tokens drop[0..drops).
struct Left {
    const float *p, *q;
    double a;
    const int *drop;
    int drops;
};
QG_DEV double left_at(const Left &l, int i) {
    double w = (double)l.p[i];
    if (l.q) w -= l.a * (double)l.q[i];
    else for (int k = 0; k < l.drops; k++) w = i == l.drop[k] ? 0.0 : w;
    return w > 0.0 ? w : 0.0;
}
// The sum of what is left, tile by tile (s_tile keeps the tiles' sums).
QG_DEV double left_sum(const Left &l, int cols, double *s_red, double *s_tile) {
    double total = 0.0;
    for (int t = 0; t * VF_TILE < cols; t++) {
        double v = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = t * VF_TILE + j * SM_THREADS + threadIdx.x;
            if (i < cols) v += left_at(l, i);
        }
        v = block_all(v, s_red, [](double a, double b) { return a + b; });
        if (threadIdx.x == 0) s_tile[t] = v;
        total += v;
    }
    __syncthreads();
    return total;
}
// The first token whose running sum passes goal (0 <= goal < total): its tile,
// then its place there.  Only tokens with something left are taken, so sums that
// round differently in the two steps cannot pick another.
QG_DEV int left_pick(const Left &l, int cols, double goal, double *s_red, const double *s_tile, int *s_int) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, tiles = (cols + VF_TILE - 1) / VF_TILE;
    double before = 0.0;
    int tile = -1;
    double at = 0.0;
    for (int t = 0; t < tiles; t++) {  // the last tile with something in it, should none pass
        const double v = s_tile[t];
        if (v > 0.0) { tile = t; at = before; if (before + v > goal) break; }
        before += v;
    }
    if (tile < 0) return -1;
    int last = -1;
    for (int j = 0; j < 4; j++) {
        const int i = tile * VF_TILE + j * SM_THREADS + tid;
        const double w = i < cols ? left_at(l, i) : 0.0;
        double sum = w;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double y = __shfl_up(sum, d);
            if (lane >= d) sum += y;
        }
        __syncthreads();
        if (lane == 63) s_red[wave] = sum;
        if (tid < 2) s_int[tid] = tid ? -1 : 0x7fffffff;
        __syncthreads();
        double all = 0.0;
        for (int k = 0; k < SM_THREADS / 64; k++) {
            if (k == wave) sum += at + all;
            all += s_red[k];
        }
        at += all;
        if (w > 0.0) {
            atomicMax(&s_int[1], i);
            if (sum > goal) atomicMin(&s_int[0], i);
        }
        __syncthreads();
        if (s_int[0] != 0x7fffffff) return s_int[0];
        last = max(last, s_int[1]);
    }
    return last;
}

__global__ __launch_bounds__(SM_THREADS) void verify_kernel(VerifyArgs A, BatchView b) {
    __shared__ double s_red[16], s_tile[VF_TILES];
    __shared__ float s_p[QG_MAX_TREE], s_q[QG_MAX_TREE], s_u[QG_MAX_TREE];
    __shared__ int s_tok[QG_MAX_TREE], s_up[QG_MAX_TREE], s_drop[QG_MAX_TREE], s_int[2];
    const int s = blockIdx.x, tid = threadIdx.x;
    int first, n;
    batch_rows(b, s, first, n);
    int *tokens = A.tokens_out + (size_t)s * b.max_rows, *path = A.path + (size_t)s * b.max_rows;
    if (tid < b.max_rows) tokens[tid] = path[tid] = -1;
    if (n == 0) {
        if (tid == 0) A.count[s] = 0;
        return;
    }
    if (tid < n) {
        const int r = first + tid, x = A.token[r];
        int up = b.parent ? tree_parent(b.parent[r], tid) : tid - 1;
        if ((unsigned)x >= (unsigned)A.cols) up = -1;
        s_tok[tid] = x;
        s_up[tid] = up;
        s_u[tid] = A.u[r];
        const size_t at = (size_t)(first + max(up, 0)) * A.cols + x;
        s_p[tid] = up >= 0 ? A.p[at] : 0.0f;
        s_q[tid] = up >= 0 && A.q ? A.q[at] : 0.0f;
    }
    __syncthreads();
    int node = 0, kept = 0, drops = 0;
    double a = 0.0, mass = 1.0;
    if (tid == 0) path[0] = 0;
    for (int i = 1; i < n; i++) {  // the same walk in every thread
        if (s_up[i] != node) continue;
        const double u = (double)s_u[i];
        double p = (double)s_p[i];
        bool accept;
        if (A.q) {
            const double q = (double)s_q[i];
            p -= a * q;
            accept = u * q * mass < p;
        } else {
            for (int k = 0; k < drops; k++) if (s_drop[k] == s_tok[i]) p = 0.0;
            accept = u * mass < p;
        }
        if (accept) {
            if (tid == 0) { tokens[kept] = s_tok[i]; path[kept + 1] = i; }
            kept++;
            node = i;
            a = 0.0; mass = 1.0; drops = 0;
            continue;
        }
        if (A.q) {
            a += mass;
            const size_t at = (size_t)(first + node) * A.cols;
            mass = left_sum(Left{A.p + at, A.q + at, a, nullptr, 0}, A.cols, s_red, s_tile);
        } else {
            mass -= p > 0.0 ? p : 0.0;
            __syncthreads();
            if (tid == 0) s_drop[drops] = s_tok[i];
            drops++;
            __syncthreads();
        }
    }
    const size_t at = (size_t)(first + node) * A.cols;
    Left l{A.p + at, A.q ? A.q + at : nullptr, a, s_drop, drops};
    double total = left_sum(l, A.cols, s_red, s_tile);
    if (!(total > 0.0)) {
        l = Left{A.p + at, nullptr, 0.0, s_drop, 0};
        total = left_sum(l, A.cols, s_red, s_tile);
    }
    const int pick = left_pick(l, A.cols, (double)A.u_last[s] * total, s_red, s_tile, s_int);
    if (tid == 0) { tokens[kept] = pick; A.count[s] = kept + 1; }
}

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
    const int heads = in->q_heads + in->kv_heads * (cache ? 2 : 1), per = 4 * (256 / D);
    const dim3 grid(in->rows, (heads + per - 1) / per);
    if (D == 64) qk_rope_kernel<64><<<grid, 256, 0, qg_stream()>>>(A, c, b, layer);
    else if (D == 128) qk_rope_kernel<128><<<grid, 256, 0, qg_stream()>>>(A, c, b, layer);
    else qk_rope_kernel<256><<<grid, 256, 0, qg_stream()>>>(A, c, b, layer);
    return hipGetLastError();
}

size_t qg_softmax_workspace_bytes(int rows, int cols) {
    if (rows < 1 || rows > QG_MAX_ROWS || cols < 1 || cols > 1 << 24) return 0;
    return 16;
}

int qg_softmax(float *out, const float *x, int rows, int cols, float temperature, void *ws, size_t ws_bytes) {
    const size_t need = qg_softmax_workspace_bytes(rows, cols);
    if (!need || !out || !x || !ws || ws_bytes < need || (((uintptr_t)out | (uintptr_t)x) & 3) || ((uintptr_t)ws & 15)) return hipErrorInvalidValue;
    if (!(temperature >= 0.0f) || !__builtin_isfinite(temperature)) return hipErrorInvalidValue;
    const size_t bytes = 4 * (size_t)rows * cols;
    if (out != x && qg_overlap(out, bytes, x, bytes)) return hipErrorInvalidValue;
    softmax_row_kernel<<<rows, SM_THREADS, 0, qg_stream()>>>(out, x, cols, temperature > 0.0f ? 1.0f / temperature : 0.0f);
    return hipGetLastError();
}

size_t qg_verify_workspace_bytes(int sequences, int cols) {
    if (sequences < 1 || sequences > QG_MAX_SEQUENCES || cols < 1 || cols > 1 << 24) return 0;
    return 16;
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
    const VerifyArgs A{tokens_out, path, count, p, q, u, u_last, token, cols};
    verify_kernel<<<sequences, SM_THREADS, 0, qg_stream()>>>(A, b);
    return hipGetLastError();
}

}  // extern "C"
