// Truncated distributions of logits (qg_sample, qg_sampling_softmax of
// include/qwen_gpu.h): temperature, top-k, top-p and min-p of each row, tokens
// drawn from what is left, or its probabilities.
//
// Weights are w_i = 2^((x_i - max) log2 e / T), in 64 bits wherever they are
// added up: which token a draw meets, and where a nucleus ends, are borders in a
// sum over the vocabulary, and an error of 1e-7 there (fp32) would move about one
// draw in two thousand to the next token.  All three filters keep the tokens from
// some value on and, of those that equal it, the first few: a cut (value, index).
// A cut is found by counting and weighing values by the leading bits of keys whose
// order is theirs; nothing is sorted.
#include "qg_kv.h"

namespace {

constexpr int SA_THREADS = 1024, SA_WAVES = SA_THREADS / 64, SA_DIGIT = 11, SA_BINS = 1 << SA_DIGIT, SA_PIECE = 4096;
constexpr int SA_MAX_COLS = 1 << 24, SA_MAX_DRAWS = 64;

struct SampleArgs {
    const float *x, *temperature, *top_p, *min_p, *u;
    const int *top_k;
    float *out, *logprob;
    int *token;
    int cols, draws, fixed;  // fixed: weights are added up as whole numbers of 2^-fixed where their order is not given
};

// Unsigned keys in the values' order; the zeros of both signs are one value.
QG_DEV uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
QG_DEV float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// 2^d for d <= 0, within 2^-52: the Taylor series of e^r, |r| <= ln 2 / 2, whose
// next term is below 1e-17.
QG_DEV double exp2_d(double d) {
    if (!(d > -1100.0)) return 0.0;
    const double n = __builtin_rint(d), r = (d - n) * 0.693147180559945309417;
    double p = 1.0 / 6227020800.0;
    const double c[13] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800,
                          1.0 / 39916800, 1.0 / 479001600};
#pragma unroll
    for (int i = 12; i >= 0; i--) p = __builtin_fma(p, r, c[i]);
    return __builtin_amdgcn_ldexp(p, (int)n);
}

// What a row asks for.  Temperature 0 (or none that counts) is the first largest
// token: top-k 1.
struct Request {
    double a, top_p, min_p;
    int top_k;
};
QG_DEV Request read_request(const SampleArgs &A, int row) {
    const float T = A.temperature ? A.temperature[row] : 1.0f, p = A.top_p ? A.top_p[row] : 1.0f, least = A.min_p ? A.min_p[row] : 0.0f;
    const int k = A.top_k ? A.top_k[row] : 0;
    Request r{1.0, 1.0, 0.0, 1};
    if (!(T >= 0x1p-126f)) return r;
    r.a = 1.44269504088896340736 / (double)fminf(T, 0x1.fffffep127f);
    r.top_k = k > 0 && k < A.cols ? k : 0;
    if (p < 1.0f) r.top_p = fmaxf(p, 0.0f);
    if (least > 0.0f) r.min_p = fminf(least, 1.0f);
    return r;
}

// Tokens stay whose key is above t, or equal to it up to index last.
struct Cut {
    uint32_t t = 0;
    int last = 0x7fffffff;
    __device__ __forceinline__ bool keeps(uint32_t key, int i) const { return key > t || (key == t && i <= last); }
};

template <typename T>
QG_DEV T wave_all_add(T v) {
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) v += __shfl_xor(v, d);
    return v;
}
template <typename T>
QG_DEV T wave_upto(T v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const T o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
// f(i, x_i) for the values of a row that are a thread's, eight on their way at once
template <int STEP, typename F>
QG_DEV void each_value(const float *x, int i0, int end, F f) {
    for (; i0 < end; i0 += 8 * STEP) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = i0 + k * STEP < end ? x[i0 + k * STEP] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (i0 + k * STEP < end) f(i0 + k * STEP, v[k]);
    }
}

struct RowShared {
    union {
        struct { unsigned long long mass[SA_BINS]; unsigned count[SA_BINS]; };
        double piece[SA_MAX_COLS / SA_PIECE];
    };
    unsigned long long wave_mass[SA_WAVES], found_mass, found_own;
    unsigned wave_count[SA_WAVES], found_count, found_ties;
    int found_bin, bad;
    float wave_max[SA_WAVES];
};

// A row of any shape by one workgroup, which reads it again for every step.
struct Row {
    const SampleArgs &A;
    RowShared &s;
    const float *x;
    const int tid, lane, wave;
    double a;
    float m;

    __device__ __forceinline__ double weight(float v) const { return exp2_d(((double)v - (double)m) * a); }
    __device__ __forceinline__ unsigned long long fixed(float v) const { return (unsigned long long)__builtin_rint(__builtin_amdgcn_ldexp(weight(v), A.fixed)); }

    // The largest value; false where nothing can be drawn from the row.
    __device__ bool largest() {
        float top = -__builtin_inff();
        bool nan = false;
        each_value<SA_THREADS>(x, tid, A.cols, [&](int, float v) { top = fmaxf(top, v); nan |= v != v; });
        top = qg_wave_max(top);
        if (__any(nan)) top = __builtin_nanf("");
        if (lane == 0) s.wave_max[wave] = top;
        __syncthreads();
        m = s.wave_max[0];
        for (int w = 1; w < SA_WAVES; w++) {
            const float o = s.wave_max[w];
            m = m != m || o != o ? __builtin_nanf("") : fmaxf(m, o);
        }
        __syncthreads();
        return __builtin_isfinite(m);
    }

    // From the cut's tokens in falling order the first ones that reach `goal` tokens
    // (by_mass false), or the share goal of their weight: never none.
    __device__ void shorten(Cut &cut, bool by_mass, double goal) {
        uint32_t prefix = 0;
        unsigned long long above = 0;
        unsigned over = 0;
        double need = goal;
        for (int left = 32; left > 0;) {
            const int bits = left < SA_DIGIT ? left : SA_DIGIT;
            const int shift = left - bits;
            for (int b = tid; b < SA_BINS; b += SA_THREADS) { s.mass[b] = 0; s.count[b] = 0; }
            __syncthreads();
            each_value<SA_THREADS>(x, tid, A.cols, [&](int i, float v) {
                const uint32_t key = order_key(v);
                if ((left < 32 && (key >> left) != prefix) || !cut.keeps(key, i)) return;
                const int bin = (key >> shift) & (SA_BINS - 1) & ((1 << bits) - 1);
                atomicAdd(&s.count[bin], 1u);
                if (by_mass) atomicAdd(&s.mass[bin], fixed(v));
            });
            __syncthreads();
            // sums from the largest bin down, two bins a thread
            const int b1 = SA_BINS - 1 - 2 * tid, b0 = b1 - 1;
            const unsigned c1 = s.count[b1], c0 = s.count[b0];
            const unsigned long long m1 = s.mass[b1], m0 = s.mass[b0];
            unsigned c = wave_upto(c1 + c0, lane);
            unsigned long long w = wave_upto(m1 + m0, lane);
            if (lane == 63) { s.wave_count[wave] = c; s.wave_mass[wave] = w; }
            if (tid == 0) s.found_bin = -1;
            __syncthreads();
            unsigned long long all = 0;
            for (int k = 0; k < SA_WAVES; k++) {
                if (k < wave) { c += s.wave_count[k]; w += s.wave_mass[k]; }
                all += s.wave_mass[k];
            }
            if (left == 32 && by_mass) need = goal * (double)all;
            c += over;
            w += above;
            // the first bin with which there is enough
            auto enough = [&](unsigned cc, unsigned long long ww) { return cc > 0 && (by_mass ? (double)ww >= need : cc >= (unsigned)need); };
            const bool e1 = c1 && enough(c - c0, w - m0), e0 = c0 && enough(c, w);
            const bool was1 = enough(c - c0 - c1, w - m0 - m1), was0 = enough(c - c0, w - m0);
            if (e1 && !was1) { s.found_bin = b1; s.found_count = c - c0 - c1; s.found_mass = w - m0 - m1; s.found_ties = c1; s.found_own = m1; }
            if (e0 && !was0) { s.found_bin = b0; s.found_count = c - c0; s.found_mass = w - m0; s.found_ties = c0; s.found_own = m0; }
            __syncthreads();
            if (s.found_bin < 0) return;  // more is asked for than there is
            prefix = prefix << bits | (uint32_t)s.found_bin;
            over = s.found_count;
            above = s.found_mass;
            left = shift;
            __syncthreads();
        }
        // of the equal ones the first r
        const unsigned ties = s.found_ties;
        unsigned r = ties;
        if (!by_mass) {
            r = (unsigned)need - over;
        } else if (ties > 1) {
            const double each = (double)(s.found_own / ties);
            const double n = __builtin_ceil((need - (double)above) / each);
            r = n >= ties ? ties : n < 1.0 ? 1 : (unsigned)n;
        }
        if (r < ties) cut.last = nth(prefix, cut, r);
        else if (prefix != cut.t) cut.last = 0x7fffffff;
        cut.t = prefix;
        __syncthreads();
    }
    // The index of the r-th of the cut's tokens with key t (r from 1), which there are.
    __device__ int nth(uint32_t t, const Cut &cut, unsigned r) {
        const int per = ((A.cols + SA_WAVES - 1) / SA_WAVES + 63) / 64 * 64, i0 = wave * per, end = min(i0 + per, A.cols);
        unsigned n = 0;
        each_value<64>(x, i0 + lane, end, [&](int i, float v) { n += order_key(v) == t && cut.keeps(t, i); });
        n = wave_all_add(n);
        __syncthreads();
        if (lane == 0) s.wave_count[wave] = n;
        __syncthreads();
        unsigned before = 0;
        for (int k = 0; k < wave; k++) before += s.wave_count[k];
        if (before < r && r <= before + n) {
            for (int i = i0; i < end; i += 64) {
                const bool is = i + lane < end && order_key(x[i + lane]) == t && cut.keeps(t, i + lane);
                unsigned long long all = __ballot(is);
                const unsigned here = __popcll(all);
                if (before + here >= r) {
                    for (unsigned k = before + 1; k < r; k++) all &= all - 1;
                    if (lane == 0) s.found_bin = i + __builtin_ctzll(all);
                    break;
                }
                before += here;
            }
        }
        __syncthreads();
        return s.found_bin;
    }
    // The least key whose weight is at least `least` (0 < least <= 1): a search in 64 ways, by every wave.
    __device__ uint32_t least_key(double least) const {
        uint32_t lo = 0x007fffffu, hi = order_key(m);  // lo's weight is less, hi's is not
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo - 1) / 64 + 1, k = lo + min((uint32_t)(lane + 1) * step, hi - lo);
            const unsigned long long ok = __ballot(weight(key_value(k)) >= least);
            const int first = __builtin_ctzll(ok);  // the last lane's is hi's
            const uint32_t up = lo + min((uint32_t)(first + 1) * step, hi - lo);
            lo += min((uint32_t)first * step, hi - lo);
            hi = up;
        }
        return hi;
    }
};

template <bool DRAW>
__global__ __launch_bounds__(SA_THREADS) void sample_row_kernel(SampleArgs A) {
    __shared__ RowShared s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Request q = read_request(A, row);
    Row r{A, s, A.x + (size_t)row * A.cols, tid, lane, wave, q.a, 0.0f};
    const bool some = r.largest();
    float *out = DRAW ? nullptr : A.out + (size_t)row * A.cols;
    if (!some) {
        if (DRAW) {
            if (tid < A.draws) {
                A.token[(size_t)row * A.draws + tid] = -1;
                if (A.logprob) A.logprob[(size_t)row * A.draws + tid] = __builtin_nanf("");
            }
        } else {
            const float none = r.m == -__builtin_inff() ? 0.0f : __builtin_nanf("");
            for (int i = tid; i < A.cols; i += SA_THREADS) out[i] = none;
        }
        return;
    }
    Cut cut;
    if (q.top_k) r.shorten(cut, false, q.top_k);
    if (q.top_p < 1.0) r.shorten(cut, true, q.top_p);
    if (q.min_p > 0.0) {
        const uint32_t k = r.least_key(q.min_p);
        if (k > cut.t) cut = Cut{k, 0x7fffffff};
    }
    // sums of pieces, each by one wave
    const int pieces = (A.cols + SA_PIECE - 1) / SA_PIECE;
    __syncthreads();
    for (int p = wave; p < pieces; p += SA_WAVES) {
        double sum = 0.0;
        each_value<64>(r.x, p * SA_PIECE + lane, min((p + 1) * SA_PIECE, A.cols), [&](int i, float v) { sum += cut.keeps(order_key(v), i) ? r.weight(v) : 0.0; });
        sum = wave_all_add(sum);
        if (lane == 0) s.piece[p] = sum;
    }
    __syncthreads();
    double total = 0.0;
    for (int p0 = 0; p0 < pieces; p0 += 64) total += wave_all_add(p0 + lane < pieces ? s.piece[p0 + lane] : 0.0);
    if (!DRAW) {
        each_value<SA_THREADS>(r.x, tid, A.cols, [&](int i, float v) { out[i] = cut.keeps(order_key(v), i) ? (float)(r.weight(v) / total) : 0.0f; });
        return;
    }
    for (int d = wave; d < A.draws; d += SA_WAVES) {
        const size_t at = (size_t)row * A.draws + d;
        const double goal = (double)A.u[at] * total;
        // the piece that passes the goal, or the last one that holds something
        double before = 0.0;
        int piece = -1;
        bool past = false;
        for (int p0 = 0; p0 < pieces && !past; p0 += 64) {
            const double v = p0 + lane < pieces ? s.piece[p0 + lane] : 0.0, upto = wave_upto(v, lane) + before;
            const unsigned long long hit = __ballot(v > 0.0 && upto > goal), any = __ballot(v > 0.0);
            if (!any) continue;
            const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
            piece = p0 + l;
            past = hit != 0;
            before = past ? __shfl(upto - v, l) : __shfl(upto, 63);
        }
        const bool last = !past;  // no token passes: the last one
        int pick = -1;
        double won = 0.0;
        past = false;
        for (int i0 = piece * SA_PIECE; i0 < min((piece + 1) * SA_PIECE, A.cols) && !past; i0 += 64) {
            const int i = i0 + lane;
            const float v = i < A.cols ? r.x[i] : -__builtin_inff();
            const double w = i < A.cols && cut.keeps(order_key(v), i) ? r.weight(v) : 0.0;
            const double upto = wave_upto(w, lane) + before;
            const unsigned long long hit = __ballot(!last && w > 0.0 && upto > goal), any = __ballot(w > 0.0);
            if (!any) continue;
            const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
            pick = i0 + l;
            won = __shfl(w, l);
            past = hit != 0;
            before = __shfl(upto, 63);
        }
        if (lane == 0) {
            A.token[at] = pick;
            if (A.logprob) A.logprob[at] = (float)log(won / total);
        }
    }
}

// Host checks that both calls share.
bool sampling_ok(const qg_sampling *p) {
    return p && !(((uintptr_t)p->temperature | (uintptr_t)p->top_k | (uintptr_t)p->top_p | (uintptr_t)p->min_p) & 3);
}
SampleArgs sample_args(const float *x, int rows, int cols, const qg_sampling *p) {
    SampleArgs A{};
    A.x = x;
    A.temperature = p->temperature;
    A.top_k = p->top_k;
    A.top_p = p->top_p;
    A.min_p = p->min_p;
    A.cols = cols;
    int bits = 0;
    while (1 << bits < cols) bits++;
    A.fixed = 62 - bits;
    return A;
}
}  // namespace

extern "C" {

size_t qg_sample_workspace_bytes(int rows, int cols) {
    if (rows < 1 || rows > QG_MAX_ROWS || cols < 1 || cols > SA_MAX_COLS || (long)rows * cols > 1L << 35) return 0;
    return 16;
}

int qg_sample(int *token, float *logprob, const float *x, int rows, int cols, int draws, const qg_sampling *sampling, const float *u,
              void *ws, size_t ws_bytes) {
    const size_t need = qg_sample_workspace_bytes(rows, cols);
    if (!need || !token || !x || !u || !ws || ws_bytes < need || ((uintptr_t)ws & 15) || !sampling_ok(sampling)) return hipErrorInvalidValue;
    if (draws < 1 || draws > SA_MAX_DRAWS || (((uintptr_t)token | (uintptr_t)logprob | (uintptr_t)x | (uintptr_t)u) & 3)) return hipErrorInvalidValue;
    const size_t xb = 4 * (size_t)rows * cols, db = 4 * (size_t)rows * draws, rb = qg_ints(rows);
    const QgSpan out[3] = {{token, db}, {logprob, db}, {ws, need}},
                 in[6] = {{x, xb}, {u, db}, {sampling->temperature, rb}, {sampling->top_k, rb}, {sampling->top_p, rb}, {sampling->min_p, rb}};
    if (qg_any_overlap(out, in) || qg_overlap(token, db, logprob, db) || qg_overlap(ws, need, token, db) || qg_overlap(ws, need, logprob, db))
        return hipErrorInvalidValue;
    SampleArgs A = sample_args(x, rows, cols, sampling);
    A.u = u;
    A.token = token;
    A.logprob = logprob;
    A.draws = draws;
    sample_row_kernel<true><<<rows, SA_THREADS, 0, qg_stream()>>>(A);
    return hipGetLastError();
}

int qg_sampling_softmax(float *out, const float *x, int rows, int cols, const qg_sampling *sampling, void *ws, size_t ws_bytes) {
    const size_t need = qg_sample_workspace_bytes(rows, cols);
    if (!need || !out || !x || !ws || ws_bytes < need || (((uintptr_t)out | (uintptr_t)x) & 3) || ((uintptr_t)ws & 15) || !sampling_ok(sampling))
        return hipErrorInvalidValue;
    const size_t xb = 4 * (size_t)rows * cols, rb = qg_ints(rows);
    const QgSpan written[2] = {{out, xb}, {ws, need}},
                 in[4] = {{sampling->temperature, rb}, {sampling->top_k, rb}, {sampling->top_p, rb}, {sampling->min_p, rb}};
    if (qg_any_overlap(written, in) || (out != x && qg_overlap(out, xb, x, xb)) || qg_overlap(ws, need, x, xb) || qg_overlap(ws, need, out, xb))
        return hipErrorInvalidValue;
    SampleArgs A = sample_args(x, rows, cols, sampling);
    A.out = out;
    sample_row_kernel<false><<<rows, SA_THREADS, 0, qg_stream()>>>(A);
    return hipGetLastError();
}

}  // extern "C"
