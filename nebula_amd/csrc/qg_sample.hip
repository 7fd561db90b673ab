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

// What the pass over a piece of a row leaves: its largest value (NaN if there is one), that
// value's place on the grid, whether weights lie below the bins, and the sum of the weights in no
// bin, in units of 2^(place / 4).
struct PieceStat { float top; int at, below, pad; double rest; };
// What a row came to: its cut, and what its probabilities are formed from.
struct RowResult { uint32_t t; int last; float top; int state; double a, total; };
enum { ROW_NAN = 0, ROW_NONE = 1, ROW_CUT = 2 };

struct SampleArgs {
    const float *x, *temperature, *top_p, *min_p, *u;
    const int *top_k;
    float *out, *logprob;
    int *token;
    int cols, draws, fixed;  // fixed: weights are added up as whole numbers of 2^-fixed where their order is not given
    unsigned long long *bins;  // [rows][pieces][SA_GRID]
    PieceStat *stats;          // [rows][pieces]
    RowResult *results;        // [rows]
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
    __device__ __forceinline__ bool filters() const { return top_k || top_p < 1.0 || min_p > 0.0; }
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
    unsigned long long mass[SA_BINS];
    unsigned count[SA_BINS];
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

// ------------------------------------------------------------------------
// One pass over the values, in pieces.  The weights' exponents x a lie on a grid of quarter
// bits; each piece counts and weighs the values of the SA_GRID bins from its
// largest down, so that all pieces together cover the 16 bits of weight below the row's
// largest, where filters usually cut.  A weight is 1..2^(1/4) times its bin's lower end: what it
// has above that, to 2^-39, is added up as a whole number under the count, in one 64-bit atomic
// whose order does not matter.
// ------------------------------------------------------------------------
constexpr int SA_GRID = 64, PIECE_THREADS = 256, PIECE_VALUES = SA_PIECE / PIECE_THREADS, GRID_COUNT = 49, GRID_BITS = 39;
constexpr double GRID_ZERO = 4400.0;        // quarter bits below which a weight is 0 in 64 bits
constexpr double GRID_FAR = (double)(1 << 21);  // places further out are left to the search over the row
constexpr int GRID_LOW = -0x7fffffff;       // in place of one: all of the piece's weights are 0 beside a row's largest within half of that

// 2^(f / 4), 0 <= f < 1, at least 1: the Taylor series about f = 1/2, whose next term is below 1e-17.
QG_DEV double quarter_power(double f) {
    constexpr double h = 0.173286795139986327354, at_half = 1.09050773266525765921;  // ln 2 / 4, 2^(1/8)
    constexpr double c1 = at_half * h, c2 = c1 * h / 2, c3 = c2 * h / 3, c4 = c3 * h / 4, c5 = c4 * h / 5, c6 = c5 * h / 6, c7 = c6 * h / 7, c8 = c7 * h / 8,
                     c9 = c8 * h / 9;
    const double c[9] = {at_half, c1, c2, c3, c4, c5, c6, c7, c8}, y = f - 0.5;
    double p = c9;
#pragma unroll
    for (int i = 8; i >= 0; i--) p = __builtin_fma(p, y, c[i]);
    return __builtin_fmax(p, 1.0);
}
QG_DEV double grid_scale(int quarters) {  // 2^(quarters / 4)
    const int j = quarters & 3;
    const double c = j == 0 ? 1.0 : j == 1 ? 1.18920711500272106672 : j == 2 ? 1.41421356237309504880 : 1.68179283050742908606;
    return __builtin_amdgcn_ldexp(c, quarters >> 2);
}
QG_DEV double grid_place(float x, double a4) { return __builtin_floor((double)x * a4); }
QG_DEV float larger_or_nan(float a, float b) { return a != a || b != b ? __builtin_nanf("") : fmaxf(a, b); }

__global__ __launch_bounds__(PIECE_THREADS) void sample_piece_kernel(SampleArgs A, int pieces) {
    constexpr int W = PIECE_THREADS / 64;
    __shared__ unsigned long long s_bin[SA_GRID];
    __shared__ float s_top[W];
    __shared__ double s_rest[W];
    __shared__ int s_below[W];
    const int row = blockIdx.x / pieces, piece = blockIdx.x % pieces, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Request q = read_request(A, row);
    const int n = min(SA_PIECE, A.cols - piece * SA_PIECE);
    const float *x = A.x + (size_t)row * A.cols + (size_t)piece * SA_PIECE + tid;
    float v[PIECE_VALUES], top = -__builtin_inff();
    if (n == SA_PIECE) {
#pragma unroll
        for (int k = 0; k < PIECE_VALUES; k++) v[k] = x[k * PIECE_THREADS];
    } else {
#pragma unroll
        for (int k = 0; k < PIECE_VALUES; k++) v[k] = k * PIECE_THREADS + tid < n ? x[k * PIECE_THREADS] : -__builtin_inff();
    }
    if (tid < SA_GRID) s_bin[tid] = 0;
    bool nan = false;
#pragma unroll
    for (int k = 0; k < PIECE_VALUES; k++) { top = fmaxf(top, v[k]); nan |= v[k] != v[k]; }
    top = qg_wave_max(top);
    if (__any(nan)) top = __builtin_nanf("");
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    top = s_top[0];
#pragma unroll
    for (int w = 1; w < W; w++) top = larger_or_nan(top, s_top[w]);
    const double a4 = q.a * 4.0, place = grid_place(top, a4);
    const size_t at = (size_t)row * pieces + piece;
    if (!(__builtin_fabs(place) < GRID_FAR)) {  // NaN and infinities too
        if (tid == 0) A.stats[at] = PieceStat{top, GRID_LOW, 0, 0, 0.0};
        return;
    }
    const bool filter = q.filters(), rest_counts = !q.top_k;
    double rest = 0.0;
    bool below = false;
#pragma unroll
    for (int k = 0; k < PIECE_VALUES; k++) {
        const double e = (double)v[k] * a4, b = __builtin_floor(e), d = place - b;
        if (!(d < GRID_ZERO)) continue;
        if (filter && d < SA_GRID) {
            const unsigned long long m = (unsigned long long)__double_as_longlong(quarter_power(e - b)) & ((1ULL << 52) - 1);
            atomicAdd(&s_bin[(int)d], ((m + (1ULL << (51 - GRID_BITS))) >> (52 - GRID_BITS)) + (1ULL << GRID_COUNT));
        } else {
            below = true;
            if (rest_counts) rest += quarter_power(e - b) * grid_scale(-(int)d);
        }
    }
    rest = wave_all_add(rest);
    below = __any(below);
    if (lane == 0) { s_rest[wave] = rest; s_below[wave] = below; }
    __syncthreads();
    if (filter && tid < SA_GRID) A.bins[at * SA_GRID + tid] = s_bin[tid];
    if (tid == 0) {
        PieceStat p{top, (int)place, 0, 0, 0.0};
#pragma unroll
        for (int w = 0; w < W; w++) { p.rest += s_rest[w]; p.below |= s_below[w]; }
        A.stats[at] = p;
    }
}

// ------------------------------------------------------------------------
// A row's cut, and its draws, by one workgroup.  The bins of all pieces together say in which one
// a filter cuts; where in it say its values, read again from the pieces that have some
// and ranked.  What the bins do not reach is left to the search over the whole row.
// ------------------------------------------------------------------------
constexpr int SA_LIST = 1024;
struct GridShared {
    unsigned count[SA_WAVES][SA_GRID];
    unsigned long long mant[SA_WAVES][SA_GRID];
    uint32_t key[SA_LIST], sorted_key[SA_LIST];
    int index[SA_LIST], sorted_index[SA_LIST];
    double upto[SA_LIST], wave_sum[SA_WAVES];
    int listed;
};
struct SelectShared {
    union { RowShared row; GridShared grid; };
    double piece[SA_MAX_COLS / SA_PIECE];  // what stays of each piece
    float top[SA_WAVES];
    int flag[SA_WAVES];
};

struct Grid {
    const SampleArgs &A;
    GridShared &s;
    const Row &r;
    const unsigned long long *bins;
    const PieceStat *stats;
    const int pieces, tid, lane, wave, place;  // place: of the row's largest value
    const double a4, unit;                     // unit: of a weight of place's lower end, the largest value's being 1
    // lane D of each wave: values in bin D from the top, their weight, and both with the bins above
    unsigned count, count_upto;
    double mass, mass_upto;
    int bin, kept;                             // the listed bin (-1: none), and how many of its values stay

    // A piece's bin of a lane, moved to the row's grid; 0 where it has none.
    __device__ __forceinline__ unsigned long long bin_of(int p, int &delta) const {
        const int at = stats[p].at;
        delta = at == GRID_LOW ? SA_GRID : min(place - at, SA_GRID);
        const unsigned long long own = delta < SA_GRID ? bins[(size_t)p * SA_GRID + lane] : 0;
        return own;
    }
    __device__ __forceinline__ unsigned long long moved(unsigned long long own, int delta) const {
        const unsigned long long b = __shfl(own, (lane - delta) & 63);
        return lane >= delta ? b : 0;
    }
    static __device__ __forceinline__ double mass_of(unsigned n, unsigned long long mant, int bin) {
        return ((double)n + (double)mant * __builtin_amdgcn_ldexp(1.0, -GRID_BITS)) * grid_scale(-bin);
    }
    // All pieces' bins; whether the row has weights below them.
    __device__ bool add_up(int *flag) {
        unsigned n = 0;
        unsigned long long m = 0;
        bool below = false;
        for (int p = wave; p < pieces; p += SA_WAVES) {
            int delta;
            const unsigned long long own = bin_of(p, delta), b = moved(own, delta);
            below |= own && lane + delta >= SA_GRID;
            if (stats[p].at != GRID_LOW && place - stats[p].at < (int)GRID_ZERO) below |= stats[p].below || delta >= SA_GRID;
            n += (unsigned)(b >> GRID_COUNT);
            m += b & ((1ULL << GRID_COUNT) - 1);
        }
        below = __any(below);
        s.count[wave][lane] = n;
        s.mant[wave][lane] = m;
        if (lane == 0) flag[wave] = below;
        __syncthreads();
        count = 0;
        m = 0;
        below = false;
#pragma unroll
        for (int w = 0; w < SA_WAVES; w++) {
            count += s.count[w][lane];
            m += s.mant[w][lane];
            below |= flag[w] != 0;
        }
        mass = mass_of(count, m, lane) * unit;
        count_upto = wave_upto(count, lane);
        mass_upto = wave_upto(mass, lane);
        return below;
    }
    __device__ __forceinline__ double above(int D) const { return D ? __shfl(mass_upto, D - 1) : 0.0; }
    // The values of bin D in falling order with the sums of their weights; false if they are too many.
    __device__ bool list(int D) {
        const unsigned n = __shfl(count, D);
        if (n > SA_LIST) return false;
        __syncthreads();
        if (tid == 0) s.listed = 0;
        __syncthreads();
        const double b = (double)(place - D);
        for (int p = wave; p < pieces; p += SA_WAVES) {
            int delta;
            const unsigned long long own = bin_of(p, delta);
            if (D < delta || !(__shfl(own, (D - delta) & 63) >> GRID_COUNT)) continue;
            each_value<64>(r.x, p * SA_PIECE + lane, min((p + 1) * SA_PIECE, A.cols), [&](int i, float v) {
                if (grid_place(v, a4) != b) return;
                const int k = atomicAdd(&s.listed, 1);
                if (k < SA_LIST) { s.key[k] = order_key(v); s.index[k] = i; }
            });
        }
        __syncthreads();
        double w = 0.0;
        if (tid < (int)n) {
            const uint32_t key = s.key[tid];
            const int i = s.index[tid];
            int rank = 0;
            for (int k = 0; k < (int)n; k++) rank += s.key[k] > key || (s.key[k] == key && s.index[k] < i);
            s.sorted_key[rank] = key;
            s.sorted_index[rank] = i;
        }
        __syncthreads();
        if (tid < (int)n) w = r.weight(key_value(s.sorted_key[tid]));
        w = wave_upto(w, lane);
        if (lane == 63) s.wave_sum[wave] = w;
        __syncthreads();
        for (int k = 0; k < wave; k++) w += s.wave_sum[k];
        s.upto[tid] = w;
        __syncthreads();
        bin = D;
        kept = (int)n;
        return true;
    }
    // The least key of place b, which is the place of some value of a piece or more: a search in 64 ways.
    __device__ uint32_t first_key(double b) const {
        uint32_t lo = 0x007fffffu, hi = order_key(r.m);
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo - 1) / 64 + 1, k = lo + min((uint32_t)(lane + 1) * step, hi - lo);
            const int first = __builtin_ctzll(__ballot(grid_place(key_value(k), a4) >= b));
            const uint32_t up = lo + min((uint32_t)(first + 1) * step, hi - lo);
            lo += min((uint32_t)first * step, hi - lo);
            hi = up;
        }
        return hi;
    }
    // The row's cut and the weight that stays; false where the bins do not reach.
    __device__ bool select(const Request &q, Cut &cut, double &total, int &last_bin, int *flag) {
        const bool below = add_up(flag);
        bin = -1;
        kept = 0;
        last_bin = SA_GRID;  // bins above it stay whole
        if (q.top_k) {
            const unsigned long long enough = __ballot(count_upto >= (unsigned)q.top_k);
            if (!enough && below) return false;
            if (enough) {
                const int D = __builtin_ctzll(enough);
                const int left = q.top_k - (int)(__shfl(count_upto, D) - __shfl(count, D));
                if (left == (int)__shfl(count, D)) {  // all of the bin
                    cut = Cut{first_key((double)(place - D)), 0x7fffffff};
                    last_bin = D + 1;
                    total = __shfl(mass_upto, D);
                } else {
                    if (!list(D)) return false;
                    kept = left;
                    last_bin = D;
                    cut = Cut{s.sorted_key[left - 1], s.sorted_index[left - 1]};
                    total = above(D) + s.upto[left - 1];
                }
            } else {
                total = __shfl(mass_upto, SA_GRID - 1);
            }
        }
        if (q.top_p < 1.0) {
            if (!q.top_k) {
                total = 0.0;  // of all pieces, whatever lies in bins
                for (int p = wave; p < pieces; p += SA_WAVES) {
                    int delta;
                    const unsigned long long own = bin_of(p, delta);
                    const double in = wave_all_add(mass_of((unsigned)(own >> GRID_COUNT), own & ((1ULL << GRID_COUNT) - 1), lane));
                    if (stats[p].at != GRID_LOW) total += (in + stats[p].rest) * grid_scale(stats[p].at - place) * unit;
                }
                __syncthreads();
                if (lane == 0) s.wave_sum[wave] = total;
                __syncthreads();
                total = 0.0;
#pragma unroll
                for (int w = 0; w < SA_WAVES; w++) total += s.wave_sum[w];
            }
            const double goal = q.top_p * total;
            const unsigned long long enough = __ballot(count_upto > 0 && mass_upto >= goal);
            if (!enough && below) return false;
            const int D = enough ? __builtin_ctzll(enough) : SA_GRID - 1;
            if (D < last_bin || D == bin) {
                if (D != bin && !list(D)) return false;
                const double before = above(D);
                // the first of the bin's values that reaches the goal
                __syncthreads();
                if (tid == 0) s.listed = kept - 1;
                __syncthreads();
                if (tid < kept && before + s.upto[tid] >= goal) atomicMin(&s.listed, tid);
                __syncthreads();
                if (kept > 0) {
                    kept = s.listed + 1;
                    last_bin = D;
                    cut = Cut{s.sorted_key[kept - 1], s.sorted_index[kept - 1]};
                    total = before + s.upto[kept - 1];
                }
            }
        }
        if (q.min_p > 0.0) {
            const uint32_t t = r.least_key(q.min_p);
            if (t > cut.t) {
                const double d = (double)place - grid_place(key_value(t), a4);
                if (!(d < SA_GRID)) {
                    if (below) return false;
                } else {
                    const int D = (int)d;
                    if (D != bin && !list(D)) return false;
                    const int n = __syncthreads_count(tid < kept && s.sorted_key[tid] >= t);
                    kept = n;
                    last_bin = D;
                    cut = Cut{t, 0x7fffffff};
                    total = above(D) + (n ? s.upto[n - 1] : 0.0);
                }
            }
        }
        if (!q.top_k && !(q.top_p < 1.0) && last_bin == SA_GRID) total = __shfl(mass_upto, SA_GRID - 1);  // min-p that drops nothing
        return true;
    }
    // What stays of each piece: its bins above the last one, and the listed values that are its.
    __device__ void weigh_pieces(int last_bin, double *piece) const {
        for (int p = wave; p < pieces; p += SA_WAVES) {
            int delta;
            const unsigned long long b = moved(bin_of(p, delta), delta);
            double sum = lane < last_bin ? mass_of((unsigned)(b >> GRID_COUNT), b & ((1ULL << GRID_COUNT) - 1), lane) * unit : 0.0;
            if (last_bin == bin)
                for (int k = lane; k < kept; k += 64)
                    if (s.sorted_index[k] / SA_PIECE == p) sum += r.weight(key_value(s.sorted_key[k]));
            sum = wave_all_add(sum);
            if (lane == 0) piece[p] = sum;
        }
    }
};

template <bool DRAW>
__global__ __launch_bounds__(SA_THREADS) void sample_select_kernel(SampleArgs A, int pieces) {
    __shared__ SelectShared s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Request q = read_request(A, row);
    const PieceStat *stats = A.stats + (size_t)row * pieces;
    float top = -__builtin_inff();
    for (int p = tid; p < pieces; p += SA_THREADS) top = larger_or_nan(top, stats[p].top);
    const bool nan = __any(top != top);
    top = nan ? __builtin_nanf("") : qg_wave_max(top);
    if (lane == 0) s.top[wave] = top;
    __syncthreads();
    top = s.top[0];
#pragma unroll
    for (int w = 1; w < SA_WAVES; w++) top = larger_or_nan(top, s.top[w]);
    if (!__builtin_isfinite(top)) {
        if (DRAW) {
            if (tid < A.draws) {
                A.token[(size_t)row * A.draws + tid] = -1;
                if (A.logprob) A.logprob[(size_t)row * A.draws + tid] = __builtin_nanf("");
            }
        } else if (tid == 0) {
            A.results[row] = RowResult{0, 0, top, top == -__builtin_inff() ? ROW_NONE : ROW_NAN, 0.0, 0.0};
        }
        return;
    }
    Row r{A, s.row, A.x + (size_t)row * A.cols, tid, lane, wave, q.a, top};
    Cut cut;
    double total = 0.0;
    const double a4 = q.a * 4.0, place = grid_place(top, a4);
    bool found = false, weighed = false;
    if (__builtin_fabs(place) < 0.5 * GRID_FAR) {
        const double unit = 1.0 / quarter_power((double)top * a4 - place);
        if (!q.filters()) {
            for (int p = tid; p < pieces; p += SA_THREADS) s.piece[p] = stats[p].at == GRID_LOW ? 0.0 : stats[p].rest * grid_scale(stats[p].at - (int)place) * unit;
            found = weighed = true;
        } else {
            Grid g{A, s.grid, r, A.bins + (size_t)row * pieces * SA_GRID, stats, pieces, tid, lane, wave, (int)place, a4, unit};
            int last_bin;
            found = g.select(q, cut, total, last_bin, s.flag);
            if (found && DRAW) {
                g.weigh_pieces(last_bin, s.piece);
                weighed = true;
            }
        }
    }
    if (!found) {
        __syncthreads();
        cut = Cut{};
        if (q.top_k) r.shorten(cut, false, q.top_k);
        if (q.top_p < 1.0) r.shorten(cut, true, q.top_p);
        if (q.min_p > 0.0) {
            const uint32_t k = r.least_key(q.min_p);
            if (k > cut.t) cut = Cut{k, 0x7fffffff};
        }
        __syncthreads();
        for (int p = wave; p < pieces; p += SA_WAVES) {
            double sum = 0.0;
            each_value<64>(r.x, p * SA_PIECE + lane, min((p + 1) * SA_PIECE, A.cols), [&](int i, float v) { sum += cut.keeps(order_key(v), i) ? r.weight(v) : 0.0; });
            sum = wave_all_add(sum);
            if (lane == 0) s.piece[p] = sum;
        }
        weighed = true;
    }
    if (weighed) {
        __syncthreads();
        total = 0.0;
        for (int p0 = 0; p0 < pieces; p0 += 64) total += wave_all_add(p0 + lane < pieces ? s.piece[p0 + lane] : 0.0);
    }
    if (!DRAW) {
        if (tid == 0) A.results[row] = RowResult{cut.t, cut.last, top, ROW_CUT, q.a, total};
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

// Probabilities of a piece; one that lies below the cut is not read.
__global__ __launch_bounds__(PIECE_THREADS) void sample_probs_kernel(SampleArgs A, int pieces) {
    const int row = blockIdx.x / pieces, piece = blockIdx.x % pieces, tid = threadIdx.x;
    const RowResult q = A.results[row];
    const float top = A.stats[(size_t)row * pieces + piece].top;
    const int c0 = piece * SA_PIECE, n = min(SA_PIECE, A.cols - c0);
    const size_t at = (size_t)row * A.cols + c0 + tid;
    float *to = A.out + at;
    const Cut cut{q.t, q.last};
    if (q.state != ROW_CUT || order_key(top) < q.t) {
        const float y = q.state == ROW_NAN ? __builtin_nanf("") : 0.0f;
        if (n == SA_PIECE) {
#pragma unroll
            for (int k = 0; k < PIECE_VALUES; k++) to[k * PIECE_THREADS] = y;
        } else {
            for (int k = tid; k < n; k += PIECE_THREADS) to[k - tid] = y;
        }
        return;
    }
    const float *x = A.x + at;
    float v[PIECE_VALUES];
#pragma unroll
    for (int k = 0; k < PIECE_VALUES; k++) v[k] = n == SA_PIECE || k * PIECE_THREADS + tid < n ? x[k * PIECE_THREADS] : -__builtin_inff();
    const double share = 1.0 / q.total;
#pragma unroll
    for (int k = 0; k < PIECE_VALUES; k++) {
        float y = 0.0f;
        if (cut.keeps(order_key(v[k]), c0 + k * PIECE_THREADS + tid)) y = (float)(exp2_d(((double)v[k] - (double)q.top) * q.a) * share);
        if (n == SA_PIECE || k * PIECE_THREADS + tid < n) to[k * PIECE_THREADS] = y;
    }
}

// Host checks that both calls share.
bool sampling_ok(const qg_sampling *p) {
    return p && !(((uintptr_t)p->temperature | (uintptr_t)p->top_k | (uintptr_t)p->top_p | (uintptr_t)p->min_p) & 3);
}
int sample_pieces(int cols) { return (cols + SA_PIECE - 1) / SA_PIECE; }
SampleArgs sample_args(const float *x, int rows, int cols, const qg_sampling *p, void *ws) {
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
    const size_t all = (size_t)rows * sample_pieces(cols);
    A.results = (RowResult *)ws;
    A.stats = (PieceStat *)(A.results + rows);
    A.bins = (unsigned long long *)(A.stats + all);
    return A;
}
}  // namespace

extern "C" {

size_t qg_sample_workspace_bytes(int rows, int cols) {
    if (rows < 1 || rows > QG_MAX_ROWS || cols < 1 || cols > SA_MAX_COLS || (long)rows * cols > 1L << 35) return 0;
    return (size_t)rows * (sizeof(RowResult) + sample_pieces(cols) * (sizeof(PieceStat) + SA_GRID * sizeof(unsigned long long)));
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
    SampleArgs A = sample_args(x, rows, cols, sampling, ws);
    A.u = u;
    A.token = token;
    A.logprob = logprob;
    A.draws = draws;
    const int pieces = sample_pieces(cols);
    sample_piece_kernel<<<(unsigned)((size_t)rows * pieces), PIECE_THREADS, 0, qg_stream()>>>(A, pieces);
    sample_select_kernel<true><<<rows, SA_THREADS, 0, qg_stream()>>>(A, pieces);
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
    SampleArgs A = sample_args(x, rows, cols, sampling, ws);
    A.out = out;
    const int pieces = sample_pieces(cols);
    sample_piece_kernel<<<(unsigned)((size_t)rows * pieces), PIECE_THREADS, 0, qg_stream()>>>(A, pieces);
    sample_select_kernel<false><<<rows, SA_THREADS, 0, qg_stream()>>>(A, pieces);
    sample_probs_kernel<<<(unsigned)((size_t)rows * pieces), PIECE_THREADS, 0, qg_stream()>>>(A, pieces);
    return hipGetLastError();
}

}  // extern "C"
