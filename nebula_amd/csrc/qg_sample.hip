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
#include "qg_lanes.h"

namespace {

constexpr int SA_DIGIT = 11, SA_BINS = 1 << SA_DIGIT, SA_PIECE = 4096;
constexpr int SA_MAX_COLS = 1 << 24, SA_MAX_DRAWS = 64;
constexpr int SA_GRID = 64, SA_LISTED = 192, SA_LISTS = 128;  // listed values of a piece: at most, and where that suffices

// What the pass over a piece of a row leaves: its largest value (NaN if there is one) and that
// value's bin, whether weights lie below the bins it keeps, the last of these, the last whose values
// are listed, how many are in bins and in the list, and the sums of the weights in no bin and of
// all, in units of 2^at.
struct PieceStat { float top; int at, below, known, cover, counted, listed, pad; double rest, all; };
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
    uint2 *listed;             // [rows][pieces][SA_LISTED] key and index
    double *kept;              // [rows][pieces] the weight that stays of a piece
    PieceStat *stats;          // [rows][pieces]
    RowResult *results;        // [rows]
};

// Unsigned keys in the values' order; the zeros of both signs are one value.
QG_DEV uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
QG_DEV float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// A weight's exponent e = n + y, n whole and |y| <= 1/2, and p = 2^y (HALF: 2^(y + 1/2), in [1, 2]) by the Taylor series,
// whose next term is below 2e-16 of it.  The whole part falls out of the sum with 1.5 2^52, in the low bits; |e| < 2^31.
struct Power { double p; int n; };
template <bool HALF>
QG_DEV Power power_of(double e) {
    constexpr double h = 0.693147180559945309417, c0 = HALF ? 1.41421356237309504880 : 1.0, whole = 6755399441055744.0;
    constexpr double c1 = c0 * h, c2 = c1 * h / 2, c3 = c2 * h / 3, c4 = c3 * h / 4, c5 = c4 * h / 5, c6 = c5 * h / 6, c7 = c6 * h / 7, c8 = c7 * h / 8,
                     c9 = c8 * h / 9, c10 = c9 * h / 10, c11 = c10 * h / 11, c12 = c11 * h / 12;
    const double c[12] = {c0, c1, c2, c3, c4, c5, c6, c7, c8, c9, c10, c11}, t = e + whole, y = e - (t - whole);
    double p = c12;
#pragma unroll
    for (int i = 11; i >= 0; i--) p = __builtin_fma(p, y, c[i]);
    return Power{p, (int)(uint32_t)__double_as_longlong(t)};
}
// p 2^n for results that are normal numbers
QG_DEV double scaled(double p, int n) { return __longlong_as_double(__double_as_longlong(p) + ((long long)n << 52)); }
constexpr int SA_ZERO = 1000;  // weights below 2^-1000 of the largest count as 0
// 2^d, d <= 0
QG_DEV double exp2_d(double d) {
    if (!(d > -SA_ZERO)) return 0.0;
    const Power x = power_of<false>(d);
    return scaled(x.p, x.n);
}

// What a row asks for.  Temperature 0 (or none that counts) is the first largest
// token: top-k 1.
struct Request {
    double a, top_p, min_p;
    int top_k;
    __device__ __forceinline__ bool filters() const { return top_k || top_p < 1.0 || min_p > 0.0; }
    // whether the sum of all weights matters
    __device__ __forceinline__ bool weighs_all() const { return !top_k && (top_p < 1.0 || !(min_p > 0.0)); }
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

// The least key up to hi for which f holds, which grows with the keys, holds at hi and not at
// -infinity: a search in 64 ways, by every wave.
template <typename F>
QG_DEV uint32_t first_key(uint32_t hi, int lane, F f) {
    for (uint32_t lo = 0x007fffffu; hi - lo > 1;) {
        const uint32_t step = (hi - lo - 1) / 64 + 1;
        // the last lane's is hi
        const int first = __builtin_ctzll(__ballot(f(key_value(lo + min((uint32_t)(lane + 1) * step, hi - lo)))) | 1ULL << 63);
        const uint32_t up = lo + min((uint32_t)(first + 1) * step, hi - lo);
        lo += min((uint32_t)first * step, hi - lo);
        hi = up;
    }
    return hi;
}

template <int WAVES>
struct RowShared {
    unsigned long long mass[SA_BINS];
    unsigned count[SA_BINS];
    unsigned long long wave_mass[WAVES], found_mass, found_own;
    unsigned wave_count[WAVES], found_count, found_ties;
    int found_bin;
};

// A row of any shape by one workgroup, which reads it again for every step, at what a CU reads and adds to shared memory.  The
// whole call: 1 row x 151936 175 us (|x / T| past 2^17, top-p or top-k) and 320 to 390 (flat, all in one 64th of a bit), 68 x 50000
// 78 to 166, 1088 x 131072 770 to 1860; rows that the bins serve 20 to 35, 20 to 40 and 330 at most.
template <int WAVES>
struct Row {
    static constexpr int THREADS = 64 * WAVES, OWN = SA_BINS / THREADS;  // bins of a thread
    const SampleArgs &A;
    RowShared<WAVES> &s;
    const float *x;
    const int tid, lane, wave;
    double a;
    float m;

    __device__ __forceinline__ double weight(float v) const { return exp2_d(((double)v - (double)m) * a); }
    __device__ __forceinline__ unsigned long long fixed(float v) const { return (unsigned long long)__builtin_rint(__builtin_amdgcn_ldexp(weight(v), A.fixed)); }

    // From the cut's tokens in falling order the first ones that reach `goal` tokens
    // (by_mass false), or the share goal of their weight: never none.
    __device__ __forceinline__ void shorten(Cut &cut, bool by_mass, double goal) {
        uint32_t prefix = 0;
        unsigned long long above = 0;
        unsigned over = 0;
        double need = goal;
        for (int left = 32; left > 0;) {
            const int bits = left < SA_DIGIT ? left : SA_DIGIT;
            const int shift = left - bits;
            for (int b = tid; b < SA_BINS; b += THREADS) { s.mass[b] = 0; s.count[b] = 0; }
            __syncthreads();
            each_value<THREADS>(x, tid, A.cols, [&](int i, float v) {
                const uint32_t key = order_key(v);
                if ((left < 32 && (key >> left) != prefix) || !cut.keeps(key, i)) return;
                const int bin = (key >> shift) & ((1 << bits) - 1);
                atomicAdd(&s.count[bin], 1u);
                if (by_mass) atomicAdd(&s.mass[bin], fixed(v));
            });
            __syncthreads();
            // sums from the largest bin down, OWN neighbours a thread
            const int b0 = SA_BINS - 1 - OWN * tid;
            unsigned c = 0;
            unsigned long long w = 0;
#pragma unroll
            for (int k = 0; k < OWN; k++) { c += s.count[b0 - k]; w += s.mass[b0 - k]; }
            const unsigned own_c = c;
            const unsigned long long own_w = w;
            c = wave_upto(c);
            w = wave_upto(w);
            if (lane == 63) { s.wave_count[wave] = c; s.wave_mass[wave] = w; }
            if (tid == 0) s.found_bin = -1;
            __syncthreads();
            unsigned long long all = 0;
            for (int k = 0; k < WAVES; k++) {
                if (k < wave) { c += s.wave_count[k]; w += s.wave_mass[k]; }
                all += s.wave_mass[k];
            }
            if (left == 32 && by_mass) need = goal * (double)all;
            c += over - own_c;
            w += above - own_w;
            // the first bin with which there is enough
            auto enough = [&](unsigned cc, unsigned long long ww) { return cc > 0 && (by_mass ? (double)ww >= need : cc >= (unsigned)need); };
#pragma unroll
            for (int k = 0; k < OWN; k++) {
                const unsigned n = s.count[b0 - k];
                const unsigned long long m = s.mass[b0 - k];
                if (n && enough(c + n, w + m) && !enough(c, w)) { s.found_bin = b0 - k; s.found_count = c; s.found_mass = w; s.found_ties = n; s.found_own = m; }
                c += n;
                w += m;
            }
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
    __device__ __forceinline__ int nth(uint32_t t, const Cut &cut, unsigned r) {
        const int per = ((A.cols + WAVES - 1) / WAVES + 63) / 64 * 64, i0 = wave * per, end = min(i0 + per, A.cols);
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
    // The least key whose weight is at least `least` (0 < least <= 1).
    __device__ __forceinline__ uint32_t least_key(double least) const {
        return first_key(order_key(m), lane, [&](float v) { return weight(v) >= least; });
    }
};

// ------------------------------------------------------------------------
// One pass over the values, in pieces.  A bin holds the weights whose exponents x a round to one whole
// number, the same for all pieces of a row, so that those of all pieces can be added; a piece keeps the
// SA_GRID bins from its largest value down, of these only as many as the row's filters
// may cut in.  A weight is 1..2 times its bin's lower end: what it has above that, to 2^-38, is
// added up as a whole number under the count, in one 64-bit atomic whose order does not
// matter.  The values of the first bins, up to SA_LISTED of them, are listed: few tokens
// stay of most rows, and then nothing is read again.
// 1088 rows x 131072 (570 MB): requests whose first filter is a small top-k 150 us (3.8 TB/s), one
// weight per value in 64 bits 200, nearly all values in bins (top-p alone, top-k 1000) 330, the ten kinds mixed
// 215 to 240.  Of 4096 values in a workgroup's registers: 16 loads of a thread on their way, eight
// workgroups on a CU; with the next piece on its way in as many registers again 474 us, 16-byte loads 264.
// ------------------------------------------------------------------------
constexpr int PIECE_THREADS = 256, PIECE_WAVES = PIECE_THREADS / 64, PIECE_VALUES = SA_PIECE / PIECE_THREADS, BIN_COUNT = 51, BIN_BITS = 38;
// Places further out are left to the search over the row.  A row's largest place is below half of it: exponents of up to 2^18 are
// off by 2^-36, weights and the largest's with them and by the bins' 2^-39 each: sums to 2^-35 of themselves (exponents up to
// 2^15: to 2^-37), which the weights of (x - max) a that follow within a piece are held against.
constexpr double GRID_FAR = (double)(1 << 19);
constexpr int GRID_LOW = -(1 << 30);            // in place of one: the piece's weights are 0 beside a row's largest within half of that

QG_DEV double grid_place(float x, double a) { return __builtin_rint((double)x * a); }
// What a weight of p times its bin's lower end adds to the bin; a bin's weights in units of the lower end of bin 0.
QG_DEV unsigned long long bin_entry(double p) {
    // p may have been rounded below 1 or up to 2
    const unsigned long long m = (unsigned long long)__double_as_longlong(__builtin_fmin(__builtin_fmax(p, 1.0), 0x1.fffffffffffffp0)) & ((1ULL << 52) - 1);
    return ((m + (1ULL << (51 - BIN_BITS))) >> (52 - BIN_BITS)) + (1ULL << BIN_COUNT);
}
QG_DEV unsigned bin_count(unsigned long long b) { return (unsigned)(b >> BIN_COUNT); }
QG_DEV unsigned long long bin_excess(unsigned long long b) { return b & ((1ULL << BIN_COUNT) - 1); }
QG_DEV double bin_mass(unsigned n, unsigned long long excess, int bin) {
    return __builtin_amdgcn_ldexp((double)n + __builtin_amdgcn_ldexp((double)excess, -BIN_BITS), -bin);
}
QG_DEV float larger_or_nan(float a, float b) { return a != a || b != b ? __builtin_nanf("") : fmaxf(a, b); }
// The last bin that a row's filters may cut in, from what they ask for: less than 2^bits values of a weight
// below 2^-d of the largest are less than 2^(bits - d) of the sum.
QG_DEV int deepest_bin(const Request &q, int bits) {
    if (q.top_k) return SA_GRID - 1;
    const double least = q.top_p < 1.0 ? (1.0 - q.top_p) * __builtin_amdgcn_ldexp(1.0, -bits) : q.min_p;
    return min(2 - __builtin_amdgcn_frexp_exp(least), SA_GRID - 1);
}

__global__ __launch_bounds__(PIECE_THREADS) void sample_piece_kernel(SampleArgs A, int pieces) {
    __shared__ unsigned long long s_bin[SA_GRID];
    __shared__ unsigned s_most[SA_GRID];
    __shared__ float s_top[PIECE_WAVES], s_value[SA_PIECE];
    __shared__ double s_rest[PIECE_WAVES];
    __shared__ int s_below[PIECE_WAVES], s_cover, s_listed[SA_GRID];
    const int row = blockIdx.x / pieces, piece = blockIdx.x % pieces, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int c0 = piece * SA_PIECE, n = min(SA_PIECE, A.cols - c0);
    const float *x = A.x + (size_t)row * A.cols + c0 + tid;
    float v[PIECE_VALUES], own = -__builtin_inff();
    if (n == SA_PIECE) {
#pragma unroll
        for (int k = 0; k < PIECE_VALUES; k++) v[k] = x[k * PIECE_THREADS];
    } else {
#pragma unroll
        for (int k = 0; k < PIECE_VALUES; k++) v[k] = k * PIECE_THREADS + tid < n ? x[k * PIECE_THREADS] : -__builtin_inff();
    }
    const Request q = read_request(A, row);
    if (tid < SA_GRID) { s_bin[tid] = 0; s_most[tid] = 0; }
    bool nan = false;
#pragma unroll
    for (int k = 0; k < PIECE_VALUES; k++) { own = fmaxf(own, v[k]); nan |= v[k] != v[k]; }
    float top = qg_wave_max(own);
    if (__any(nan)) top = __builtin_nanf("");
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    top = s_top[0];
#pragma unroll
    for (int w = 1; w < PIECE_WAVES; w++) top = larger_or_nan(top, s_top[w]);
    const double far = grid_place(top, q.a);
    const size_t at = (size_t)row * pieces + piece;
    if (!(__builtin_fabs(far) < GRID_FAR)) {  // NaN and infinities too
        if (tid == 0) A.stats[at] = PieceStat{top, GRID_LOW, 0, SA_GRID - 1, SA_GRID - 1, 0, 0, 0, 0.0, 0.0};
        return;
    }
    const int place = (int)far;
    const bool filter = q.filters(), weigh = q.weighs_all();
    int known = filter ? deepest_bin(q, 62 - A.fixed) : -1;
    if (q.top_k && q.top_k <= PIECE_THREADS - 16) {
        // the row's top_k values are not below the piece's, and these not below the top_k-th of its threads' largest
        const double d = far - grid_place(own, q.a);
        if (d < SA_GRID) atomicAdd(&s_most[(int)d], 1u);
        __syncthreads();
        const unsigned long long enough = __ballot(wave_upto(s_most[lane]) >= (unsigned)q.top_k);
        if (enough) known = __builtin_ctzll(enough);
    }
    const float zero = (float)(((double)place - SA_ZERO) / q.a);
    double rest = 0.0;
    bool below = false;
    auto weigh_one = [&](float y) {  // not below zero
        const Power w = power_of<true>((double)y * q.a);
        const int d = place - w.n;
        if (d <= known) {
            atomicAdd(&s_bin[d], bin_entry(w.p));
        } else {
            below = true;
            rest += scaled(w.p, -d);
        }
    };
    if (weigh) {
#pragma unroll
        for (int k = 0; k < PIECE_VALUES; k++)
            if (v[k] > zero) weigh_one(v[k]);
    } else {
        // the wave's values that may be in a bin go together, so that few of its steps form a weight
        float *mine = s_value + wave * (64 * PIECE_VALUES);
        const float near = fmaxf((float)((double)(place - known - 1) / q.a), zero);
        int held = 0;
#pragma unroll
        for (int k = 0; k < PIECE_VALUES; k++) {
            const bool is = v[k] > near;
            const unsigned long long all = __ballot(is);
            if (is) mine[held + __popcll(all & ((1ULL << lane) - 1))] = v[k];
            held += __popcll(all);
            below |= !is && v[k] > zero;
        }
        __builtin_amdgcn_wave_barrier();  // a wave's own values
        for (int i = lane; i < held; i += 64) weigh_one(mine[i]);
    }
    if (weigh) rest = wave_all_add(rest);
    below = __any(below);
    if (lane == 0) { s_rest[wave] = rest; s_below[wave] = below; }
    __syncthreads();
    if (wave == 0) {
        // a piece may hold all top_k, of a bin's about half; the full length only where the row's top_k may fill most of the usual one
        // (us, usual / full length: 68 rows x 24576 with top-k 500 40 / 34, x 50000 with 500 38 / 39, 1000 52 / 40, x 131072 with 1000
        // 51 / 52, 1500 80 / 83, 2500 117 / 101; next to the limit, 68 x 80000 with 1000, 43 / 44; 1088 x 131072 with 1000 352 / 362.
        // Room for it costs the rows that do not use it 4 %)
        const int most = q.top_k > 48 * pieces ? SA_LISTED : q.top_k ? min(max(2 * q.top_k, 32), SA_LISTS) : SA_LISTS;
        const unsigned long long b = s_bin[lane];
        const unsigned upto = wave_upto(bin_count(b));
        const int cover = min((int)__popcll(__ballot(upto <= (unsigned)most)) - 1, known), listed = cover < 0 ? 0 : (int)of_lane(upto, cover);
        const int counted = (int)of_lane(upto, SA_GRID - 1);
        const double in = weigh && filter ? wave_all_add(bin_mass(bin_count(b), bin_excess(b), lane)) : 0.0;
        if (filter) A.bins[at * SA_GRID + lane] = b;
        if (lane == 0) {
            s_cover = cover;
            PieceStat p{top, place, 0, known, cover, counted, listed, 0, 0.0, 0.0};
#pragma unroll
            for (int w = 0; w < PIECE_WAVES; w++) { p.rest += s_rest[w]; p.below |= s_below[w]; }
            p.all = in + p.rest;
            A.stats[at] = p;
        }
    }
    if (!filter) return;
    __syncthreads();
    // the values down to bin `cover`, in order
    const int cover = s_cover;
    if (cover < 0) return;
    const float near = (float)((double)(place - cover - 1) / q.a);
    unsigned mine = 0;
    int counts = 0;  // lane k: the wave's of value k
#pragma unroll
    for (int k = 0; k < PIECE_VALUES; k++) {
        bool is = v[k] > near;
        if (!__any(is)) continue;
        is = is && far - grid_place(v[k], q.a) <= (double)cover;
        const int n = __popcll(__ballot(is));
        if (lane == k) counts = n;
        mine |= (unsigned)is << k;
    }
    if (lane < PIECE_VALUES) s_listed[lane * PIECE_WAVES + wave] = counts;
    __syncthreads();
    const int before = wave_upto(s_listed[lane]) - s_listed[lane];  // of value lane / 4 and wave lane % 4
    uint2 *listed = A.listed + at * SA_LISTED;
#pragma unroll
    for (int k = 0; k < PIECE_VALUES; k++) {
        const unsigned long long all = __ballot(mine >> k & 1);
        if (!all) continue;
        const int to = __builtin_amdgcn_readlane(before, k * PIECE_WAVES + wave) + __popcll(all & ((1ULL << lane) - 1));
        if ((mine >> k & 1) && to < SA_LISTED) listed[to] = make_uint2(order_key(v[k]), c0 + k * PIECE_THREADS + tid);
    }
}

// ------------------------------------------------------------------------
// A row's cut, and its draws, by one workgroup.  The bins of all pieces say in which one a filter cuts; its
// values, from the lists where these reach and else read again from the pieces that have some, are
// ranked (of a bin with too many, those of the 64th part in which the cut is).  What the bins do not
// hold is left to the search over the whole row.  Bound by dependent steps (statistics, bins, the cut's bin, its values in
// order, sums, draws): a row 14 us, 1088 rows of the ten kinds 58, two of them on a CU (114 registers a lane; three with
// 80 spill and gain nothing).  Past 64 pieces nothing is held, and lists are read once more: 4 rows x 262145 with top-k 20 33 us,
// x 262144 22.
// ------------------------------------------------------------------------
constexpr int SA_LIST = 1024, SA_HELD = 2 * SA_LIST;  // values that are ranked; that are held
template <int WAVES>
struct GridShared {
    unsigned count[WAVES][SA_GRID];
    unsigned long long excess[WAVES][SA_GRID];
    union {
        struct {
            unsigned long long put[SA_LIST];  // key, then the complement of the index: of equal keys the lower index is the larger
            uint32_t sorted_key[SA_LIST];
            int sorted_index[SA_LIST];
        };
        double in_order[SA_HELD];             // sums of the held values' weights
    };
    double upto[SA_LIST], wave_sum[WAVES];
    uint2 held[SA_HELD];                      // key and index, in the tokens' order
    int n, hits, of_piece[64];
};
template <int WAVES>
struct SelectShared {
    union { RowShared<WAVES> row; GridShared<WAVES> grid; };
    float top[WAVES];
    int flag[WAVES], reach[WAVES], known[WAVES];
};

template <int WAVES>
struct Grid {
    static constexpr int THREADS = 64 * WAVES;
    GridShared<WAVES> &s;
    const float *x;
    const unsigned long long *bins;
    const PieceStat *stats;
    const PieceStat &mine;                           // of up to 64 pieces the lane's
    const uint2 *lists;
    const int cols, pieces, tid, lane, wave, place;  // place: of the row's largest value
    const float m;
    const double a, unit;                            // unit: what the largest value, whose weight is 1, adds to its bin
    int reach, known;                                // bins 0..reach are in the lists, 0..known in the bins
    bool below;                                      // whether the row has weights below the known bins
    // lane D of each wave: values in bin D from the top and with the bins above, and their weight
    unsigned count, count_upto;
    double mass, mass_upto;
    int deepest;                                     // the bin of the cut
    int bin, kept;                                   // the ranked bin (-1: none, or a part of one), and how many of the ranked values stay
    bool part;                                       // the cut is in a part of its bin
    int held;                                        // values in s.held: all of the bins that any cut can leave; 0: not held

    __device__ __forceinline__ double weight(uint32_t key) const { return exp2_d(((double)key_value(key) - (double)m) * a); }
    __device__ __forceinline__ double place_of(uint32_t key) const { return grid_place(key_value(key), a); }
    // the 64th of its bin that a value is in, from the top
    static __device__ __forceinline__ int part_of(double e) { return 63 - min(max((int)((e - __builtin_rint(e) + 0.5) * 64.0), 0), 63); }
    // A piece's bin of a lane, moved to the row's.
    __device__ __forceinline__ int moved_by(int p) const {
        const int at = pieces <= 64 ? of_lane(mine.at, p) : stats[p].at;  // p is the wave's
        return at == GRID_LOW ? SA_GRID : min(place - at, SA_GRID);
    }
    __device__ __forceinline__ unsigned long long row_bin(int p) const {
        const int delta = moved_by(p);
        return lane >= delta ? bins[(size_t)p * SA_GRID + lane - delta] : 0;
    }
    __device__ __forceinline__ void all_waves(unsigned n, unsigned long long excess, unsigned &c, unsigned long long &e) {
        __syncthreads();
        s.count[wave][lane] = n;
        s.excess[wave][lane] = excess;
        __syncthreads();
        c = 0;
        e = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) { c += s.count[w][lane]; e += s.excess[w][lane]; }
    }
    __device__ __forceinline__ void add_up() {
        unsigned n = 0;
        unsigned long long e = 0;
        for (int p0 = wave; p0 < pieces; p0 += 4 * WAVES) {
            unsigned long long b[4];
#pragma unroll
            for (int k = 0; k < 4; k++) b[k] = p0 + k * WAVES < pieces ? row_bin(p0 + k * WAVES) : 0;
#pragma unroll
            for (int k = 0; k < 4; k++) { n += bin_count(b[k]); e += bin_excess(b[k]); }
        }
        all_waves(n, e, count, e);
        mass = bin_mass(count, e, lane) / unit;
        count_upto = wave_upto(count);
        mass_upto = wave_upto(mass);
        deepest = SA_GRID - 1;
        bin = -1;
        kept = 0;
        part = false;
        held = 0;
    }
    // Holds the listed values of bins 0..D, where lists reach that far and they are not too many.
    static constexpr int EACH = 64 / WAVES, PER = SA_LISTED / 64;  // pieces of a wave, listed values of a lane
    static __device__ __forceinline__ void read_lists(const uint2 *lists, int pieces, const PieceStat &mine, int wave, int lane, uint2 (&y)[EACH][PER]) {
        const bool longer = __any(mine.listed > SA_LISTS);
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            const int p = k * WAVES + wave, listed = p < pieces ? of_lane(mine.listed, p) : 0;
#pragma unroll
            for (int i = 0; i < PER; i++) y[k][i] = (i * 64 < SA_LISTS || longer) && i * 64 + lane < listed ? lists[(size_t)p * SA_LISTED + i * 64 + lane] : make_uint2(0, 0);
        }
    }
    __device__ __forceinline__ void hold(int D, const uint2 (&y)[EACH][PER]) {
        const int n = D < 0 || D > reach || pieces > 64 ? 0 : (int)of_lane(count_upto, D);
        if (n == 0 || n > SA_HELD) return;
        unsigned is = 0;
        const bool longer = __any(mine.listed > SA_LISTS);
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            int all = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (i * 64 >= SA_LISTS && !longer) continue;
                const bool in = y[k][i].x && (double)place - place_of(y[k][i].x) <= (double)D;
                is |= (unsigned)in << (k * PER + i);
                all += (int)__popcll(__ballot(in));
            }
            if (lane == 0) s.of_piece[k * WAVES + wave] = all;
        }
        __syncthreads();
        const int own = s.of_piece[lane], before = wave_upto(own) - own;
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            int to = of_lane(before, k * WAVES + wave);
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (i * 64 >= SA_LISTS && !longer) continue;
                const bool in = is >> (k * PER + i) & 1;
                const unsigned long long all = __ballot(in);
                const int at = to + (int)__popcll(all & ((1ULL << lane) - 1));
                if (in && at < SA_HELD) s.held[at] = y[k][i];
                to += (int)__popcll(all);
            }
        }
        held = min(of_lane(before + own, 63), SA_HELD);
        __syncthreads();
    }
    // The bin in which the row's first filter cuts, -1 for none.
    __device__ __forceinline__ int first_cut(const Request &q, double all, uint32_t least) const {
        if (q.top_k || q.top_p < 1.0) {
            const unsigned long long enough =
                __ballot(lane <= known && count > 0 && (q.top_k ? count_upto >= (unsigned)q.top_k : mass_upto >= q.top_p * all));
            return enough ? (int)__builtin_ctzll(enough) : -1;
        }
        const double d = (double)place - place_of(least);
        return d <= (double)known ? (int)d : -1;
    }
    __device__ __forceinline__ void put(uint32_t key, int i) {
        const int k = atomicAdd(&s.n, 1);
        if (k < SA_LIST) s.put[k] = (unsigned long long)key << 32 | ~(uint32_t)i;
    }
    // f(key, index) of the values in bin D (every lane of some waves each), and of more
    template <typename F>
    __device__ __forceinline__ void each_of_bin(int D, F f) {
        if (held) {
            for (int i = tid; i < held; i += THREADS) f(s.held[i].x, (int)s.held[i].y);
            return;
        }
        if (D <= reach) {
            for (int e0 = wave; e0 < pieces * (SA_LISTED / 64); e0 += 4 * WAVES) {
                uint2 y[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int e = e0 + k * WAVES, p = e / (SA_LISTED / 64), i = e % (SA_LISTED / 64) * 64 + lane;
                    y[k] = e < pieces * (SA_LISTED / 64) && stats[p].at != GRID_LOW && i < min(stats[p].listed, SA_LISTED) ? lists[(size_t)p * SA_LISTED + i] : make_uint2(0, 0);
                }
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (y[k].x) f(y[k].x, (int)y[k].y);
            }
            return;
        }
        // the pieces that have some, then their quarters
        int *hits = s.sorted_index;
        __syncthreads();
        if (tid == 0) s.hits = 0;
        __syncthreads();
        for (int p = tid; p < pieces; p += THREADS) {
            const int at = stats[p].at, delta = at == GRID_LOW ? SA_GRID : min(place - at, SA_GRID);
            if (D >= delta && bins[(size_t)p * SA_GRID + D - delta]) {
                const int k = atomicAdd(&s.hits, 1);
                if (k < SA_LIST) hits[k] = p;
            }
        }
        __syncthreads();
        const bool fit = s.hits <= SA_LIST;
        const int items = (fit ? s.hits : pieces) * 4;
        const float low = (float)((double)(place - D - 1) / a), high = (float)((double)(place - D + 1) / a);
        for (int it = wave; it < items; it += WAVES) {
            const int i0 = (fit ? hits[it >> 2] : it >> 2) * SA_PIECE + (it & 3) * (SA_PIECE / 4) + lane;
            float v[16];
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] = i0 + k * 64 < cols ? x[i0 + k * 64] : -__builtin_inff();
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (v[k] > low && v[k] < high) f(order_key(v[k]), i0 + k * 64);
        }
    }
    // Ranks what was put by falling value, with the sums of the weights.
    __device__ __forceinline__ void rank(int n) {
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) {
            const unsigned long long own = s.put[i];
            int rank = 0;
#pragma unroll 8
            for (int k = 0; k < n; k++) rank += s.put[k] > own;
            s.sorted_key[rank] = (uint32_t)(own >> 32);
            s.sorted_index[rank] = (int)~(uint32_t)own;
        }
        __syncthreads();
        sum_up(s.upto, n, [&](int i) { return weight(s.sorted_key[i]); });
    }
    // to[i] = w(0) + .. + w(i), i < n
    template <typename F>
    __device__ __forceinline__ void sum_up(double *to, int n, F f) {
        double before = 0.0;
        for (int i0 = 0; i0 < n; i0 += THREADS) {
            const int i = i0 + tid;
            double w = wave_upto(i < n ? f(i) : 0.0);
            __syncthreads();
            if (lane == 63) s.wave_sum[wave] = w;
            __syncthreads();
            double all = 0.0;
#pragma unroll
            for (int k = 0; k < WAVES; k++) {
                if (k < wave) w += s.wave_sum[k];
                all += s.wave_sum[k];
            }
            if (i < n) to[i] = before + w;
            before += all;
        }
        __syncthreads();
    }
    // Shortens the cut: to the first `target` tokens, to the first that weigh `target`, or to keys from t on; total: what
    // stays weighs.  False where the known bins do not reach.
    enum { BY_COUNT, BY_MASS, BY_KEY };
    template <int BY>
    __device__ __forceinline__ bool shorten(double target, uint32_t t, Cut &cut, double &total) {
        int D;
        if (BY == BY_KEY) {
            const double d = (double)place - place_of(t);
            if (!(d <= (double)known)) return !below;  // nothing that weighs lies below
            D = (int)d;
        } else {
            // a bin that holds something: the sums up to an empty one may be larger than those before it by their last bits
            const unsigned long long enough = __ballot(lane <= known && count > 0 && (BY == BY_MASS ? mass_upto >= target : (double)count_upto >= target));
            if (!enough) return BY == BY_COUNT && !below;
            D = __builtin_ctzll(enough);
        }
        const int n = (int)of_lane(count, D);
        int first = (int)of_lane(count_upto, D) - n;
        double before = D ? of_lane(mass_upto, D - 1) : 0.0;
        if (BY == BY_COUNT && first + n == (int)target) {  // all of the bin
            cut = Cut{first_key(order_key(m), lane, [&](float v) { return grid_place(v, a) >= (double)(place - D); }), 0x7fffffff};
            deepest = D;
            total = of_lane(mass_upto, D);
            return true;
        }
        if (D != bin) {
            const double b = (double)(place - D);
            int sub = -1;
            // ranking compares all with all: many held values go by parts too (1088 rows x 131072 251 us, all ranked 267; sorted in
            // 55 steps 270); where they are not held, a part would cost another reading of the pieces (45 us for a row, ranked 38)
            if (n > (held ? SA_LIST / 8 : SA_LIST)) {
                __syncthreads();
                if (wave == 0) { s.count[0][lane] = 0; s.excess[0][lane] = 0; }
                __syncthreads();
                each_of_bin(D, [&](uint32_t key, int i) {
                    const double e = (double)key_value(key) * a;
                    if (__builtin_rint(e) != b || !cut.keeps(key, i)) return;
                    atomicAdd(&s.count[0][part_of(e)], 1u);
                    // up to 2^24 values of at most 2^38 beside their count
                    atomicAdd(&s.excess[0][part_of(e)], bin_excess(bin_entry(power_of<true>(e).p)));
                });
                __syncthreads();
                const unsigned c = s.count[0][lane], c_upto = wave_upto(c);
                const double w = bin_mass(c, s.excess[0][lane], D) / unit, w_upto = wave_upto(w);
                if (BY == BY_KEY) {
                    sub = part_of((double)key_value(t) * a);
                } else {
                    const unsigned long long enough = __ballot(c > 0 && (BY == BY_MASS ? before + w_upto >= target : (double)first + c_upto >= target));
                    const unsigned long long some = __ballot(c > 0);
                    if (!some) return false;
                    sub = enough ? __builtin_ctzll(enough) : 63 - __builtin_clzll(some);
                }
                if (of_lane(c, sub) > SA_LIST) return false;
                first += (int)of_lane(c_upto - c, sub);
                before += of_lane(w_upto - w, sub);
            }
            __syncthreads();
            if (tid == 0) s.n = 0;
            __syncthreads();
            each_of_bin(D, [&](uint32_t key, int i) {
                const double e = (double)key_value(key) * a;
                if (__builtin_rint(e) == b && cut.keeps(key, i) && (sub < 0 || part_of(e) == sub)) put(key, i);
            });
            __syncthreads();
            kept = min(s.n, SA_LIST);
            rank(kept);
            part = sub >= 0;
            bin = part ? -1 : D;
        }
        int stay;
        if (BY == BY_COUNT) {
            stay = min((int)target - first, kept);
        } else {
            __syncthreads();
            if (tid == 0) s.n = kept;
            __syncthreads();
            for (int i = tid; i < kept; i += THREADS)
                if (BY == BY_MASS ? before + s.upto[i] >= target : s.sorted_key[i] < t) atomicMin(&s.n, i);
            __syncthreads();
            stay = BY == BY_MASS ? min(s.n + 1, kept) : s.n;
        }
        if (BY != BY_KEY && stay <= 0) return false;  // a filter that would not be applied
        kept = stay;
        deepest = D;
        cut = BY == BY_KEY ? Cut{t, 0x7fffffff} : Cut{s.sorted_key[kept - 1], s.sorted_index[kept - 1]};
        total = before + (kept ? s.upto[kept - 1] : 0.0);
        return true;
    }
    // What stays of each piece: from its list where this holds it, or its bins above the last one and the ranked values
    // that are its.  False where neither says.
    __device__ __forceinline__ bool in_lists() const { return deepest <= reach; }
    __device__ __forceinline__ bool weigh_pieces(const Cut &cut, double *piece) const {
        if (!in_lists() && part) return false;
        const int whole = deepest != bin ? deepest + 1 : deepest;
        for (int p = wave; p < pieces; p += WAVES) {
            double sum = 0.0;
            if (in_lists()) {
                const int n = stats[p].at == GRID_LOW ? 0 : min(stats[p].listed, SA_LISTED);
                for (int i = lane; i < n; i += 64) {
                    const uint2 y = lists[(size_t)p * SA_LISTED + i];
                    if (cut.keeps(y.x, (int)y.y)) sum += weight(y.x);
                }
            } else {
                const unsigned long long b = row_bin(p);
                if (lane < whole) sum = bin_mass(bin_count(b), bin_excess(b), lane) / unit;
                if (whole == deepest)
                    for (int k = lane; k < kept; k += 64)
                        if (s.sorted_index[k] / SA_PIECE == p) sum += weight(s.sorted_key[k]);
            }
            sum = wave_all_add(sum);
            if (lane == 0) piece[p] = sum;
        }
        return true;
    }
};

// A row from which nothing can be drawn.
template <bool DRAW>
QG_DEV void no_draw(const SampleArgs &A, int row, int tid, float top) {
    if (DRAW) {
        if (tid < A.draws) {
            A.token[(size_t)row * A.draws + tid] = -1;
            if (A.logprob) A.logprob[(size_t)row * A.draws + tid] = __builtin_nanf("");
        }
    } else if (tid == 0) {
        A.results[row] = RowResult{0, 0, top, top == -__builtin_inff() ? ROW_NONE : ROW_NAN, 0.0, 0.0};
    }
}

template <bool DRAW, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void sample_select_kernel(SampleArgs A, int pieces) {
    constexpr int THREADS = 64 * WAVES;
    __shared__ SelectShared<WAVES> s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PieceStat *stats = A.stats + (size_t)row * pieces;
    // a piece a lane, the same in every wave, or where they are more a piece a thread
    const bool few = pieces <= 64;
    const int from = few ? lane : tid, step = few ? 64 : THREADS;
    const PieceStat none{-__builtin_inff(), GRID_LOW, 0, 0, 0, 0, 0, 0, 0.0, 0.0}, mine = from < pieces ? stats[from] : none;
    const Request q = read_request(A, row);
    uint2 lists[Grid<WAVES>::EACH][Grid<WAVES>::PER];  // on their way from here
    if (few && q.filters()) Grid<WAVES>::read_lists(A.listed + (size_t)row * pieces * SA_LISTED, pieces, mine, wave, lane, lists);
    float top = mine.top;
    for (int p = from + step; p < pieces; p += step) top = larger_or_nan(top, stats[p].top);
    const bool nan = __any(top != top);
    top = nan ? __builtin_nanf("") : qg_wave_max(top);
    if (!few) {
        if (lane == 0) s.top[wave] = top;
        __syncthreads();
        top = s.top[0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) top = larger_or_nan(top, s.top[w]);
    }
    if (!__builtin_isfinite(top)) return no_draw<DRAW>(A, row, tid, top);
    Row<WAVES> r{A, s.row, A.x + (size_t)row * A.cols, tid, lane, wave, q.a, top};
    double *piece = A.kept + (size_t)row * pieces;
    Cut cut;
    double total = 0.0;
    const double place = grid_place(top, q.a);
    bool found = false, weighed = false, listed = false;  // listed: the pieces' lists hold what stays
    if (__builtin_fabs(place) < 0.5 * GRID_FAR) {
        // as bins have it, and a quotient: values that equal the largest weigh whole numbers, of which a top-p may be one
        const double p_top = power_of<true>((double)top * q.a).p, unit = q.filters() ? bin_mass(1, bin_excess(bin_entry(p_top)), 0) : p_top;
        // the bins that every piece's list and bins cover, and the weight of all
        int reach = SA_GRID - 1, known = SA_GRID - 1, counted = 0;
        bool below = false;
        double all = 0.0;
        for (int p = from; p < pieces; p += step) {
            const PieceStat y = p == from ? mine : stats[p];
            const int delta = (int)place - y.at;
            const bool counts = y.at != GRID_LOW && delta < SA_ZERO;
            const double w = counts ? __builtin_amdgcn_ldexp(y.all, -delta) / unit : 0.0;
            if (!q.filters()) piece[p] = w;
            all += w;
            if (!counts) continue;
            reach = min(reach, delta + y.cover);
            known = min(known, delta + y.known);
            counted += y.counted;
            below |= y.below != 0;
        }
        if (!q.filters()) {
            found = weighed = true;
        } else {
            all = wave_all_add(all);
            reach = -(int)qg_wave_max(-(float)reach);
            known = -(int)qg_wave_max(-(float)known);
            long in_all = (long)wave_all_add(counted) + (__any(below) ? 1 << 30 : 0);  // as many as there are, or more
            if (!few) {
                if (lane == 0) { s.reach[wave] = reach; s.known[wave] = known; s.flag[wave] = (int)min(in_all, 1L << 30); s.grid.wave_sum[wave] = all; }
                __syncthreads();
                in_all = 0;
                all = 0.0;
#pragma unroll
                for (int w = 0; w < WAVES; w++) {
                    reach = min(reach, s.reach[w]);
                    known = min(known, s.known[w]);
                    in_all += s.flag[w];
                    all += s.grid.wave_sum[w];
                }
            }
            Grid<WAVES> g{s.grid, r.x, A.bins + (size_t)row * pieces * SA_GRID, stats, mine, A.listed + (size_t)row * pieces * SA_LISTED, A.cols, pieces,
                          tid, lane, wave, (int)place, top, q.a, unit, reach, known, false};
            g.add_up();
            g.below = in_all > (long)of_lane(g.count_upto, known);
            total = q.weighs_all() ? all : of_lane(g.mass_upto, SA_GRID - 1);
            const uint32_t least = q.min_p > 0.0 ? r.least_key(q.min_p) : 0;
            g.hold(g.first_cut(q, all, least), lists);
            found = true;
            if (q.top_k) found = g.template shorten<Grid<WAVES>::BY_COUNT>(q.top_k, 0, cut, total);
            if (found && q.top_p < 1.0) found = g.template shorten<Grid<WAVES>::BY_MASS>(q.top_p * total, 0, cut, total);
            if (found && least > cut.t) found = g.template shorten<Grid<WAVES>::BY_KEY>(0.0, least, cut, total);
            if (found && DRAW && g.held) {
                const int n = g.held;
                __syncthreads();
                g.sum_up(s.grid.in_order, n, [&](int i) { return cut.keeps(s.grid.held[i].x, (int)s.grid.held[i].y) ? g.weight(s.grid.held[i].x) : 0.0; });
                for (int d = wave; d < A.draws; d += WAVES) {
                    // the first sum past the goal, in two steps of 64 and at most 32
                    const size_t at = (size_t)row * A.draws + d;
                    const double sum = s.grid.in_order[n - 1], goal = (double)A.u[at] * sum;
                    const int each = (n + 63) / 64;
                    unsigned long long hit = __ballot(lane * each < n && s.grid.in_order[min((lane + 1) * each, n) - 1] > goal);
                    const int i0 = hit ? (int)__builtin_ctzll(hit) * each : 0;
                    hit = __ballot(hit && lane < each && i0 + lane < n && s.grid.in_order[min(i0 + lane, n - 1)] > goal);
                    int pick = hit ? i0 + (int)__builtin_ctzll(hit) : n - 1;
                    while (pick > 0 && !cut.keeps(s.grid.held[pick].x, (int)s.grid.held[pick].y)) pick--;  // past the last one: it is
                    if (lane == 0) {
                        const uint2 y = s.grid.held[pick];
                        A.token[at] = (int)y.y;
                        if (A.logprob) A.logprob[at] = (float)log(g.weight(y.x) / sum);
                    }
                }
                return;
            }
            if (found && DRAW) {
                weighed = g.weigh_pieces(cut, piece);
                listed = g.in_lists();
            }
        }
    }
    if (!found) {
        __syncthreads();
        cut = Cut{};
        for (int by = 0; by < 2; by++)
            if (by ? q.top_p < 1.0 : q.top_k > 0) r.shorten(cut, by != 0, by ? q.top_p : q.top_k);
        if (q.min_p > 0.0) {
            const uint32_t k = r.least_key(q.min_p);
            if (k > cut.t) cut = Cut{k, 0x7fffffff};
        }
    }
    if (!weighed && (DRAW || !found)) {
        for (int p = wave; p < pieces; p += WAVES) {
            double sum = 0.0;
            each_value<64>(r.x, p * SA_PIECE + lane, min((p + 1) * SA_PIECE, A.cols), [&](int i, float v) { sum += cut.keeps(order_key(v), i) ? r.weight(v) : 0.0; });
            sum = wave_all_add(sum);
            if (lane == 0) piece[p] = sum;
        }
        weighed = true;
    }
    if (weighed) {
        __syncthreads();
        total = 0.0;
        for (int p0 = 0; p0 < pieces; p0 += 64) total += wave_all_add(p0 + lane < pieces ? piece[p0 + lane] : 0.0);
    }
    if (!DRAW) {
        if (tid == 0) A.results[row] = RowResult{cut.t, cut.last, top, ROW_CUT, q.a, total};
        return;
    }
    for (int d = wave; d < A.draws; d += WAVES) {
        const size_t at = (size_t)row * A.draws + d;
        const double goal = (double)A.u[at] * total;
        // the piece that passes the goal, or the last one that holds something
        double before = 0.0;
        int p = -1;
        bool past = false;
        for (int p0 = 0; p0 < pieces && !past; p0 += 64) {
            const double v = p0 + lane < pieces ? piece[p0 + lane] : 0.0, upto = wave_upto(v) + before;
            const unsigned long long hit = __ballot(v > 0.0 && upto > goal), any = __ballot(v > 0.0);
            if (!any) continue;
            const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
            p = p0 + l;
            past = hit != 0;
            before = past ? of_lane(upto - v, l) : of_lane(upto, 63);
        }
        const bool last = !past;  // no token passes: the last one
        int pick = -1;
        double won = 0.0;
        past = false;
        if (listed) {
            const uint2 *list = A.listed + ((size_t)row * pieces + p) * SA_LISTED;
            const int n = min(stats[p].listed, SA_LISTED);
            for (int i0 = 0; i0 < n && !past; i0 += 64) {
                const uint2 y = i0 + lane < n ? list[i0 + lane] : make_uint2(0, 0);
                const double w = i0 + lane < n && cut.keeps(y.x, (int)y.y) ? r.weight(key_value(y.x)) : 0.0, upto = wave_upto(w) + before;
                const unsigned long long hit = __ballot(!last && w > 0.0 && upto > goal), any = __ballot(w > 0.0);
                if (!any) continue;
                const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
                pick = (int)of_lane(y.y, l);
                won = of_lane(w, l);
                past = hit != 0;
                before = of_lane(upto, 63);
            }
        }
        // Read again, the piece may weigh less than what was recorded of it, and the goal lie between the two: bins round, and powers
        // of x a differ from those of (x - max) a by what the products were rounded.  Then it is the last token that stays.
        const int end = min((p + 1) * SA_PIECE, A.cols);
        int full = -1;  // the last chunk that holds something, if it was passed over
        bool take = last;
        for (int i0 = listed ? end : p * SA_PIECE; i0 < end && !past; i0 += 16 * 64) {
            float v[16];
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] = i0 + k * 64 + lane < A.cols ? r.x[i0 + k * 64 + lane] : -__builtin_inff();
            unsigned stays = 0;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                if (v[k] > -__builtin_inff() && cut.keeps(order_key(v[k]), i0 + k * 64 + lane)) { stays |= 1u << k; sum += r.weight(v[k]); }
            }
            sum = wave_all_add(sum);
            if (sum > 0.0 && !take && !(before + sum * (1.0 + 1e-12) > goal)) {
                before += sum;
                full = i0;
            } else if (sum > 0.0) {
                full = -1;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    if (past || !__any(stays >> k & 1)) continue;
                    const double w = stays >> k & 1 ? r.weight(v[k]) : 0.0, upto = wave_upto(w) + before;
                    const unsigned long long hit = __ballot(!take && w > 0.0 && upto > goal), any = __ballot(w > 0.0);
                    if (!any) continue;
                    const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
                    pick = i0 + k * 64 + l;
                    won = of_lane(w, l);
                    past = hit != 0;
                    before = of_lane(upto, 63);
                }
            }
            if (full >= 0 && i0 + 16 * 64 >= end) {  // no token passed, and the last one has not been looked at
                take = true;
                i0 = full - 16 * 64;
            }
        }
        if (lane == 0) {
            A.token[at] = pick;
            if (A.logprob) A.logprob[at] = (float)log(won / total);
        }
    }
}
// Workgroups of sixteen waves, or of eight where the rows are more than the CUs: 300 rows x 151936 97 us (sixteen 105), 512 x 50000
// 70 (89), 1088 x 131072 243 (274).  Up to 256 rows eight take 1 us less where the bins and lists serve (68 x 50000 35.3 and 36.4),
// but much longer where rows are read again: a flat row of 151936 442 (sixteen 386), top-k 5000 of 17 such rows 68 (54), 4 rows x
// 2^20 114 (76).
template <bool DRAW>
void select_rows(const SampleArgs &A, int rows, int pieces, hipStream_t s) {
    if (rows > 256) sample_select_kernel<DRAW, 8><<<rows, 512, 0, s>>>(A, pieces);
    else sample_select_kernel<DRAW, 16><<<rows, 1024, 0, s>>>(A, pieces);
}

// Probabilities of a piece; one that lies below the cut is not read.  Bound by memory: 1088 rows x 131072 140 us, 570 MB
// written at 4.1 TB/s.
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
    A.listed = (uint2 *)(A.bins + all * SA_GRID);
    A.kept = (double *)(A.listed + all * SA_LISTED);
    return A;
}
}  // namespace

extern "C" {

size_t qg_sample_workspace_bytes(int rows, int cols) {
    if (rows < 1 || rows > QG_MAX_ROWS || cols < 1 || cols > SA_MAX_COLS || (long)rows * cols > 1L << 35) return 0;
    return (size_t)rows * (sizeof(RowResult) + sample_pieces(cols) * (sizeof(PieceStat) + SA_GRID * sizeof(unsigned long long) + SA_LISTED * sizeof(uint2) + sizeof(double)));
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
    select_rows<true>(A, rows, pieces, qg_stream());
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
    select_rows<false>(A, rows, pieces, qg_stream());
    sample_probs_kernel<<<(unsigned)((size_t)rows * pieces), PIECE_THREADS, 0, qg_stream()>>>(A, pieces);
    return hipGetLastError();
}

}  // extern "C"
