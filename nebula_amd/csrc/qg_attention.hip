// Attention of a batch's rows over the paged cache (qg_tree_attention of
// include/qwen_gpu.h).
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), in one pass over the
// keys with a running m.  A kv head's rows (its group's heads of every row of the
// batch, in groups of 16 RT) share one read of its keys and values.  Keys are
// split over workgroups (the number follows from the lengths, on the device),
// over a workgroup's waves and within a wave into tiles of 32 (16 for F32); the
// parts are joined in shared memory, and by a second kernel where a sequence has
// more than one workgroup.
//
// A wave needs nothing of the others while it walks: keys and values go from
// memory to its registers.  Scores are formed transposed, S^T = K Q^T (keys the
// rows of the product), so that a lane ends with the scores of 8 consecutive
// keys of one query row, which is what the second product, O^T = V^T P^T, wants
// of it as an operand; for V^T a lane holds 8 keys x D/16 dimensions as they lie
// in memory and pairs them with byte permutes.  Neither product moves a value
// between lanes.
//
// What bounds it (MI355X, fp16 cache, 16 heads over 2, 128 dimensions).  Up to 48 rows
// of a head (one row group): memory, 16 sequences x 98304 keys 282 us with 1 row of each,
// 286 with 2 and 291 with 6, 5.6 to 5.7 TB/s (a large read reaches 6.1).  More row groups
// share the reads in the L2 but each adds its products and softmax: 431 us with 12 rows,
// 621 with 17 (the matrix cores busy for a third of the time, the rest a wave's latencies
// with two waves per SIMD).  One sequence of 24576 keys, 17 rows (bf16): 34 us and 5 for the
// join, of which 13 before the first product and after the last.
//
// Precision: q and p enter as planes that the 16-bit cores multiply exactly with
// the cache's values: two fp16 planes (22 bits; q scaled by a power of two per
// row), three bf16 planes (24 bits); an F32 cache uses the fp32 cores.
#include "qg_kv.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// p is held times 2^P_BASE, and a new maximum counts once it is 2^M_LAG above the old.
// fp16 planes end at 2^-24 and at 2^16: what the base and the lag leave of that below the
// range's end is what small weights have for their bits.  Base 13 and lag 2 hold a weight
// within 2^-22 of itself or 2^-38 of the largest (base 6 and lag 8, rounded towards zero:
// 2^-30, always too little).  bf16 planes and fp32 have the exponent for any weight.
constexpr float p_base(int type) { return type == QT_F16 ? 13.0f : 0.0f; }
constexpr float m_lag(int type) { return type == QT_F16 ? 2.0f : 8.0f; }

struct AttnArgs {
    float *out;
    const float *q;
    float *part_o;   // [slots][row group][D]
    float2 *part_ml; // [slots][row group]
    int4 *joins;     // [rows][q_heads]: what attention_join_kernel has to do, see Join
    float scale;     // times log2 e
    int q_heads, group, layer, resident, slots, run;  // resident: workgroups that run at once; run: see plan_find
    unsigned group_inv;                          // 2^32 / group, rounded up
};

// x / group for x < 2^24: the product is over by less than x / 2^32 < 1 / group.
QG_DEV int by_group(const AttnArgs &A, int x) { return A.group == 1 ? x : (int)__umulhi((unsigned)x, A.group_inv); }

// How the work is cut, the same in every wave.  Sequence s has
// `groups` row groups and `keys` keys; its keys are cut into parts of `chunk`,
// chosen so that about as many workgroups have work as run at once.
struct Plan {
    int s, first, n, len, groups, chunk, part, z, h;  // of one unit
    size_t slot;  // of part 0, row group 0, head 0 of the sequence
};
constexpr int CHUNK = 128;  // keys per workgroup, at least and in steps of

// A lane's sequence: its rows, tokens and row groups.
struct PlanLane { int first, n, len, groups; };
template <int RG>
QG_DEV PlanLane plan_lane(const KvView &c, const BatchView &b, const AttnArgs &A, int s) {
    PlanLane x{0, 0, 0, 0};
    if (s < c.sequences) {
        batch_rows(b, s, x.first, x.n);
        x.len = kv_length(c, s);
        x.groups = (x.n * A.group + RG - 1) / RG;
    }
    return x;
}

// The unit of a workgroup.  Units run through the sequences (parts x heads x row
// groups) in runs that go to one XCD, so that row groups with the same keys meet
// in its L2: an eighth of them all where they are alike (each XCD then gets as many
// as it runs at once), sixteen and sixteen where a prompt's rows see more and more.
// False if there is none.
template <int RG>
QG_DEV bool plan_find(const KvView &c, const BatchView &b, const AttnArgs &A, int lane, int block, Plan &p) {
    const PlanLane mine = plan_lane<RG>(c, b, A, lane);
    // a sum over all sequences of what `f` says of each
    auto over = [&](auto f) {
        float v = f(mine);
        for (int s = lane + 64; s < c.sequences; s += 64) v += f(plan_lane<RG>(c, b, A, s));
        v = qg_row_sum(v);
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 64; i += 16) x += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
        return x * (float)c.heads;
    };
    // One round of resident workgroups, each with one unit: a second round for a few
    // units would cost as much as the first.  Where the row groups alone come to half
    // a round, two rounds.
    const float least = over([](const PlanLane &x) { return (float)x.groups; });
    const bool single = 2.0f * least <= (float)A.resident;
    const float room = single ? (float)A.resident : 2.0f * (float)A.resident;
    // 1.0001: above the sum whatever its roundings, so that the slots suffice
    const float even = 1.0001f * over([](const PlanLane &x) { return (float)x.groups * (float)(x.len + x.n); }) / room;
    int chunk = ((int)fminf(even, (float)(1 << 28)) / CHUNK + 1) * CHUNK;
    for (int i = 0; i < 4 && !A.run && least <= room; i++) {  // the parts round up: longer ones until they fit
        const float units = over([&](const PlanLane &x) { return x.n ? (float)(((x.len + x.n - 1) / chunk + 1) * x.groups) : 0.0f; });
        if (units <= room) break;
        chunk = max((int)fminf((float)chunk * units / room, (float)(1 << 28)) / CHUNK, chunk / CHUNK) * CHUNK + CHUNK;
    }
    auto scan = [&](int s0, PlanLane &x, int &parts, int &upto, int &upto_slots) {
        x = s0 ? plan_lane<RG>(c, b, A, s0 + lane) : mine;
        parts = x.n ? (x.len + x.n - 1) / chunk + 1 : 0;
        upto = parts * x.groups * c.heads;
        upto_slots = parts > 1 ? upto : 0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int u = __shfl_up(upto, d), e = __shfl_up(upto_slots, d);
            if (lane >= d) { upto += u; upto_slots += e; }
        }
    };
    PlanLane x;
    int parts, upto, upto_slots, units = 0;
    for (int s0 = 0; s0 < c.sequences; s0 += 64) {
        scan(s0, x, parts, upto, upto_slots);
        units += __builtin_amdgcn_readlane(upto, 63);
    }
    if (units <= 0) return false;
    const int run = A.run ? A.run : (units + 7) / 8, k = block >> 3;
    const int unit = (k / run * 8 + (block & 7)) * run + k % run;
    if (unit >= units) return false;
    int before = 0;
    size_t slots = 0;
    for (int s0 = 0; s0 < c.sequences; s0 += 64) {
        if (c.sequences > 64) scan(s0, x, parts, upto, upto_slots);
        const int own = parts * x.groups * c.heads, own_slots = parts > 1 ? own : 0;
        const unsigned long long here = __ballot(unit < before + upto && unit >= before + upto - own);
        if (here) {
            const int l = __builtin_ctzll(here);
            p.s = s0 + l;
            p.first = __builtin_amdgcn_readlane(x.first, l);
            p.n = __builtin_amdgcn_readlane(x.n, l);
            p.len = __builtin_amdgcn_readlane(x.len, l);
            p.groups = __builtin_amdgcn_readlane(x.groups, l);
            p.slot = slots + __builtin_amdgcn_readlane(upto_slots - own_slots, l);
            const int rest = unit - (before + __builtin_amdgcn_readlane(upto - own, l));
            if (rest < 0 || rest >= __builtin_amdgcn_readlane(own, l)) return false;  // row starts that overlap, past 2^31 units
            p.part = rest / (p.groups * c.heads);
            p.h = rest / p.groups % c.heads;
            p.z = p.groups - 1 - rest % p.groups;  // the last rows, which see the most, first
            p.chunk = chunk;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(upto_slots, 63);
    }
    return false;
}

// What is left to do for a row and head: nothing (parts 1, odd 0), to join `parts`
// partial results from `slot` on, `step` apart, or to take the row up again (odd 1).
struct Join {
    int parts, slot, step, odd;
    // Inside the slots: not what the memory held where row starts that overlap leave a unit out.
    __device__ bool inside(long slots) const {
        return parts > 0 && parts <= slots && slot >= 0 && slot < slots && step > 0 && step <= slots && slot + (parts - 1L) * step < slots;
    }
};

// v_perm of two words into (a.lo, b.lo) or (a.hi, b.hi)
QG_DEV uint32_t pair_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
QG_DEV uint32_t pair_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Eight floats as the planes of an operand: their sum is the value (bf16, exactly) or
// within 2^-23 of it, and 2^-25 where that is more (fp16, both rounded to nearest).
template <int TYPE> struct Planes;
template <> struct Planes<QT_F16> {
    static constexpr int N = 2;
    uint4 p[2];
    __device__ __forceinline__ explicit Planes(const float (&x)[8]) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            hi[i] = cvt2(x[2 * i], x[2 * i + 1]);
            // x - hi in one instruction each
            float a, b;
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(hi[i]), "v"(x[2 * i]));
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(hi[i]), "v"(x[2 * i + 1]));
            lo[i] = cvt2(a, b);
        }
        p[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        p[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    static __device__ __forceinline__ uint32_t cvt2(float a, float b) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
    }
    static __device__ __forceinline__ qg_f4 mul(uint4 a, uint4 b, qg_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(qg_half8, a), __builtin_bit_cast(qg_half8, b), c, 0, 0, 0);
    }
};
template <> struct Planes<QT_BF16> {
    static constexpr int N = 3;
    uint4 p[3];
    __device__ __forceinline__ explicit Planes(const float (&x)[8]) {
        uint32_t w[3][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
                w[k][i] = pair_hi(ua, ub);
                a -= __uint_as_float(ua & 0xffff0000u);
                b -= __uint_as_float(ub & 0xffff0000u);
            }
        }
#pragma unroll
        for (int k = 0; k < 3; k++) p[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    }
    static __device__ __forceinline__ qg_f4 mul(uint4 a, uint4 b, qg_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

// A tile's keys and values in a wave's registers and their products, by the cache's
// type.  Lane l: n = l % 16, g = l / 16.  KEYS keys per tile, E of them (E g .. E g +
// E - 1) in a lane's scores and values; DL = D/16 dimensions (DL n ..) in its values.
template <int TYPE, int D>
struct Tile {
    static constexpr int KEYS = 32, E = 8, DL = D / 16, S = D / 32, PL = Planes<TYPE>::N, ES = 2;
    uint4 k[2][S];
    uint32_t v[8][DL / 2];
    // the key (of the tile) whose row a lane loads as the first operand's row n of sub-tile j
    static __device__ __forceinline__ int key_of(int n, int j) { return 8 * (n >> 2) + (n & 3) + 4 * j; }
    // at: byte offset of key 8 (n / 4)'s row; the next keys follow
    __device__ __forceinline__ void load_k(const uint8_t *at, int n, int g) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int s = 0; s < S; s++) k[j][s] = *(const uint4 *)(at + ((n & 3) + 4 * j) * (D * 2) + s * 64 + g * 16);
    }
    __device__ __forceinline__ void load_v(const uint8_t *at, int n) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint8_t *p = at + e * (D * 2) + n * (DL * 2);
            if constexpr (DL == 4) {
                const uint2 x = *(const uint2 *)p;
                v[e][0] = x.x; v[e][1] = x.y;
            } else {
#pragma unroll
                for (int w = 0; w < DL / 8; w++) {
                    const uint4 x = *(const uint4 *)(p + 16 * w);
                    v[e][4 * w] = x.x; v[e][4 * w + 1] = x.y; v[e][4 * w + 2] = x.z; v[e][4 * w + 3] = x.w;
                }
            }
        }
    }
    __device__ __forceinline__ void drop_v(int e) {
#pragma unroll
        for (int w = 0; w < DL / 2; w++) v[e][w] = 0;
    }
    // q fragments: [s][plane][lane] of 16 bytes
    static constexpr int Q_BYTES = S * PL * 1024;
    static __device__ __forceinline__ void put_q(uint8_t *frag, int n, int d0, const float (&x)[8], int first) {
        const Planes<TYPE> p(x);
#pragma unroll
        for (int k = 0; k < PL; k++) {
            uint8_t *to = frag + (((d0 >> 5) * PL + k) * 64 + ((d0 >> 3) & 3) * 16 + n) * 16;
            if constexpr (DL == 4) *(uint2 *)(to + (d0 & 4) * 2) = make_uint2(p.p[k].x, p.p[k].y);
            else *(uint4 *)to = p.p[k];
        }
    }
    // The row tiles' queries are read half a tile ahead of their products where
    // registers are left for it (two fp16 planes: 16 x 17 rows x 98304 keys 656 -> 628
    // us; three bf16 planes at 128 dimensions, or one row tile with a third wave per
    // SIMD, lose more to the registers: 1 row x 98304 keys 33 -> 37).
    template <int RT>
    __device__ __forceinline__ void scores(const uint8_t *frag, int lane, float (&z)[RT][8]) const {
        constexpr bool AHEAD = RT > 1 && (TYPE == QT_F16 || D == 256);
        constexpr int H = S / 2 * PL;  // fragments of a half
        uint4 q[2][H];
        auto read = [&](int half, uint4 (&to)[H]) {
#pragma unroll
            for (int i = 0; i < H; i++) to[i] = *(const uint4 *)(frag + (size_t)half * (H * 1024) + i * 1024 + lane * 16);
        };
        if (AHEAD) read(0, q[0]);
#pragma unroll
        for (int r = 0; r < RT; r++) {
            qg_f4 a[2] = {};
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (!AHEAD) read(2 * r + half, q[half]);
                else if (2 * r + half + 1 < 2 * RT) read(2 * r + half + 1, q[1 - half]);
                if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < H; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) a[j] = Planes<TYPE>::mul(k[j][half * (S / 2) + i / PL], q[half][i], a[j]);
                if (AHEAD || half) __builtin_amdgcn_sched_barrier(0);  // one row tile's queries in registers at a time
            }
#pragma unroll
            for (int i = 0; i < 4; i++) { z[r][i] = a[0][i]; z[r][4 + i] = a[1][i]; }
        }
    }
    template <int RT>
    __device__ __forceinline__ void outputs(const float (&p)[RT][8], qg_f4 (&o)[RT][DL]) const {
        uint4 w[RT][PL];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const Planes<TYPE> x(p[r]);
#pragma unroll
            for (int k = 0; k < PL; k++) w[r][k] = x.p[k];
        }
        // two dimension tiles at a time: products that add to one sum lie apart
#pragma unroll
        for (int t = 0; t < DL; t += 2) {
            uint4 a[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] = h ? pair_hi(v[2 * i][t / 2], v[2 * i + 1][t / 2]) : pair_lo(v[2 * i][t / 2], v[2 * i + 1][t / 2]);
                a[h] = make_uint4(u[0], u[1], u[2], u[3]);
            }
#pragma unroll
            for (int k = 0; k < PL; k++)
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int h = 0; h < 2; h++) o[r][t + h] = Planes<TYPE>::mul(a[h], w[r][k], o[r][t + h]);
        }
    }
};
template <int D>
struct Tile<QT_F32, D> {
    static constexpr int KEYS = 16, E = 4, DL = D / 16, S = D / 16, ES = 4;
    float4 k[S];
    float v[4][DL];
    __device__ __forceinline__ void load_k(const uint8_t *at, int n, int g) {
#pragma unroll
        for (int s = 0; s < S; s++) k[s] = *(const float4 *)(at + (n & 3) * (D * 4) + s * 64 + g * 16);
    }
    __device__ __forceinline__ void load_v(const uint8_t *at, int n) {
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int w = 0; w < DL / 4; w++) {
                const float4 x = *(const float4 *)(at + e * (D * 4) + n * (DL * 4) + 16 * w);
                v[e][4 * w] = x.x; v[e][4 * w + 1] = x.y; v[e][4 * w + 2] = x.z; v[e][4 * w + 3] = x.w;
            }
    }
    __device__ __forceinline__ void drop_v(int e) {
#pragma unroll
        for (int w = 0; w < DL; w++) v[e][w] = 0.0f;
    }
    static constexpr int Q_BYTES = S * 1024;
    static __device__ __forceinline__ void put_q(uint8_t *frag, int n, int d0, const float (&x)[8], int count) {
#pragma unroll
        for (int i = 0; i < 8; i += 4)
            if (i < count) {
                const int d = d0 + i;
                *(float4 *)(frag + ((d >> 4) * 64 + ((d >> 2) & 3) * 16 + n) * 16) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
            }
    }
    template <int RT>
    __device__ __forceinline__ void scores(const uint8_t *frag, int lane, float (&z)[RT][4]) const {
#pragma unroll
        for (int r = 0; r < RT; r++) {
            qg_f4 a = {};
#pragma unroll
            for (int s = 0; s < S; s++) {
                const float4 q = *(const float4 *)(frag + ((r * S + s) * 64 + lane) * 16);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s].x, q.x, a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s].y, q.y, a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s].z, q.z, a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s].w, q.w, a, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) z[r][i] = a[i];
            __builtin_amdgcn_sched_barrier(0);  // one row tile's queries in registers at a time
        }
    }
    template <int RT>
    __device__ __forceinline__ void outputs(const float (&p)[RT][4], qg_f4 (&o)[RT][DL]) const {
#pragma unroll
        for (int t = 0; t < DL; t++)
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[r][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e][t], p[r][e], o[r][t], 0, 0, 0);
    }
};

// Sums that are no numbers, or a weight that is none.  The planes' products make NaN
// of an infinite key, query or value (0 x inf, inf - inf) where the score may be minus
// infinity, and a value that is no number reaches the rows of its tile that do not see
// it (0 x NaN); such rows are taken up again, key by key, and so are sums of finite
// values past the type's range, which their division by the weight may bring back.  Weights are at most
// 2^(m_lag + p_base), so their sum is never infinite.
QG_DEV bool odd_sums(float a, float b, float weight) { return !__builtin_isfinite(a + b + weight); }

QG_DEV unsigned first_bits(int n, int most) { return (1u << min(max(n, 0), most)) - 1u; }

// What a part's sums (under its largest score m, weights l) count under another
// maximum; below zero for one without a visible key, whose sums may be anything.
QG_DEV float part_weight(float m, float l, float top) {
    return m == -__builtin_inff() && l == 0.0f ? -1.0f : m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

template <int TYPE, int D, int RT, int NW>
__global__ __launch_bounds__(64 * NW, (D / 64) * RT <= 6 ? 2 : 1) void attention_kernel(AttnArgs A, KvView c, BatchView b) {
    typedef Tile<TYPE, D> T;
    constexpr int RG = 16 * RT, E = T::E, DL = T::DL, KEYS = T::KEYS, JOIN = NW * 16 * (D + 4) * 4;
    // a wave in its products goes before one in its softmax (2048-row chunk at 256 dimensions 540 -> 502 us; at 64
    // dimensions, where the softmax is most of the time, 204 -> 213: not there)
    constexpr bool FIRST = D > 64;
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[RT * T::Q_BYTES > JOIN ? RT * T::Q_BYTES : JOIN];
    __shared__ float s_m[NW][RG], s_l[NW][RG], s_back[RG];
    __shared__ unsigned long long s_seen[QG_MAX_TREE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    Plan p;
    if (!plan_find<RG>(c, b, A, lane, blockIdx.x, p)) return;
    const int row0 = p.z * RG, rows = p.n * A.group;  // this group's first row, all rows of the head
    // the group's keys, the first one that some row may not see, and this unit's
    const int last_t = by_group(A, min(row0 + RG, rows) - 1), begin = p.part * p.chunk;
    const int keys = p.len + (b.parent ? p.n : last_t + 1), open = p.len + (b.parent ? 0 : by_group(A, row0) + 1);
    const int parts = (keys - 1) / p.chunk + 1, end = min(begin + p.chunk, keys);
    if (p.part >= parts) return;  // rows that come before the sequence's last keys
    // the queries first: what is read in front of them would have to arrive before them
    float x[RG / (4 * NW)][DL];
    size_t at_q[RG / (4 * NW)];  // the row and head, or -1
#pragma unroll
    for (int i = 0; i < RG / (4 * NW); i++) {
        const int at = row0 + (i * NW + wave) * 4 + g, t = by_group(A, at);
        at_q[i] = at < rows ? (size_t)(p.first + t) * A.q_heads + p.h * A.group + (at - t * A.group) : (size_t)-1;
#pragma unroll
        for (int d = 0; d < DL; d += 4) {
            const float4 y = at < rows ? *(const float4 *)(A.q + at_q[i] * D + n * DL + d) : make_float4(0, 0, 0, 0);
            x[i][d] = y.x; x[i][d + 1] = y.y; x[i][d + 2] = y.z; x[i][d + 3] = y.w;
        }
    }
    const size_t page_bytes = ((size_t)c.heads << c.shift) * D * T::ES;
    const uint8_t *kbase = c.k + (((size_t)A.layer * c.pages * c.heads + p.h) << c.shift) * D * T::ES;
    const uint8_t *vbase = c.v + (((size_t)A.layer * c.pages * c.heads + p.h) << c.shift) * D * T::ES;
    const int slot_mask = (1 << c.shift) - 1;
    // a run of E keys from position pos, aligned to E: inside one page
    auto run = [&](const uint8_t *base, int page, int pos) { return base + (size_t)max(page, 0) * page_bytes + (size_t)((pos & slot_mask) * (D * T::ES)); };
    // the first tile's keys and values, and the second's pages, are on their way while the queries are laid out
    T tile;
    int t0 = begin + wave * KEYS, kpos = t0 + E * (n >> 2), vpos = t0 + E * g;
    int kpage = kv_page(c, p.s, kpos), vpage = kv_page(c, p.s, vpos);
    int kpage1 = kv_page(c, p.s, kpos + NW * KEYS), vpage1 = kv_page(c, p.s, vpos + NW * KEYS);
    if (t0 < end) {
        tile.load_k(run(kbase, kpage, kpos), n, g);
        tile.load_v(run(vbase, vpage, vpos), n);
    }

    // the rows' queries, in planes and in the order of the products' operand; the
    // power of two that a row was scaled by (fp16 planes) comes off the scores
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
        if (n == 0) s_back[r] = back;
        if (n == 0 && p.part == 0 && at_q[i] != (size_t)-1)
            A.joins[at_q[i]] = make_int4(parts, (int)(p.slot + (size_t)p.h * p.groups + p.z), c.heads * p.groups, 0);
        uint8_t *frag = s_mem + (r >> 4) * T::Q_BYTES;
#pragma unroll
        for (int d = 0; d < DL; d += 8) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = d + j < DL ? x[i][(d + j) % DL] : 0.0f;
            T::put_q(frag, r & 15, n * DL + d, y, DL - d);
        }
    }
    if (b.parent && wave == 0) s_seen[lane] = tree_ancestors(b.parent + p.first, p.n, lane);
    __syncthreads();

    qg_f4 o[RT][DL];
    float m[RT], l[RT], back[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) back[r] = TYPE == QT_F16 ? s_back[16 * r + n] : 1.0f;
#pragma unroll
    for (int r = 0; r < RT; r++) {
        m[r] = -__builtin_inff();
        l[r] = 0.0f;
#pragma unroll
        for (int t = 0; t < DL; t++) o[r][t] = qg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (; t0 < end; t0 += NW * KEYS) {
        float z[RT][E];
        if (FIRST) __builtin_amdgcn_s_setprio(1);
        tile.template scores<RT>(s_mem, lane, z);
        if (FIRST) __builtin_amdgcn_s_setprio(0);
        // the next tile's keys, whose pages are known, and the pages of the one after it
        const int here = vpage, here_pos = vpos;
        const bool more = t0 + NW * KEYS < end;
        kpos += NW * KEYS;
        vpos += NW * KEYS;
        vpage = vpage1;
        if (more) {
            tile.load_k(run(kbase, kpage1, kpos), n, g);
            kpage1 = kv_page(c, p.s, kpos + NW * KEYS);
            vpage1 = kv_page(c, p.s, vpos + NW * KEYS);
        }
        if (t0 + KEYS > open || !__all(here >= 0)) {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (here < 0 || here_pos + e >= end) tile.drop_v(e);
#pragma unroll
            for (int r = 0; r < RT; r++) {
                // bit e: key here_pos + e, below the row's prefix or among the rows that it descends from
                const int t = by_group(A, row0 + 16 * r + n), prefix = b.parent ? p.len : p.len + t + 1, k = here_pos - p.len;
                unsigned seen = first_bits(prefix - here_pos, E);
                if (b.parent && t < p.n && k < 64 && k > -E) seen |= (unsigned)(k < 0 ? s_seen[t] << -k : s_seen[t] >> k);
                seen = here < 0 ? 0 : seen & first_bits(end - here_pos, E);
#pragma unroll
                for (int e = 0; e < E; e++) z[r][e] = seen >> e & 1 ? z[r][e] : -__builtin_inff();
            }
        }
        // scores to weights: the maximum is renewed only where it moves by more than M_LAG
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
        if (g == 0) { s_m[wave][16 * r + n] = m[r]; s_l[wave][16 * r + n] = l[r]; }
    }
    __syncthreads();  // the queries' fragments are done with, too
    const size_t slot = p.slot + ((size_t)p.part * c.heads + p.h) * p.groups + p.z;
    const bool fits = slot < (size_t)A.slots;
    if (tid < RG) {
        float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) top = fmaxf(top, s_m[w][tid]);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float lw = s_l[w][tid], f = part_weight(s_m[w][tid], lw, top);
            if (f >= 0.0f) sum = __builtin_fmaf(f, lw, sum);
            s_m[w][tid] = f;
        }
        s_l[0][tid] = sum;
        if (parts > 1 && fits) A.part_ml[slot * RG + tid] = make_float2(top, sum);
    }
    float *join = (float *)s_mem;
#pragma unroll
    for (int r = 0; r < RT; r++) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < DL; t += 4)
                *(float4 *)(join + (wave * 16 + n) * (D + 4) + DL * (4 * g + i) + t) =
                    make_float4(o[r][t][i], o[r][t + 1][i], o[r][t + 2][i], o[r][t + 3][i]);
        __syncthreads();
#pragma unroll
        for (int x0 = 0; x0 < 16 * D / 4; x0 += 64 * NW) {
            const int x = x0 + tid, row = x / (D / 4), d = x % (D / 4) * 4, at = row0 + 16 * r + row;
            if (16 * D / 4 < 64 * NW && x >= 16 * D / 4) break;
            float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float f = s_m[w][16 * r + row];
                const float4 u = *(const float4 *)(join + (w * 16 + row) * (D + 4) + d);
                y.x = f < 0.0f ? y.x : __builtin_fmaf(f, u.x, y.x);
                y.y = f < 0.0f ? y.y : __builtin_fmaf(f, u.y, y.y);
                y.z = f < 0.0f ? y.z : __builtin_fmaf(f, u.z, y.z);
                y.w = f < 0.0f ? y.w : __builtin_fmaf(f, u.w, y.w);
            }
            if (at >= rows) continue;
            const float sum = s_l[0][16 * r + row];
            if (parts == 1) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int t = by_group(A, at);
                const size_t to = (size_t)(p.first + t) * A.q_heads + p.h * A.group + (at - t * A.group);
                *(float4 *)(A.out + to * D + d) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
                if (odd_sums(y.x, y.y, sum) || odd_sums(y.z, y.w, sum)) A.joins[to].w = 1;
            } else if (fits) {
                *(float4 *)(A.part_o + (slot * RG + 16 * r + row) * D + d) = y;
            }
        }
        __syncthreads();
    }
}

// One row and head, key by key: a lane scores one of 64 keys at a time, the
// output's dimensions lie across the lanes.  The weights' sum first, so that the values
// are taken by weights that sum to 1: nothing overflows that the output holds.  A NaN in
// the query or in that sum is the row's.  A wave's latencies bound it: a sequence's rows
// over 98304 keys 18 ms with 16 bytes of a key and eight values on their way at once, 42
// with one; NaN queries cost nothing.
template <int TYPE, int D>
QG_DEV void attend_row(const AttnArgs &A, const KvView &c, const BatchView &b, int s, int first, int n, int row, int head, int lane, float *s_q) {
    constexpr int V = D / 64, E = TYPE == QT_F32 ? 4 : 8;
    const int place = row - first, len = kv_length(c, s), kv = by_group(A, head);
    const unsigned long long seen = b.parent ? __shfl(tree_ancestors(b.parent + first, n, lane), place) : 0;
    const float *q = A.q + ((size_t)row * A.q_heads + head) * D;
    float *out = A.out + ((size_t)row * A.q_heads + head) * D + lane * V;
    bool nan = false;
    for (int d = lane; d < D; d += 64) {
        s_q[d] = q[d] * A.scale;
        nan |= q[d] != q[d];
    }
    __builtin_amdgcn_wave_barrier();  // one wave's own
    const int end = len + (b.parent ? n : place + 1);
    // key t: whether the row sees it, where it lies, its score
    auto score = [&](int t, size_t &at, float &z) {
        const int page = t < end ? kv_page(c, s, t) : -1;
        const bool visible = page >= 0 && (t < len || !b.parent || (seen >> (t - len) & 1));
        at = kv_at(c, A.layer, max(page, 0), kv, t & ((1 << c.shift) - 1));
        z = -__builtin_inff();
        if (visible) {
            z = 0.0f;
            const uint4 *key = (const uint4 *)(c.k + at * (16 / E));
#pragma unroll 2
            for (int d = 0; d < D; d += E) {
                const uint4 w = key[d / E];
#pragma unroll
                for (int e = 0; e < E; e++) z = __builtin_fmaf(s_q[d + e], kv_load<TYPE>((const uint8_t *)&w, e), z);
            }
        }
        return visible;
    };
    size_t at;
    float m = -__builtin_inff(), l = 0.0f, z, o[V];
    for (int t0 = 0; t0 < end && !__any(nan); t0 += 64) {
        const bool visible = score(t0 + lane, at, z);
        const float top = fmaxf(m, qg_wave_max(z)), base = top == -__builtin_inff() ? 0.0f : top;
        l = l * __builtin_amdgcn_exp2f(m - base) + qg_sum_lanes<64>(visible ? __builtin_amdgcn_exp2f(z - base) : 0.0f);
        m = top;
        nan |= l != l;
    }
    nan = __any(nan);
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = nan ? __builtin_nanf("") : 0.0f;
    const float base = m == -__builtin_inff() ? 0.0f : m;
    for (int t0 = 0; t0 < end && l != 0.0f && !nan; t0 += 64) {
        const bool visible = score(t0 + lane, at, z);
        const float p = visible ? __builtin_amdgcn_exp2f(z - base) / l : 0.0f;
        const unsigned long long all = __ballot(visible);
        for (int k0 = 0; k0 < 64; k0 += 8) {
            if (!(all >> k0 & 0xff)) continue;
            float u[8][V];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const size_t v = __shfl((unsigned long long)at, k0 + k);
#pragma unroll
                for (int i = 0; i < V; i++) u[k][i] = kv_load<TYPE>(c.v, v + lane * V + i);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float w = __shfl(p, k0 + k);
                const bool is = all >> (k0 + k) & 1;
#pragma unroll
                for (int i = 0; i < V; i++) o[i] = is ? __builtin_fmaf(w, u[k][i], o[i]) : o[i];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = o[i];
}

// Joins the parts of sequences that were cut, and takes up odd rows again.  Few
// rows and heads: a workgroup each, whose four waves take a quarter of the parts.
// Many (then each has few parts): a wave each.  A chunk behind 2000 keys, whole call,
// workgroup / wave each: 1024 rows and heads 25.5 / 26.1 us, 2048 31.5 / 29.7, 4096
// 47.7 / 42.7; but one row of 16 heads over 98304 keys 30 / 54.
constexpr int JOIN_WAVES = 4;
constexpr size_t JOIN_FEW = 1024;

// Parts i0, i0 + by, .. of a row: their largest m, and sums under it.  A lane holds
// the weight of one part, so that the parts' loads wait for nothing.
template <int D, int RG>
QG_DEV void join_parts(const AttnArgs &A, const Join &j, int in_group, int i0, int by, int lane, float &top, float &sum, float (&y)[D / 64]) {
    constexpr int V = D / 64;
    const float2 *ml = A.part_ml + (size_t)j.slot * RG + in_group;
    const float *po = A.part_o + ((size_t)j.slot * RG + in_group) * D + lane * V;
    top = -__builtin_inff();
    sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; v++) y[v] = 0.0f;
    for (; i0 < j.parts; i0 += 64 * by) {
        const int mine = i0 + lane * by, count = min((j.parts - i0 + by - 1) / by, 64);
        const float2 x = mine < j.parts ? ml[(size_t)mine * j.step * RG] : make_float2(-__builtin_inff(), 0.0f);
        const float next = fmaxf(top, qg_wave_max(x.x));
        const float old = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - next);
        const float f = part_weight(x.x, x.y, next);
        top = next;
        sum = sum * old + qg_sum_lanes<64>(f < 0.0f ? 0.0f : f * x.y);
#pragma unroll
        for (int v = 0; v < V; v++) y[v] *= old;
        for (int i = 0; i < count; i += 8) {
            float u[8][V];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float *from = po + (size_t)(i0 + min(i + k, count - 1) * by) * j.step * RG * D;
#pragma unroll
                for (int v = 0; v < V; v++) u[k][v] = from[v];
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float w = i + k < count ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), (i + k) & 63)) : -1.0f;
#pragma unroll
                for (int v = 0; v < V; v++) y[v] = w < 0.0f ? y[v] : __builtin_fmaf(w, u[k][v], y[v]);
            }
        }
    }
}
// Divides and stores a joined row; true if it is odd.
template <int D>
QG_DEV bool join_done(const AttnArgs &A, size_t at, int lane, float sum, const float (&y)[D / 64]) {
    bool odd = false;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int v = 0; v < D / 64; v++) {
        odd |= odd_sums(y[v], 0.0f, sum);
        A.out[at * D + lane * (D / 64) + v] = y[v] * inv;
    }
    return __any(odd);
}
template <int TYPE, int D, int RG, int EACH>
__global__ __launch_bounds__(64 * JOIN_WAVES) void attention_join_kernel(AttnArgs A, KvView c, BatchView b) {
    constexpr int V = D / 64;
    __shared__ float s_y[JOIN_WAVES][D];
    __shared__ float2 s_w[JOIN_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t at = EACH == 1 ? blockIdx.x : (size_t)blockIdx.x * EACH + wave;
    if (at >= (size_t)b.rows * A.q_heads) return;
    const int row = (int)(at / A.q_heads), head = (int)(at % A.q_heads);
    const int4 x = A.joins[at];
    const Join j{x.x, x.y, x.z, x.w};
    int first, n;
    const int s = batch_sequence(b, c.sequences, row, lane, first, n);
    if (s < 0) return;  // nothing was written for it
    bool odd = j.odd == 1;
    if (j.parts > 1) {
        if (!j.inside(A.slots)) return;
        const int in_group = ((row - first) * A.group + (head - by_group(A, head) * A.group)) % RG;
        float top, sum, y[V];
        if (EACH > 1) {
            join_parts<D, RG>(A, j, in_group, 0, 1, lane, top, sum, y);
        } else {
            join_parts<D, RG>(A, j, in_group, wave, JOIN_WAVES, lane, top, sum, y);
#pragma unroll
            for (int v = 0; v < V; v++) s_y[wave][lane * V + v] = y[v];
            if (lane == 0) s_w[wave] = make_float2(top, sum);
            __syncthreads();
            if (wave) return;
            const float most = fmaxf(fmaxf(s_w[0].x, s_w[1].x), fmaxf(s_w[2].x, s_w[3].x));
            sum = 0.0f;
#pragma unroll
            for (int v = 0; v < V; v++) y[v] = 0.0f;
#pragma unroll
            for (int w = 0; w < JOIN_WAVES; w++) {
                const float2 u = s_w[w];
                const float f = part_weight(u.x, u.y, most);
                if (f < 0.0f) continue;
                sum = __builtin_fmaf(f, u.y, sum);
#pragma unroll
                for (int v = 0; v < V; v++) y[v] = __builtin_fmaf(f, s_y[w][lane * V + v], y[v]);
            }
        }
        odd = join_done<D>(A, at, lane, sum, y);
    }
    if (odd && (EACH > 1 || wave == 0)) attend_row<TYPE, D>(A, c, b, s, first, n, row, head, lane, s_y[wave]);
}

// Row tiles per wave: as few row groups as the registers allow, and no more tiles than those need.
constexpr int most_tiles(int dim) { return dim == 256 ? 2 : dim == 128 ? 3 : 4; }
int row_tiles(int dim, long rows) {
    const long most = most_tiles(dim), groups = (rows + 16 * most - 1) / (16 * most);
    return (int)((rows + 16 * groups - 1) / (16 * groups));
}
constexpr int WAVES = 4;

template <int TYPE, int D, int RT>
void launch(const AttnArgs &A, const KvView &c, const BatchView &b, hipStream_t s) {
    const long groups = (long)b.rows * A.group / (16 * RT) + c.sequences;  // of all sequences: each rounds up
    const long units = 2 * A.resident + groups * c.heads + 8;
    attention_kernel<TYPE, D, RT, WAVES><<<(unsigned)((units + 127) / 128 * 128), 64 * WAVES, 0, s>>>(A, c, b);
    const size_t jobs = (size_t)b.rows * A.q_heads;
    if (jobs > JOIN_FEW) attention_join_kernel<TYPE, D, 16 * RT, 4><<<(unsigned)((jobs + 3) / 4), 256, 0, s>>>(A, c, b);
    else attention_join_kernel<TYPE, D, 16 * RT, 1><<<(unsigned)jobs, 256, 0, s>>>(A, c, b);
}
template <int TYPE, int D>
void launch_rt(int rt, const AttnArgs &A, const KvView &c, const BatchView &b, hipStream_t s) {
    if (rt == 1) launch<TYPE, D, 1>(A, c, b, s);
    else if (rt == 2) launch<TYPE, D, 2>(A, c, b, s);
    else if constexpr (D != 256) {
        if (rt == 3) launch<TYPE, D, 3>(A, c, b, s);
        else if constexpr (D == 64) launch<TYPE, D, 4>(A, c, b, s);
    }
}
template <int TYPE>
void launch_dim(int rt, const AttnArgs &A, const KvView &c, const BatchView &b, hipStream_t s) {
    if (c.dim == 64) launch_rt<TYPE, 64>(rt, A, c, b, s);
    else if (c.dim == 128) launch_rt<TYPE, 128>(rt, A, c, b, s);
    else launch_rt<TYPE, 256>(rt, A, c, b, s);
}

// Workgroups that run at once: a wave per SIMD each, so what the registers allow
// (in 64-dimension row tiles: 1 takes up to 110 registers, 2 up to 160, 6 up to 256).
int resident(int dim, int rt) {
    const int w = dim / 64 * rt;
    return qg_cu_count() * (w == 1 ? 4 : w == 2 ? 3 : w <= 6 ? 2 : 1);
}
// Partial results that the plan can ask for: a cut sequence has fewer parts than
// twice its keys / chunk, and the chunk is at least all sequences' keys x row
// groups x heads / two rounds.
size_t slots(int dim, int rt) { return 4 * (size_t)resident(dim, rt); }
// Rows of them: of the shape that needs the most, so that a workspace serves every
// batch of no more rows.
size_t part_rows(int dim) {
    size_t most = 0;
    for (int rt = 1; rt <= most_tiles(dim); rt++) most = most > slots(dim, rt) * 16 * rt ? most : slots(dim, rt) * 16 * rt;
    return most;
}
constexpr long JOBS = 1L << 25;  // rows x heads: of the join kernel, a wave each, within 2^32 threads
}  // namespace

extern "C" {

size_t qg_tree_attention_workspace_bytes(const qg_kv_cache *cache, const qg_kv_batch *batch, int q_heads) {
    if (qg_kv_check(cache, false, nullptr) || qg_batch_check(batch, false, nullptr)) return 0;
    if (q_heads < 1 || q_heads % cache->kv_heads || q_heads / cache->kv_heads > 128) return 0;
    if ((long)batch->rows * q_heads > JOBS) return 0;
    return part_rows(cache->head_dim) * (4 * (size_t)cache->head_dim + sizeof(float2)) + sizeof(int4) * (size_t)batch->rows * q_heads;
}

int qg_tree_attention(float *out, const float *q, int q_heads, float scale, const qg_kv_cache *cache, int layer,
                      const qg_kv_batch *batch, void *ws, size_t ws_bytes) {
    KvView c;
    BatchView b;
    const size_t need = qg_tree_attention_workspace_bytes(cache, batch, q_heads);
    if (!need || qg_kv_check(cache, false, &c) || qg_batch_check(batch, false, &b)) return hipErrorInvalidValue;
    if (!out || !q || !ws || ws_bytes < need || (((uintptr_t)out | (uintptr_t)q | (uintptr_t)ws) & 15)) return hipErrorInvalidValue;
    if (layer < 0 || layer >= c.layers || !__builtin_isfinite(scale * 1.44269504088896341f)) return hipErrorInvalidValue;
    const size_t bytes = 4 * (size_t)b.rows * q_heads * c.dim;
    if (qg_overlap(out, bytes, q, bytes) || qg_overlap(ws, need, q, bytes) || qg_overlap(ws, need, out, bytes)) return hipErrorInvalidValue;
    const int group = q_heads / c.heads, rt = row_tiles(c.dim, (long)b.max_rows * group);
    float *part_o = (float *)ws;
    const int run = !b.parent && b.max_rows > QG_MAX_TREE ? 16 : 0;
    const size_t parts = slots(c.dim, rt) * 16 * rt;
    float2 *part_ml = (float2 *)(part_o + parts * c.dim);
    const AttnArgs A{out, q, part_o, part_ml, (int4 *)(part_ml + parts), scale * 1.44269504088896341f, q_heads, group, layer, resident(c.dim, rt),
                     (int)slots(c.dim, rt), run,
                     (unsigned)(((1ULL << 32) + group - 1) / group)};
    if (c.type == QT_F32) launch_dim<QT_F32>(rt, A, c, b, qg_stream());
    else if (c.type == QT_F16) launch_dim<QT_F16>(rt, A, c, b, qg_stream());
    else launch_dim<QT_BF16>(rt, A, c, b, qg_stream());
    return hipGetLastError();
}

}  // extern "C"
