// Tiles of attention over the paged cache, shared by its kernels: keys and values
// in a wave's registers, their products with planes of queries and weights, the
// rules of partial results, and a row taken key by key.
#pragma once
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

struct AttnRows {
    float *out;
    const float *q;
    float scale;         // times log2 e
    int q_heads, group, layer;
    unsigned group_inv;  // 2^32 / group, rounded up
};
inline AttnRows attn_rows(float *out, const float *q, int q_heads, int group, int layer, float scale) {
    return AttnRows{out, q, scale * 1.44269504088896341f, q_heads, group, layer, (unsigned)(((1ULL << 32) + group - 1) / group)};
}

// x / group for x < 2^24: the product is over by less than x / 2^32 < 1 / group.
QG_DEV int by_group(const AttnRows &A, int x) { return A.group == 1 ? x : (int)__umulhi((unsigned)x, A.group_inv); }

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

// One row and head, key by key: a lane scores one of 64 keys at a time, the
// output's dimensions lie across the lanes.  The weights' sum first, so that the values
// are taken by weights that sum to 1: nothing overflows that the output holds.  A NaN in
// the query or in that sum is the row's.  A wave's latencies bound it: a sequence's rows
// over 98304 keys 18 ms with 16 bytes of a key and eight values on their way at once, 42
// with one; NaN queries cost nothing.
template <int TYPE, int D>
QG_DEV void attend_row(const AttnRows &A, const KvView &c, const BatchView &b, int s, int first, int n, int row, int head, int lane, float *s_q) {
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

// Row tiles per wave: as few row groups as the registers allow, and no more tiles than those need.
constexpr int most_tiles(int dim) { return dim == 256 ? 2 : dim == 128 ? 3 : 4; }
int row_tiles(int dim, long rows) {
    const long most = most_tiles(dim), groups = (rows + 16 * most - 1) / (16 * most);
    return (int)((rows + 16 * groups - 1) / (16 * groups));
}
constexpr int WAVES = 4;

// Workgroups that run at once: a wave per SIMD each, so what the registers allow
// (in 64-dimension row tiles: 1 takes up to 110 registers, 2 up to 160, 6 up to 256).
int resident(int dim, int rt) {
    const int w = dim / 64 * rt;
    return qg_cu_count() * (w == 1 ? 4 : w == 2 ? 3 : w <= 6 ? 2 : 1);
}
}  // namespace
