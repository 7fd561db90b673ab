// Attention of a batch's rows over the paged cache (qg_tree_attention of
// include/qwen_gpu.h).
#include "qg_kv.h"

namespace {

// One wave per row and head: a lane scores one key of 64 at a time; the output's
// dimensions lie across the lanes.
template <int TYPE, int D>
__global__ __launch_bounds__(64) void attention_row_kernel(float *out, const float *q, int q_heads, float scale, KvView c, int layer, BatchView b) {
    __shared__ float s_q[D];
    const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, kv = head / (q_heads / c.heads);
    int first, n;
    const int s = batch_sequence(b, c.sequences, row, lane, first, n);
    if (s < 0) return;
    const int place = row - first, len = kv_length(c, s);
    const unsigned long long seen = b.parent ? __shfl(tree_ancestors(b.parent + first, n, lane), place) : 0;
    const float *qr = q + ((size_t)row * q_heads + head) * D;
    for (int d = lane; d < D; d += 64) s_q[d] = qr[d] * scale;
    __syncthreads();
    float m = -__builtin_inff(), l = 0.0f, o[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; i++) o[i] = 0.0f;
    const int end = len + (b.parent ? n : place + 1);
    for (int t0 = 0; t0 < end; t0 += 64) {
        const int t = t0 + lane, page = t < end ? kv_page(c, s, t) : -1;
        const bool visible = page >= 0 && (t < len || !b.parent || (seen >> (t - len) & 1));
        float sc = -__builtin_inff();
        const size_t at = kv_at(c, layer, max(page, 0), kv, t & ((1 << c.shift) - 1));
        if (visible) {
            sc = 0.0f;
            for (int d = 0; d < D; d++) sc = __builtin_fmaf(s_q[d], kv_load<TYPE>(c.k, at + d), sc);
        }
        float top = m;
        for (int i = 0; i < 64; i++) { const float x = __shfl(sc, i); top = x != x || x > top ? x : top; }
        if (top == -__builtin_inff()) continue;
        const float a = expf(m - top), pr = visible ? expf(sc - top) : 0.0f;
        m = top;
        l = l * a + qg_sum_lanes<64>(pr);
#pragma unroll
        for (int i = 0; i < D / 64; i++) o[i] *= a;
        for (unsigned long long left = __ballot(visible); left; left &= left - 1) {
            const int k = __builtin_ctzll(left);
            const float w = __shfl(pr, k);
            const size_t vat = __shfl((unsigned long long)at, k);
#pragma unroll
            for (int i = 0; i < D / 64; i++) o[i] = __builtin_fmaf(w, kv_load<TYPE>(c.v, vat + lane + 64 * i), o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < D / 64; i++) out[((size_t)row * q_heads + head) * D + lane + 64 * i] = l == 0.0f ? 0.0f : o[i] / l;
}

template <int TYPE>
void launch_rows(float *out, const float *q, int q_heads, float scale, const KvView &c, int layer, const BatchView &b, hipStream_t s) {
    const dim3 grid(b.rows, q_heads);
    if (c.dim == 64) attention_row_kernel<TYPE, 64><<<grid, 64, 0, s>>>(out, q, q_heads, scale, c, layer, b);
    else if (c.dim == 128) attention_row_kernel<TYPE, 128><<<grid, 64, 0, s>>>(out, q, q_heads, scale, c, layer, b);
    else attention_row_kernel<TYPE, 256><<<grid, 64, 0, s>>>(out, q, q_heads, scale, c, layer, b);
}
}  // namespace

extern "C" {

size_t qg_tree_attention_workspace_bytes(const qg_kv_cache *cache, const qg_kv_batch *batch, int q_heads) {
    if (qg_kv_check(cache, false, nullptr) || qg_batch_check(batch, false, nullptr)) return 0;
    if (q_heads < 1 || q_heads % cache->kv_heads || q_heads / cache->kv_heads > 128) return 0;
    return 16;
}

int qg_tree_attention(float *out, const float *q, int q_heads, float scale, const qg_kv_cache *cache, int layer,
                      const qg_kv_batch *batch, void *ws, size_t ws_bytes) {
    KvView c;
    BatchView b;
    const size_t need = qg_tree_attention_workspace_bytes(cache, batch, q_heads);
    if (!need || qg_kv_check(cache, false, &c) || qg_batch_check(batch, false, &b)) return hipErrorInvalidValue;
    if (!out || !q || !ws || ws_bytes < need || (((uintptr_t)out | (uintptr_t)q | (uintptr_t)ws) & 15)) return hipErrorInvalidValue;
    if (layer < 0 || layer >= c.layers || !__builtin_isfinite(scale)) return hipErrorInvalidValue;
    const size_t bytes = 4 * (size_t)b.rows * q_heads * c.dim;
    if (qg_overlap(out, bytes, q, bytes) || qg_overlap(ws, need, q, bytes) || qg_overlap(ws, need, out, bytes)) return hipErrorInvalidValue;
    if (c.type == QT_F32) launch_rows<QT_F32>(out, q, q_heads, scale, c, layer, b, qg_stream());
    else if (c.type == QT_F16) launch_rows<QT_F16>(out, q, q_heads, scale, c, layer, b, qg_stream());
    else launch_rows<QT_BF16>(out, q, q_heads, scale, c, layer, b, qg_stream());
    return hipGetLastError();
}

}  // extern "C"
