/* libqwen_gpu.so: MI355X (gfx950) implementation of the routed-MoE subset of
 * the reference's GPU C ABI.  Names, argument lists, return conventions and
 * semantics follow /root/reference/qwen/gpu.h, so the reference's ctypes
 * caller (test_gpu.py:12-36) and host engine (qwen.c) bind unchanged.
 *
 * Conventions (gpu.h:4-10, gpu.cu:38-46,181-189):
 *  - device arrays are token-major; the caller owns every device buffer;
 *  - int returns are runtime error codes (hipError_t here, cudaError_t in the
 *    reference), 0 = success, text from qg_error(); argument errors return
 *    the "invalid value" code;
 *  - operator wrappers are asynchronous on the calling thread's stream and
 *    return the launch status; qg_write/qg_read are synchronous;
 *  - between qg_graph_begin and qg_graph_end the calling thread's launches
 *    are captured (per-thread capture stream, gpu.cu:10,21-34).
 * Entry points whose reference signature carries no width (gather, scatter,
 * reduce, mtp_moe, shared_add) use the hidden/FFN widths set by
 * qg_moe_configure (default 2560/640, the reference's hard-coded shapes,
 * gpu.cu:508-553). */
#ifndef NEBULA_QWEN_GPU_H
#define NEBULA_QWEN_GPU_H
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

/* ---- runtime (gpu.h:11-21,24,30-36; gpu.cu:13-85,114-120) ---- */
void *qg_alloc(size_t bytes);                                   /* gpu.h:11, NULL on failure */
void qg_free(void *p);                                          /* gpu.h:12 */
int qg_write(void *dst, const void *src, size_t bytes);         /* gpu.h:13, synchronous H2D */
int qg_read(void *dst, const void *src, size_t bytes);          /* gpu.h:14, synchronous D2H */
int qg_copy(void *dst, const void *src, size_t bytes);          /* gpu.h:15, async D2D */
int qg_zero(void *dst, size_t bytes);                           /* gpu.h:16, async fill */
int qg_sync(void);                                              /* gpu.h:17 */
int qg_graph_begin(void **graph);                               /* gpu.h:18 */
int qg_graph_end(void *graph);                                  /* gpu.h:19 */
int qg_graph_launch(void *graph);                               /* gpu.h:20 */
void qg_graph_destroy(void *graph);                             /* gpu.h:21 */
int qg_graph_recording(void);   /* 1 between the calling thread's qg_graph_begin and qg_graph_end (an addition) */
int qg_memory(size_t *free_bytes, size_t *total_bytes);         /* gpu.h:24 */
const char *qg_error(int error);                                /* gpu.h:30 */
int qg_tensor_bytes(int type, const uint64_t dims[4], uint64_t *bytes); /* gpu.h:31 */
void *qg_upload_create(size_t expert_bytes);                    /* gpu.h:32 */
void qg_upload_destroy(void *uploader);                         /* gpu.h:33 */
int qg_upload_expert(void *uploader, void *dst, const void *gate, size_t gate_bytes,
                     const void *up, size_t up_bytes, const void *down, size_t down_bytes); /* gpu.h:34-35 */
double qg_upload_seconds(void *uploader);                       /* gpu.h:36 */

/* ---- operators on the MoE path (gpu.h:37-43,62-78) ---- */
/* out[t,r] = sum_c deq(W)[r,c] x[t,c]; types 0,1,30,2,6,7,8,12,13,14,20;
 * tokens 1..8192; the reference's fixed summation order (gpu.cu:154-189,
 * cpu.c:119-148), so results equal cpu.c's qc_matmul bit for bit. */
int qg_matmul(float *out, const void *w, int type, int rows, int cols, const float *x, int tokens); /* gpu.h:37-38 */
int qg_gather(float *out, const void *w, int type, int cols, int row);          /* gpu.h:39 */
int qg_norm(float *out, const float *x, const float *weight, int width,
            int groups, int tokens, int weight_groups, int l2, float eps);      /* gpu.h:40-41 */
int qg_unary(float *out, const float *x, int count, int op, float scale);      /* gpu.h:42 */
int qg_binary(float *out, const float *a, const float *b, int count, int op);  /* gpu.h:43 */
int qg_route(int *ids, float *weights, const float *logits, int tokens);        /* gpu.h:62 */
typedef struct {
    uint64_t token_layers, missing_selections, skipped_selections, avoided_token_handoffs;
    double skipped_mass;
} qg_prune_stats;                                                               /* gpu.h:63-66 */
int qg_prune_routes(int *ids, float *weights, const unsigned char *resident,
                    int tokens, double threshold, qg_prune_stats *stats);       /* gpu.h:67-68 */
int qg_moe_map(int *map, const int *ids, int tokens);                          /* gpu.h:69 */
int qg_moe_gather(float *out, const float *x, const int *token_map, int selected_tokens);   /* gpu.h:70 */
int qg_moe_scatter(float *slots, const float *expert, const float *weights, const int *ids,
                   const int *token_map, int expert_id, int selected_tokens);  /* gpu.h:71-72 */
int qg_moe_reduce(float *out, const float *slots, int tokens);                 /* gpu.h:73 */
int qg_mtp_moe(float *slots, float *mid, const float *x, const int *ids, const float *weights,
               const void *gate, int gate_type, const void *up, int up_type,
               const void *down, int down_type, int tokens);                    /* gpu.h:74-76 */
int qg_dequant(float *out, const void *packed, int type, int rows, int cols);  /* gpu.h:77 */
int qg_shared_add(float *out, const float *shared, const float *gate, int tokens); /* gpu.h:78 */

/* ---- additions (no reference counterpart; the reference hard-codes the
 * shapes and drives the layer from the host, qwen.c:633-735) ---- */

/* Hidden width D and expert FFN width F used by the width-less entry points
 * above: a process-wide setting (initially 2560/640), seen by every thread.
 * D multiple of 256, F multiple of 32, D <= 8192, F <= 4096. */
int qg_moe_configure(int width, int ff);
/* A per-thread override of that setting for the calling thread's width-less
 * calls (a thread driving a model of its own shape); (0, 0) removes it.
 * Added entry point, no counterpart in gpu.h. */
int qg_moe_configure_thread(int width, int ff);

/* Dispatch of routing ids into per-expert contiguous row lists (CSR), the
 * device-side histogram/prefix-sum/permutation replacing qg_moe_map's
 * [512, tokens] map and the host count loop of qwen.c:650-655.  offsets[513];
 * entries offsets[e]..offsets[e+1]-1 list (ascending token) the selections of
 * expert e: row_token = t, row_slot = t*10+k.  Ids in [-513,-2] (pruned) are
 * skipped; any other id outside [0,512), or a token listing an expert twice,
 * makes *status nonzero (the lists are then unspecified). */
int qg_moe_dispatch(int *offsets, int *row_token, int *row_slot, int *status, const int *ids, int tokens);

/* One routed-MoE layer, device-driven (no host read of routing ids), so it
 * can be captured into a graph: router -> top-10 -> [coverage/prune] ->
 * dispatch -> gate/up + SwiGLU -> down + router-rank combine -> shared expert.
 * Replaces moe()/grouped_moe()/shared_direct() of qwen.c:633-735 for one
 * layer.  Arithmetic: router logits in fp32 in the reference's fixed order
 * (ids and weights bit-exact); expert products on fp16 matrix cores with fp32
 * accumulation: each weight enters exactly (Q4_K as the integer s*q, at most
 * 945; IQ4_NL as its table value), each activation as two fp16 planes (hi =
 * fp16(x), lo = fp16(x - hi), about 22 significant bits), superblock and
 * block scales and the Q4_K min term applied in fp32 (the sums of 32 activations
 * that the min term multiplies are held like activations, as two fp16 values,
 * whose range is +-65504; in fp32 by the generic kernels and the batches of up
 * to 17 tokens at D = 1024); outputs agree with the reference's fp32 path
 * within max-abs 1e-3 / rel-L2 1e-4 (about 1e-6 relative in practice). */
typedef struct {
    int width, ff;                              /* D, F */
    const float *router;                        /* F32 [512, D] (ffn_gate_inp) */
    const void *gate, *up, *down;               /* [512][F][row(D)], [512][F][row(D)], [512][D][row(F)] */
    int gate_type, up_type, down_type;
    const void *sh_gate, *sh_up, *sh_down;      /* shared expert or NULL (ffn_*_shexp) */
    int sh_gate_type, sh_up_type, sh_down_type;
    const float *sh_gate_inp;                   /* F32 [1, D] (ffn_gate_inp_shexp) */
    const unsigned char *resident;              /* 512-byte device mask or NULL */
    double threshold;                           /* omitted-mass threshold (0.10, config.py:9) */
    const float *router_bias;                   /* F32 [512] added to every logit before routing, or NULL
                                                   (synthetic workloads; the reference's router has no bias) */
} qg_moe_layer;

/* Device workspace bytes for qg_moe_forward / qg_moe_forward_residual at up
 * to `tokens` tokens.  The workspace needs no initialisation; one workspace
 * per concurrent caller. */
size_t qg_moe_workspace_bytes(int width, int ff, int tokens);

/* out [tokens, D]; ids/weights [tokens, 10] (after pruning); flags [tokens]
 * or NULL: 0 all selections resident, 1 pruned (omitted mass < threshold),
 * 2 handoff (coverage below 1-threshold), 3 invalid router distribution;
 * stats may be NULL.  With flags==2 the token's routed part is not computed
 * here (it belongs to the host handoff, qwen.c:658-678): its row holds only
 * the sigmoid-gated shared expert (which stays on the device, qwen.c:661-663),
 * or 0 without one; qg_moe_handoff_pack/merge move the routed part through
 * the host.  flags==3 rows are 0.
 * Device pointers to weights, activations, outputs and the workspace must be
 * 16-byte aligned (qg_alloc returns 256-byte aligned memory); otherwise the
 * call returns an invalid-value error and launches nothing.
 * tokens 1..8192: up to 17 any format qg_matmul takes (the decode kernels, at
 * D = 1024 the prefill's, or the generic ones; qg_moe_kernel_events lists which);
 * above, the prefill grouped GEMMs, which need Q4_K gate/up, Q4_K or IQ4_NL
 * down, D a multiple of 256 and F a multiple of 128 (else an error).  The order
 * of the fp32 sums, and so an output's last bits, may differ between shapes and
 * batch sizes. */
int qg_moe_forward(float *out, int *ids, float *weights, unsigned char *flags, qg_prune_stats *stats,
                   const float *x, int tokens, const qg_moe_layer *layer, void *workspace, size_t workspace_bytes);

/* No reference counterpart: for callers that cannot allocate device memory
 * (code under graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  qg_moe_forward with the library's own workspace, a static
 * 16 MiB array in device memory per GPU (held until the process ends); no
 * allocation of any kind happens.  Layers whose qg_moe_workspace_bytes at
 * `tokens` exceeds 16 MiB are rejected with the invalid-value code before
 * anything is launched (every decode batch of 1..17 tokens fits up to
 * D=8192/F=4096; at D=2048/F=512 prefill batches up to about 120 tokens
 * fit).  Calls that overlap on one GPU share the workspace and race. */
int qg_moe_forward_noalloc(float *out, int *ids, float *weights, unsigned char *flags, qg_prune_stats *stats,
                           const float *x, int tokens, const qg_moe_layer *layer);

/* The layer applied to a residual stream, as one layer of qwen_target's loop
 * without attention (qwen.c:759-762): x = RMSNorm(h) (eps 1e-6, unit weight,
 * the norm of gpu.cu:204-214), h += MoE(x).  xn_out [tokens, D] (the
 * normalised input) and out [tokens, D] (the MoE output) may be NULL.  Other
 * arguments as qg_moe_forward. */
int qg_moe_forward_residual(float *h, int *ids, float *weights, unsigned char *flags, qg_prune_stats *stats,
                            float *xn_out, float *out, int tokens, const qg_moe_layer *layer,
                            void *workspace, size_t workspace_bytes);

/* ---- a speculative step over a paged cache: per-head norms and rotation,
 * attention, softmax, draft verification, page management.  Additions beside
 * qg_norm, qg_matmul and qg_moe_forward: with them the rows of one target
 * batch (qwen.c:748-768: the last accepted token and its drafts) pass through
 * a layer's attention and the drafts are accepted on the device, so a whole
 * step can be captured into a graph.
 *
 * Conventions.  Device pointers of the current device; int arrays are read on
 * the device at launch order, so one captured graph serves every step.  What
 * the host can see is checked before anything is launched (invalid-value
 * code); what only the device can see is bounded there: a page entry outside
 * [0, pages) holds nothing, a length is taken as 0..table_pages * page_tokens,
 * the rows of a sequence as at most max_rows inside [0, rows), and a parent
 * that is not an earlier row of its sequence as none.  Nothing outside the
 * given buffers is read or written.  A workspace belongs to one call until that
 * has run: calls of one stream may share it, others (and graphs that may run at
 * once) may not. */

/* Keys and values of `sequences` sequences in pages of page_tokens tokens.
 * Position t of sequence s lies in page table[s][t / page_tokens] at token
 * t % page_tokens.  A page may be held by several sequences (qg_kv_fork). */
typedef struct {
    void *k, *v;                /* [layers][pages][kv_heads][page_tokens][head_dim], 16-byte aligned */
    int type;                   /* 0 F32, 1 F16, 30 BF16 */
    int layers, pages, kv_heads; /* layers 1..65536, pages 1..2^30, kv_heads 1..128 */
    int page_tokens;            /* a power of two, 8..1024 */
    int head_dim;               /* 64, 128 or 256 */
    int *refs;                  /* [pages] table entries that hold each page, 0 = free; NULL without page calls */
    int *table;                 /* [sequences][table_pages] page or -1 */
    int *length;                /* [sequences] tokens held */
    int sequences, table_pages; /* 1..1024 sequences; table_pages * page_tokens <= 2^28 */
} qg_kv_cache;

/* The rows of one batch: sequence s of the cache has rows start[s] ..
 * start[s+1]-1 of the activations (none is allowed), row i of them takes the
 * cache position length[s] + i.  parent NULL: each row follows the one before
 * it (a chain, a prompt chunk).  Else parent[r] is the place in its sequence
 * of the row that row r continues, -1 for none, and max_rows is at most 64. */
typedef struct {
    int rows, max_rows;         /* rows 1..65536; rows of one sequence at most max_rows */
    const int *start;           /* [sequences + 1], ascending */
    const int *parent;          /* [rows] or NULL */
} qg_kv_batch;

/* Query, key and value rows as a projection wrote them: head h of row t of q
 * starts at q + t * q_row + h * q_head (floats); k and v likewise.  Pointers
 * 16-byte aligned, strides multiples of 4. */
typedef struct {
    const float *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    int rows, q_heads, kv_heads, head_dim; /* head_dim 64, 128 or 256; heads 1..1024 */
    const float *q_norm, *k_norm; /* [head_dim] RMS-norm weights, or NULL: that side is not normalised */
    float eps;
    int rope_dims;              /* leading dimensions rotated: a multiple of 8, 0..head_dim */
    int interleaved;            /* pairs (2i, 2i+1); 0: (i, i + rope_dims/2) */
    const double *freq;         /* [rope_dims/2] radians per position (theta^(-2i/rope_dims), or a scaled form) */
    const int *position;        /* [rows], or NULL: length[s] + the row's depth below its root in the batch */
} qg_qk_rows;

/* Per-head RMS norm (as qg_norm) and rotation of q and k, in one pass; q_out
 * [rows][q_heads][head_dim], k_out [rows][kv_heads][head_dim] fp32 (k_out may
 * be NULL).  With a cache, k (normed, rotated) and v are rounded to its type
 * and stored at their positions of `layer`; a row whose position has no page,
 * or one that another table entry holds too (where the cache has refs; see
 * qg_kv_reserve), is not stored.  Without a cache, batch is NULL, v is ignored and
 * position is needed where rope_dims > 0.  Angles are formed in 64 bits.  An output may be its own
 * input where both have the same layout; otherwise they must not overlap.
 * Rows of no sequence are left as they were. */
int qg_qk_norm_rope(float *q_out, float *k_out, const qg_qk_rows *in, const qg_kv_cache *cache, int layer,
                    const qg_kv_batch *batch);

/* Attention of the batch's rows over the cache: row i of sequence s sees the
 * length[s] cached tokens, itself and the rows it descends from (all stored
 * before the call).  out, q [rows][q_heads][head_dim] fp32, q_heads a multiple
 * of kv_heads up to 128 times as many, both 16-byte aligned; no overlap.
 * Scores, statistics and sums are held in fp32; the products run on the matrix
 * cores with queries and probabilities in planes of the cache's type that
 * together carry at least 22 bits, over an F16 cache down to 2^-38 of a row's
 * largest probability or query value.  A row that sees no token (or none with a
 * score above -infinity) is 0, one with a NaN or a score of +infinity is NaN.
 * Rows that see infinities, or values whose sum passes fp32's range, are computed
 * key by key, which is slow (18 ms over 98304 tokens).  Rows of no sequence are
 * left as they were.
 * rows x q_heads at most 2^25.  The workspace of a batch serves every batch of
 * no more rows. */
size_t qg_tree_attention_workspace_bytes(const qg_kv_cache *cache, const qg_kv_batch *batch, int q_heads);
int qg_tree_attention(float *out, const float *q, int q_heads, float scale, const qg_kv_cache *cache, int layer,
                      const qg_kv_batch *batch, void *workspace, size_t workspace_bytes);

/* Sequences that begin with the same pages (qg_kv_fork), as the attention below
 * takes them: shared[s] = the most leading tokens, in whole pages, that a
 * sequence s with rows in the batch has in common with an earlier one that has
 * rows, link[s] the first such (-1 and 0: none, or s has no rows).  A page
 * counts where both tables hold the same one and both sequences' cached tokens
 * fill it.  link, shared [sequences], or NULL.  `prefixes` (16-byte aligned) is
 * filled for the attention of every layer, up to the next change of the cache's
 * tables or lengths or of the batch's rows; after one it must not be used (nothing
 * outside the buffers is then touched, but outputs may be anything).  Outputs
 * overlap neither each other nor table, length and start. */
size_t qg_kv_prefixes_bytes(const qg_kv_cache *cache, const qg_kv_batch *batch);
int qg_kv_prefixes(int *link, int *shared, const qg_kv_cache *cache, const qg_kv_batch *batch, void *prefixes, size_t prefixes_bytes);

/* How many bytes of keys and values the sequences of a batch must save in each
 * layer for qg_kv_prefixes to have them shared (sharing costs 2 to 10 us a layer
 * whatever is saved; prompt chunks, sequences of more than 64 rows, gain nothing and
 * do not count): a setting of the calling thread, 48 MiB at first and for negative
 * values; 0 shares whatever there is.  link and shared do not depend on it, outputs
 * only within the attention's error.  A captured qg_kv_prefixes keeps the setting of
 * its capture.  Returns the previous setting. */
int64_t qg_prefix_least_saving(int64_t bytes);

/* qg_tree_attention of a batch in which sequences share pages: the same outputs
 * (within the same error), but a page that several sequences hold is read once
 * for all of them.  `prefixes` as qg_kv_prefixes filled it for this cache and batch;
 * other arguments, refusals and special values as there.  For few rows a sequence
 * over a long common text.  Where nothing is shared it takes longer: 1 to 4 us for up to
 * 8 sequences of one row and few heads, up to half as long again for many rows and wide
 * heads.  Finding what is shared takes 5 to 30 us, once for all layers, and about 1 us
 * for each sequence of a line where every one branches from the one before it.
 * The workspace serves every batch of no more rows over a cache of no more
 * sequences and the same heads and head_dim. */
size_t qg_prefix_attention_workspace_bytes(const qg_kv_cache *cache, const qg_kv_batch *batch, int q_heads);
int qg_prefix_attention(float *out, const float *q, int q_heads, float scale, const qg_kv_cache *cache, int layer,
                        const qg_kv_batch *batch, const void *prefixes, size_t prefixes_bytes, void *workspace,
                        size_t workspace_bytes);

/* out = softmax(x / temperature) of each row of [rows][cols]; out may be x.
 * temperature 0: 1 at the lowest index of the largest value; others from 2^-126
 * on.  -infinity gives 0; a row of nothing but -infinity is 0; a row with NaN or
 * +infinity is NaN.
 * rows 1..65536, cols 1..2^24, at most 2^35 values; 4-byte aligned.  The
 * workspace of a number of rows serves fewer of them too. */
size_t qg_softmax_workspace_bytes(int rows, int cols);
int qg_softmax(float *out, const float *x, int rows, int cols, float temperature, void *workspace, size_t workspace_bytes);

/* Verification of drafts by rejection sampling; the accepted tokens are
 * distributed as the target's.  Row 0 of a sequence is its last accepted
 * token, each further row a draft, token[r], of the row it continues
 * (qg_kv_batch; max_rows <= 64).  p [rows][cols]: the target's probabilities
 * after each row.  q [rows][cols]: the probabilities that a row's drafts were
 * drawn from (independently), or NULL: each draft was chosen, not drawn.
 * From row 0 the drafts of the current row are tried in order: with a = 0 and
 * B = 1, draft x is accepted if u[r] q(x) B < p(x) - a q(x) and becomes the
 * current row, else a += B, B = sum_i max(p_i - a q_i, 0).  (With q NULL:
 * if u[r] B < p(x), else B -= p(x) and p(x) counts as 0.)  At a row
 * without an accepted draft the last token is the first i with
 * sum_{j<=i} w_j > u_last[s] sum_j w_j, w = max(p - a q, 0), or p where that
 * sum is not positive; -1 where p has none either.  Products and sums in 64 bits.
 * u, u_last in [0, 1).  Outputs: count[s] = accepted rows with row 0 (0 for a
 * sequence without rows); path[s][0..count-1] their places; tokens_out[s]
 * [0..count-1] the accepted tokens and the last one; -1 behind them
 * ([sequences][max_rows] both).  The outputs overlap neither each other nor p, q,
 * u_last and start, the workspace nothing.  A token outside [0, cols) is never
 * accepted.  The workspace of a number of sequences serves fewer of them too. */
size_t qg_verify_workspace_bytes(int sequences, int cols);
int qg_verify_drafts(int *tokens_out, int *path, int *count, const float *p, const float *q, const int *token,
                     const float *u, const float *u_last, int cols, int sequences, const qg_kv_batch *batch,
                     void *workspace, size_t workspace_bytes);

/* Truncated distributions.  What each row's request asks for: device arrays
 * [rows], or NULL for all rows without.  Of the weights w_i = exp((x_i - max) /
 * temperature) stay: with top_k > 0 the top_k largest values; of these, with
 * top_p < 1, in falling order those before which less than top_p of their sum
 * lies; of these, with min_p > 0, those of at least min_p times the largest.  Of
 * equal values the lower index counts as larger (0 and -0 are equal); the
 * largest always stays.  temperature 0, and one that is not at least 2^-126,
 * is the first largest token alone; top_k <= 0 or >= cols, a top_p that is not
 * below 1 and a min_p that is not above 0 keep all.  Weights below 2^-1000
 * count as 0. */
typedef struct {
    const float *temperature;   /* NULL: 1 */
    const int *top_k;
    const float *top_p, *min_p;
} qg_sampling;

/* token[rows][draws]: the first i with sum_{j<=i} w_j > u[r][d] sum_j w_j over
 * what stays of row r of x [rows][cols], u [rows][draws] in [0, 1);
 * logprob[rows][draws] (or NULL): log(w_i / sum_j w_j).  Weights and sums in 64
 * bits; the sums that draws and top-p are held against to 2^-35 of themselves (2^-37
 * where |x / T| is at most 2^14), or to 2^(2 b - 63), 2^b >= cols, those of top-p in a
 * row that is searched as a whole (over 1024 values within a 64th of a bit of weight
 * where a filter cuts, cuts further than 2^-62 below the largest weight, |x / T| past
 * 2^17).  -infinity is never drawn; a row of nothing else, or with NaN or
 * +infinity, gives -1 and NaN.  draws 1..64 of each row, independent of each
 * other (drafted siblings, several answers' first tokens).
 * qg_sampling_softmax: out = w_i / sum_j w_j, 0 where a token does not stay,
 * what the draws of qg_sample are distributed as: p and q of qg_verify_drafts.
 * out may be x; a row of nothing but -infinity is 0, one with NaN or +infinity
 * NaN.  Both: rows 1..65536, cols 1..2^24, at most 2^35 values, 4-byte aligned;
 * no output or workspace overlaps what else is given.  The workspace of a number
 * of rows serves fewer of them too. */
size_t qg_sample_workspace_bytes(int rows, int cols);
int qg_sample(int *token, float *logprob, const float *x, int rows, int cols, int draws, const qg_sampling *sampling,
              const float *u, void *workspace, size_t workspace_bytes);
int qg_sampling_softmax(float *out, const float *x, int rows, int cols, const qg_sampling *sampling, void *workspace,
                        size_t workspace_bytes);

/* Pages.  Calls that change tables take one stream at a time; each result is
 * the same on every run.  The arrays given overlap neither each other nor the
 * cache's where one of them is written, but for lengths as said.
 * qg_kv_workspace_bytes serves fork (of up to `sequences` pairs) and reserve. */
size_t qg_kv_workspace_bytes(const qg_kv_cache *cache);
/* Room for the batch's rows behind each sequence's tokens: pages are taken in
 * ascending order, for the sequences in order.  A held page that would be
 * written and that another sequence holds too is replaced, its tokens copied
 * (every layer); of several sequences of the batch that share a page no other holds, the
 * first keeps it.  status[s]: 0; 1 there are not enough free pages for the batch
 * (nothing is taken for any of its sequences); 2 the sequence's table is too
 * short (nothing is taken for it, the others are served).  The rest of a captured
 * step may run on where status[s] is not 0: rows of such a sequence are stored in
 * pages of its own only, so that no other sequence's tokens change; its length
 * grows by the k accepted rows that found one (qg_kv_compact), and of its tokens_out
 * the first k hold (0: none), since they follow rows that were stored. */
int qg_kv_reserve(const qg_kv_cache *cache, const qg_kv_batch *batch, int *status, void *workspace, size_t workspace_bytes);
/* For each pair i < n: sequence dst[i] lets go of its pages and shares those
 * of src[i]'s tokens; its length is src[i]'s.  Sources are read as before the
 * call; of several pairs with one dst the last counts; a pair with dst == src
 * or an index out of range is left out.  n 1..sequences. */
int qg_kv_fork(const qg_kv_cache *cache, const int *dst, const int *src, int n, void *workspace, size_t workspace_bytes);
/* length[s] = min(length[s], new_length[s]) (new_length NULL: as it is), and
 * the pages behind it are let go; 0 frees a sequence.  new_length may be the
 * cache's length. */
int qg_kv_truncate(const qg_kv_cache *cache, const int *new_length);
/* The accepted rows (qg_verify_drafts' path and count) move to the front: the
 * token at length[s] + path[s][i] goes to length[s] + i, in every layer, and
 * new_length[s] = length[s] + count[s], or the rows followed if fewer (new_length
 * may be the cache's length).
 * max_rows is at most 64, for chains too: a longer prompt chunk, all of whose
 * rows stay where they are, is taken by adding its rows to `length`.
 * A path is followed while it ascends inside its sequence's rows, and up to the
 * first row whose page, or the page that it would move to, another table entry
 * holds too (where the cache has refs); rows behind the last one with both pages
 * are left out, so that a length does not grow over rows that found no room. */
int qg_kv_compact(const qg_kv_cache *cache, const qg_kv_batch *batch, const int *path, const int *count, int *new_length);
/* Pages dst[i] = copies of pages src[i] in every layer, i < n <= 4096.  A
 * pair whose destination is among the sources or comes again later is left
 * out, as is one with an index out of range. */
int qg_kv_copy_pages(const qg_kv_cache *cache, const int *dst, const int *src, int n);

/* CPU handoff of the flag-2 tokens (replaces the whole-batch reads of
 * qwen.c:665-666 and the write of qwen.c:672).  Device arrays; async on the
 * calling thread's stream.  pack: count[0] = number of tokens with
 * flags[t] == 2, rows[i] = the i-th of them (ascending), and row i of x_pack
 * [tokens, width], ids_pack / w_pack [tokens, 10] = that token's input row,
 * ids and weights (only the first count[0] rows are written).  merge:
 * out[rows[i]] += y_pack[i] for i < count[0], y_pack [tokens, width] being
 * the host's routed rows (qc_moe, cpu.c:235-261, of the packed tokens).
 * tokens 1..8192. */
int qg_moe_handoff_pack(int *count, int *rows, float *x_pack, int *ids_pack, float *w_pack,
                        const unsigned char *flags, const float *x, const int *ids, const float *weights,
                        int tokens, int width);
int qg_moe_handoff_merge(float *out, const float *y_pack, const int *count, const int *rows, int tokens, int width);
/* After qg_moe_handoff_pack: count[0] is stored into *host_word, a word of
 * qg_host_alloc memory, by a kernel on the calling thread's stream, so the
 * host learns the number of handed-off tokens by polling the word instead of
 * a device-to-host copy.  Added entry point, no counterpart in gpu.h. */
int qg_moe_handoff_notify(int *host_word, const int *count);
/* Page-locked host memory that device code may access through the same
 * pointer (NULL on failure), and its release.  Added entry points (the
 * reference allocates its pinned staging inside qg_upload_create). */
void *qg_host_alloc(size_t bytes);
void qg_host_free(void *p);

/* Benchmark support: events[2i] and events[2i+1] (qg_event_create handles)
 * are recorded at the start and end of kernel i of this thread's
 * qg_moe_forward calls, timestamped by the dispatch itself
 * (hipExtLaunchKernelGGL).  Decode kernels (up to 17 tokens, D of 2048 or 2560,
 * F of 512 or 640, Q4_K gate/up, Q4_K or IQ4_NL down): 0 router, 1 routing, 2
 * gate/up, 3 down, 4 combine.
 * Prefill kernels (above 17 tokens; also up to 17 at D = 1024, F of 256, 512 or
 * 640, in those formats with one down format): 0 router, 1 routing, 2 scan, 3 fill, 4 gate/up dense pass,
 * 5 gate/up other experts, 6 down dense pass, 7 down other experts,
 * 8 shared-expert down (when its format differs), 9 combine, 10 chunk
 * histogram (up to 256 tokens 2 covers 3 and 10 too).  At D = 2560 (129..640
 * tokens) and D = 1024 (385..896) gate/up is launched in two forms, 4 for long
 * and 5 for short expert lists, of which one returns at once.  n <= 32;
 * n = 0 disables. */
int qg_moe_kernel_events(void **events, int n);

/* Benchmark support: record events[i] (qg_event_create handles) on the
 * launch stream at the phase boundaries of this thread's qg_moe_forward
 * calls of up to 17 tokens that the decode kernels (see qg_moe_kernel_events)
 * do not serve: 0 start, 1 after the router, 2 after routing/dispatch, 3 after
 * gate/up, 4 after down, 5 after the combine.  The decode kernels and batches
 * above 17 tokens record none.  n = 0 disables. */
int qg_moe_phase_events(void **events, int n);

/* Timing helpers for the benchmark (events on the calling thread's stream). */
void *qg_event_create(void);
void qg_event_destroy(void *event);
int qg_event_record(void *event);
int qg_event_elapsed(float *ms, void *begin, void *end);
int qg_device_info(char *name, size_t name_len, int *cus, int *clock_khz, int *mem_clock_khz, int *bus_bits);

/* Synthetic inputs generated on the device (benchmark/test support; not a
 * reference interface).  Value (r,c) of tensor `stream` under `seed` is
 * sigma*N(0,1) from a counter-based hash; encoded to type 0/12/20.  The
 * bytes equal the CPU generator's in oracle/nb_synth.c. */
int qg_synth_matrix(void *out, int type, uint64_t seed, uint64_t stream, int rows, int cols, float sigma);
/* `experts` such matrices in one launch: matrix e uses stream
 * (tensor << 32 | e) and starts e * rows * row_bytes(type, cols) bytes after
 * out, the per-tensor expert layout of a layer. */
int qg_synth_experts(void *out, int type, uint64_t seed, int tensor, int experts, int rows, int cols, float sigma);

/* No reference counterpart: how the calling thread's prefill layers launch
 * gate/up.  mode 0 (the default): one launch over every expert group.
 * mode 1: the dense experts (256 or more rows) in a launch of their own on
 * int8 matrix cores (two int8 activation planes per token row with a row
 * scale, the Q4_K nibbles as int8, per-group int32 -> fp32 scaling), then the
 * rest on fp16.  mode 2: the same split with both launches on fp16 hi/lo
 * planes.  Other values select mode 0.  Returns the previous mode.  A
 * measurement switch for the benchmark's int8-vs-fp16 comparison of the dense
 * experts and its parity test. */
int qg_prefill_int8_dense(int mode);

#ifdef __cplusplus
}
#endif
#endif
