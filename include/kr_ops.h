/*
 * KernRelay-MI355X op-level C ABI (exported by libkernrelay.so).
 *
 * These are the hand-written HIP kernels behind the runtimes, callable on
 * caller-owned device memory. Each replaces one closed CANN aclnn call site
 * of the reference (cited per function). All calls are asynchronous on
 * `stream` (a hipStream_t, NULL = default stream), return 0 on success and a
 * non-zero code on invalid arguments or launch failure; kr_ops_last_error()
 * then describes the failure (thread-local, valid until the next call).
 *
 * Tensors are row-major; 16-bit element types are passed as raw bits.
 * Pointers to 16-bit tensors must be 16-byte aligned and row lengths
 * multiples of 8 elements (the kernels move 16-byte vectors).
 */
#ifndef KR_OPS_H
#define KR_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum { KR_BF16 = 0, KR_F16 = 1, KR_F32 = 2 };

/* Elementwise ops for kr_op_elementwise. */
enum {
    KR_EW_GELU = 0,
    KR_EW_SILU = 1,
    KR_EW_CAST = 2,
    KR_EW_MUL = 3,
    KR_EW_ADD = 4,
    KR_EW_SWIGLU = 5,     /* y = bf16(silu(x0)) * x1 */
    KR_EW_SWIGLU_GU = 6   /* x0 = fused [rows, 2*cols] gate/up in 8-column groups */
};

/* Row-reduction ops for kr_op_rowop. */
enum {
    KR_ROW_SOFTMAX = 0,
    KR_ROW_RMSNORM = 1,
    KR_ROW_ADD_RMSNORM = 2,
    KR_ROW_LAYERNORM = 3  /* gamma = weight [cols], x1 = bias [cols] (aclnnLayerNorm,
                             reference exec/runtime/op_impl.cpp:237-254) */
};

/* Relay control blocks: 8 x int32 each, zero-initialised once by the owner
 * (layout: published, consumed, status, arrive, done, timed_out, left, -; the
 * first three words are the reference's kernels/kr_sync_common.h:10-15). */
#define KR_CTRL_WORDS 8

/* Consumer side: wait for the producer tiles that cover the rows a launch
 * reads. Local row r is producer row r + row_off; producer tile k covers
 * rows [k*prod_rows, (k+1)*prod_rows), its flag is block flag0 + k and the
 * consumer's state for it is block state0 + k; state blocks adv_lo..adv_hi-1
 * are consumed by this launch. ctrl == NULL disables waiting.
 * Replaces reference kernels/kr_wait_aiv.cpp:7-36 (kr_wait_aiv/aic). */
typedef struct kr_wait {
    int32_t *ctrl;
    int32_t flag0;
    int32_t state0;
    int32_t prod_rows;
    int32_t row_off;
    int32_t adv_lo;
    int32_t adv_hi;
    uint32_t max_spins; /* 0 = default bound */
} kr_wait;

/* Producer side: tile t (rows [t*rows_per_tile, (t+1)*rows_per_tile) of the
 * launch) releases flag block flag0 + t when its last workgroup finishes.
 * `arrivals` is filled in by the library. ctrl == NULL disables publishing.
 * Replaces reference kernels/kr_publish_aiv.cpp:6-23 (kr_publish_aiv/aic). */
typedef struct kr_pub {
    int32_t *ctrl;
    int32_t flag0;
    int32_t rows_per_tile;
    int32_t arrivals;
} kr_pub;

const char *kr_ops_last_error(void);

/* C[M,N] = A[M,K] . Bt[N,K]^T (+ bias[N], rounded as matmul-then-add);
 * bf16/f16 in and out, fp32 accumulate. bm = M tile (0 = automatic; 64,
 * 128 or 256). pub may be NULL. wait may be NULL; else every workgroup waits
 * for the producer tiles covering its rows of A before loading them (the
 * GEMM as a relay consumer), and the launch consumes wait->adv_lo..adv_hi.
 * Replaces aclnnMatmul (reference exec/qwen_main.cpp:499-512,
 * exec/runtime/op_impl.cpp:175-201) and the fused QKV bias Add (:1336-1344);
 * the wait replaces a kr_wait_aic launch ahead of it (qwen_main.cpp:672-688). */
int kr_op_gemm(int dtype, const void *A, int64_t lda, const void *Bt, int64_t ldb, void *C,
               int64_t ldc, const void *bias, int M, int N, int K, int bm, const kr_wait *wait,
               const kr_pub *pub, void *stream);

/* Gate/up GEMM with its SwiGLU consumer in the same launch: C[M, 2*cols] =
 * A[M,K] . Bt[2*cols,K]^T (gate/up interleaved in groups of 8 columns) is
 * released in row tiles through pub (required; rows_per_tile divides M), and
 * workgroups appended after the GEMM's own wait for each released tile and
 * write act[M, cols] = SwiGLU over its rows (silu rounded to 16 bits before
 * the multiply, as kr_op_elementwise's swiglu_gu). Appended workgroups are
 * dispatched after every GEMM workgroup, so they only take CUs the GEMM's
 * last round leaves idle. tail_tiles (0 = all) limits the appended consumer
 * to the first relay tiles (the caller runs SwiGLU on the rest); order_rows
 * (0 = the relay tile) sets the row runs in which the GEMM produces. Replaces the relay edge matmul_gate/up ->
 * Silu -> Mul of the reference (exec/qwen_main.cpp:616-644, 888-889). */
int kr_op_gemm_swiglu(int dtype, const void *A, int64_t lda, const void *Bt, int64_t ldb, void *C,
                      void *act, int M, int cols, int K, const kr_pub *pub, int tail_tiles,
                      int order_rows, void *stream);

/* Gate/up GEMM with SwiGLU applied in its epilogue (the relay of
 * matmul_gate/up -> Silu -> Mul at MFMA-tile granularity, handed over in
 * registers): for A[M,K] . Bt[2*cols,K]^T with gate/up interleaved in groups
 * of 8 columns, writes act[M, cols] (row stride ld_act) =
 * bf16(bf16(silu(gate)) * up) with the rounding of kr_op_elementwise's
 * swiglu_gu over the stored product; the [M, 2*cols] product itself is not
 * written. cols must be a multiple of 8. Replaces the same reference call
 * sites as kr_op_gemm_swiglu (exec/qwen_main.cpp:616-644, 888-889). */
int kr_op_gemm_swiglu_epilogue(int dtype, const void *A, int64_t lda, const void *Bt, int64_t ldb, void *act,
                               int64_t ld_act, int M, int cols, int K, void *stream);

/* Row-tiled relay of a projection to its Add+RMSNorm consumer (the
 * reference's down -> Add+RMSNorm tile loop, exec/qwen_main.cpp:1274-1302,
 * on one device and without the all-reduce; the consumer is aclnnAddRmsNorm,
 * :548-565): C[M,N] = A . Bt^T is released in relay tiles of
 * pub->rows_per_tile rows through pub's control blocks, and as soon as a
 * tile is released the launch's own workgroups compute, for each of its rows,
 * sum = bf16(res + C) and y = bf16(gamma * bf16(sum * rstd)),
 * rstd = 1/sqrt(mean(sum^2) + eps) (rstd_out fp32 [M], optional; sum may be
 * NULL), bit-identical to kr_op_rowop(KR_ROW_ADD_RMSNORM) over C. Each
 * release is consumed by the same launch: the tile's block ends with
 * consumed advanced and status 1 (2 if a wait ran past max_spins). C, res,
 * y and sum are packed [M, N]; N in 136..4096, a multiple of 8. ws/counters
 * as for kr_op_gemm_streamk (NULL: data-parallel tiles). Fails (non-zero)
 * when a relay tile's producer workgroups cannot all be resident at once:
 * use smaller relay tiles. Other work on the device may keep them from being
 * placed together (another such call on another stream takes up to every
 * CU): waits then end after about half a millisecond without the release and
 * the workgroup that releases the tile works the rows left over, so the call
 * gets slower and its results stay the same. */
int kr_op_gemm_add_rmsnorm(int dtype, const void *A, int64_t lda, const void *Bt, int64_t ldb, void *C, int M,
                           int N, int K, const void *res, const void *gamma, void *y, void *sum, float *rstd_out,
                           float eps, const kr_pub *pub, uint32_t max_spins, void *ws, size_t ws_bytes,
                           int32_t *counters, int n_counters, void *stream);

/* Split-K GEMM for shapes whose output tiles are fewer than the CUs
 * (the reference's q/k/v, o and down projections at prefill sizes,
 * exec/qwen_main.cpp:499-512, 1336-1344): each tile (256x256, or 64 / 128 x
 * 128 below 1920 rows) runs in pieces of K on as many CUs, summed in fixed
 * piece order by the last of them, so the bits depend on the shape only (a
 * row-split launch of the same GEMM would differ; use it where no launch is
 * split). Same operands and rounding as kr_op_gemm (bias added to the
 * stored product). ws/counters: caller-owned device memory of at least the
 * sizes kr_op_gemm_streamk_workspace reports; the counters must be zero
 * before the first launch and are left zero; launches sharing them must be
 * ordered (one stream). A shape the plan does not cover (0 bytes reported)
 * runs as kr_op_gemm. */
int kr_op_gemm_streamk_workspace(int M, int N, int K, size_t *ws_bytes, int *counters);
int kr_op_gemm_streamk(int dtype, const void *A, int64_t lda, const void *Bt, int64_t ldb, void *C, int64_t ldc,
                       const void *bias, int M, int N, int K, void *ws, size_t ws_bytes, int32_t *counters,
                       int n_counters, void *stream);

/* kr_op_gemm_streamk without a workspace argument, allocating nothing: the
 * partial sums and tile counters live in a device array of the library
 * (48 MiB of partials, 1024 counters; each GPU it runs on holds one until
 * the process ends). No counterpart in the reference: for callers that
 * cannot allocate device memory (code under HIP graph capture, serving loops
 * that forbid hipMalloc). Same plan, piece order and bits as
 * kr_op_gemm_streamk; the counters are cleared at every call. Shapes whose
 * split needs more than the array holds fail with an error naming both
 * sizes. All calls on one GPU share the array: calls that may overlap in
 * time on one GPU (different streams, or host threads without ordering)
 * race and must not be issued. Products with M or N below 256 or K below 2048
 * take none of it: they run, and have the bits, as kr_op_gemm, and may
 * overlap with anything. */
int kr_op_gemm_streamk_noalloc(int dtype, const void *A, int64_t lda, const void *Bt, int64_t ldb, void *C,
                               int64_t ldc, const void *bias, int M, int N, int K, void *stream);

/* Elementwise op on [rows, cols]; x1 used by mul/add/swiglu; dtype_out
 * differs from dtype_in only for cast. tile_rows = relay granularity
 * (0 = rows); grid = workgroups (0 = sized to the tensor). wait/pub may be
 * NULL. Replaces aclnnGelu / aclnnCast (reference
 * exec/runtime/op_impl.cpp:214-228), aclnnSilu / aclnnMul / aclnnAdd
 * (exec/qwen_main.cpp:514-529, 616-644). */
int kr_op_elementwise(int op, int dtype_in, int dtype_out, const void *x0, const void *x1, void *y,
                      int rows, int cols, int tile_rows, int grid, const kr_wait *wait,
                      const kr_pub *pub, void *stream);

/* Row op on [rows, cols]: softmax along cols; rmsnorm; add_rmsnorm (x1 =
 * second addend, sum_out = rounded sum). rstd_out (fp32 [rows]) and sum_out
 * may be NULL. Replaces aclnnSoftmax dim=1 (reference
 * exec/runtime/op_impl.cpp:229-233), aclnnRmsNorm and aclnnAddRmsNorm
 * (exec/qwen_main.cpp:531-565). */
int kr_op_rowop(int op, int dtype, const void *x0, const void *x1, const void *gamma, void *y,
                void *sum_out, float *rstd_out, int rows, int cols, float eps, int tile_rows,
                int grid, const kr_wait *wait, const kr_pub *pub, void *stream);

/* Standalone one-workgroup wait for producer rows [lo, hi) (the reference's
 * separate kr_wait_* launch) and standalone release of tile `tile` (the
 * reference's kr_publish_* launch). */
int kr_op_wait(const kr_wait *wait, int lo, int hi, void *stream);
int kr_op_publish(const kr_pub *pub, int tile, void *stream);

/* out[r,:] = table[ids[r],:] (ids int64; out-of-range ids give zero rows).
 * Replaces aclnnEmbedding (reference exec/qwen_main.cpp:646-659). */
int kr_op_embedding(const void *table, const int64_t *ids, void *out, int rows, int cols,
                    int64_t vocab, void *stream);

/* In-place rotate-half RoPE on x[S, heads, D] (row stride ld elements) with
 * cos/sin tables [>=S, D]. Replaces aclnnApplyRotaryPosEmb layout 1
 * (reference exec/qwen_main.cpp:567-582). */
int kr_op_rope(int dtype, void *x, int64_t ld, int S, int heads, int D, const void *cos_t,
               const void *sin_t, void *stream);

/* Causal GQA attention, q [S,HQ,D], k/v [S,HKV,D], out [S,HQ,D], D in {64,128};
 * ld* = row strides in elements (0 = packed heads*D).
 * Replaces aclnnFlashAttentionScore (reference exec/qwen_main.cpp:591-614). */
int kr_op_attention(int dtype, const void *q, int64_t ldq, const void *k, int64_t ldk,
                    const void *v, int64_t ldv, void *out, int64_t ldo, int S, int HQ, int HKV,
                    int D, float scale, void *stream);

/* kr_op_attention with long causal rows split across workgroups: query
 * blocks of more than 16 key blocks are cut into up to 4 pieces whose fp32
 * partials the last piece sums in piece order (deterministic; the bits
 * depend on S only). ws / counters of the sizes kr_op_attention_workspace
 * reports (0 bytes: nothing to split, the call runs unsplit); counters zero
 * before the first call and left zero by every call; calls sharing them must
 * not overlap. Same role as kr_op_attention (reference
 * exec/qwen_main.cpp:591-614, FlashN); the split is a scheduling choice of
 * this library with no reference counterpart. */
int kr_op_attention_workspace(int S, int HQ, int D, size_t *ws_bytes, int *counters);
int kr_op_attention_split(int dtype, const void *q, int64_t ldq, const void *k, int64_t ldk,
                          const void *v, int64_t ldv, void *out, int64_t ldo, int S, int HQ, int HKV,
                          int D, float scale, void *ws, size_t ws_bytes, int32_t *counters,
                          int n_counters, void *stream);

/* dst[C,R] = src[R,C]^T for 16-bit elements (weight re-layout at load; the
 * reference stores matmul weights as weight_t [K,N], scripts/export_model.py:159-161). */
int kr_op_transpose(const void *src, void *dst, int R, int C, void *stream);

/* A stream with a hardware queue of its own (CU-masked to every CU). Two
 * relay parties that wait on each other on the device must not share a queue
 * (a queue runs its kernels in order); ordinary streams are multiplexed onto
 * a few queues. Returns NULL on failure. No reference counterpart: the
 * reference's two streams feed separate AIC and AIV engines
 * (exec/qwen_main.cpp:206-209). */
void *kr_op_stream_create(void);
int kr_op_stream_destroy(void *stream);

/* ------------------------------------------------------------------------
 * Paged key/value cache: what a program that goes on after the prompt needs
 * (no counterpart in the reference, which stops at the prefill). Plain host
 * structs; the pointers in them are device memory and outlive the calls.
 */

/* The cache of a model: k and v are [layers, pages, page_size, heads,
 * head_dim] 16-bit tensors with the same strides (elements; rows of head_dim
 * contiguous; strides positive, multiples of 8, below 2^31 but for the
 * layers'). Token t of a sequence is row t % page_size of the page that its
 * table names at t / page_size. page_size >= 1, head_dim 64 or 128. */
typedef struct kr_cache {
    void *k;
    void *v;
    int64_t layer_stride;
    int64_t page_stride;
    int64_t token_stride;
    int64_t head_stride;
    int32_t layers;
    int32_t pages;
    int32_t page_size;
    int32_t heads;
    int32_t head_dim;
    int32_t dtype; /* KR_BF16 or KR_F16 */
} kr_cache;

/* A launch's sequences. Sequence b has lens[b] tokens in the cache before the
 * launch's own, and rows starts[b] .. starts[b+1]-1 of the launch are its new
 * tokens (none is allowed), whose keys and values stand in the cache behind
 * them, at positions lens[b], lens[b]+1, ..; table[b] names its pages.
 * tree == NULL: a new token sees the cached ones, the new ones before it and
 * itself. Otherwise row r's words tree[r * ld_tree ..] say which new tokens
 * of its sequence it sees: bit j % 64 of word j / 64 for new token j (its own
 * bit too); every cached one is seen.
 * The arrays are read on the device when the launch runs, so a captured graph
 * follows their contents. Nothing in them can lead outside the tensors: rows
 * outside the launch's and new tokens past max_new are not worked, tokens past the
 * table's end are not there, and the keys of a page id outside 0..pages-1 are
 * seen by nobody. */
typedef struct kr_seqs {
    const int32_t *table;  /* [seqs, table_pages], row stride ld_table */
    int64_t ld_table;
    const int32_t *lens;   /* [seqs] */
    const int32_t *starts; /* [seqs + 1], ascending */
    const uint64_t *tree;  /* [rows of the launch, tree_words], row stride ld_tree; or NULL */
    int64_t ld_tree;
    int32_t table_pages;
    int32_t seqs;
    int32_t max_new;    /* no sequence has more new tokens; <= 64 * tree_words with a tree */
    int32_t tree_words;
} kr_seqs;

/* Rotation tables [positions, head_dim] and, optionally, the gains of the
 * per-head norms of q and k (both or none; of the activations' type).
 * table_dtype: KR_F32 or the activations' type. chain != 0 rounds as the
 * separate calls do (x * rstd, then the gain's product to 16 bits before the
 * rotation: the bits of kr_op_rowop and kr_op_rope); 0 rounds once. */
typedef struct kr_rope {
    const void *cos_t;
    const void *sin_t;
    const void *q_gamma;
    const void *k_gamma;
    int64_t positions;
    int32_t head_dim;
    int32_t table_dtype;
    int32_t chain;
    float eps;
} kr_rope;

/* Per-head RMSNorm (with gammas) and rotate-half RoPE of q [rows, HQ, D] and
 * k [rows, HKV, D] in one pass (D 64, 128 or 256; ld* = row strides, 0 =
 * packed). Row r stands at positions[r] (NULL: r); a position outside the
 * tables gives zero rows. An output may be its own input (the same rows);
 * one that overlaps an input or the other output otherwise is refused. Same
 * role as kr_op_rowop's rmsnorm and kr_op_rope in sequence (reference
 * EmitQkNorm, exec/qwen_main.cpp:1346-1357, and Rope, :567-582). */
int kr_op_qk_norm_rope(int dtype, const kr_rope *rope, const void *q, int64_t ldq, const void *k, int64_t ldk,
                       void *q_out, int64_t ldqo, void *k_out, int64_t ldko, const int64_t *positions, int rows,
                       int HQ, int HKV, void *stream);

/* The same with k and v [rows, heads, D] written to their cache slots
 * (slots[r] = page * page_size + row in the page; outside the cache, -1 say:
 * not written). No two rows may share a slot: it would hold a mixture. q_out
 * overlaps neither k, v nor the layer (refused), and q only as its own input. */
int kr_op_qk_norm_rope_cache(const kr_rope *rope, const kr_cache *cache, int layer, const void *q, int64_t ldq,
                             const void *k, int64_t ldk, const void *v, int64_t ldv, void *q_out, int64_t ldqo,
                             const int64_t *positions, const int64_t *slots, int rows, int HQ, void *stream);

/* Attention of a launch's new tokens over the pages: out [rows, HQ, D] (rows
 * of no sequence are left alone; refused where out overlaps q or the layer, the
 * gaps between its rows included), query head h reads key head h / (HQ /
 * heads), scores scaled by `scale` (> 0). A row that sees no key gives zeros.
 * What a row does not see has no part in its result, NaN and infinities
 * included. ws / counters: caller-owned device memory of at least the sizes
 * kr_op_attention_paged_workspace reports (functions of the handles' host
 * fields alone; both 0 where no sequence is long enough), with which long
 * sequences are cut into pieces that run side by side and are summed in order;
 * the counters must be zero before the first call and are left zero; calls
 * sharing them must be ordered. NULL: uncut. The bits depend on the batch's
 * lengths, not on which piece ends when. */
int kr_op_attention_paged_workspace(const kr_cache *cache, const kr_seqs *seqs, int HQ, size_t *ws_bytes,
                                    int *counters);
int kr_op_attention_paged(const kr_cache *cache, int layer, const kr_seqs *seqs, const void *q, int64_t ldq,
                          void *out, int64_t ldo, int rows, int HQ, float scale, void *ws, size_t ws_bytes,
                          int32_t *counters, int n_counters, void *stream);

/* kr_op_attention_paged that also writes lse[r * ld_lse + head] = ln sum
 * exp(scale q.k) over the keys that the row sees (-infinity where it sees
 * none), fp32 [rows, HQ], ld_lse = 0 for packed rows: what
 * kr_op_attention_paged_weigh takes. The same results and workspace; lse
 * overlaps no other tensor of the call (refused for all that it passes). */
int kr_op_attention_paged_lse(const kr_cache *cache, int layer, const kr_seqs *seqs, const void *q, int64_t ldq,
                              void *out, int64_t ldo, float *lse, int64_t ld_lse, int rows, int HQ, float scale,
                              void *ws, size_t ws_bytes, int32_t *counters, int n_counters, void *stream);

/* Attention weight that cached tokens got so far: fp32 [layers, entries,
 * heads, width], the strides in elements (rows of width contiguous, no two
 * overlapping). Sequence b of a launch has entry[b] (device [seqs]; NULL: b),
 * token t of it column t. A sequence whose entry is outside 0..entries-1 has
 * none: the calls below leave it alone. No two sequences of a launch may have
 * the same entry. */
typedef struct kr_weights {
    float *w;
    int64_t layer_stride;
    int64_t entry_stride;
    int64_t head_stride;
    int32_t layers;
    int32_t entries;
    int32_t heads;
    int32_t width;
    const int32_t *entry;
} kr_weights;

/* Adds what the cached tokens get from a launch's new tokens to their weights
 * of a layer: for key head h and column j of sequence b
 *   sum over new tokens i that see j, query heads g of h: exp(scale q_ig.k_j - lse[i, g])
 * is added to decay times the old value for a cached token (decay = 0: the old
 * value is not read), and stands for itself for a new one. q, lse as of
 * kr_op_attention_paged_lse for the same handles; a row whose lse is
 * -infinity, and what a row does not see, count nothing, whatever is there.
 * last > 0: only the last `last` new tokens of each sequence count. Columns
 * past the width are left out, sequences without new tokens left alone.
 * path != NULL: the drafts of seqs have been accepted and moved together
 * (kr_op_cache_compact with this path and these handles); new token i of
 * sequence b is row starts[b] + path[b][i], i < path_lens[b], and sees the
 * cached ones and the path up to itself (the handle's tree is not looked at);
 * entries of the path that name no row of the sequence count nothing. path:
 * device [seqs, path_width], row stride ld_path. ws: caller-owned device
 * memory of at least kr_op_attention_paged_weigh_workspace's size, for one
 * stream at a time (it may hold anything). The same bits at every call. */
int kr_op_attention_paged_weigh_workspace(const kr_cache *cache, const kr_seqs *seqs, int HQ, size_t *ws_bytes);
int kr_op_attention_paged_weigh(const kr_cache *cache, int layer, const kr_seqs *seqs, const void *q, int64_t ldq,
                                const float *lse, int64_t ld_lse, int rows, int HQ, float scale,
                                const kr_weights *weights, int last, float decay, const int32_t *path,
                                int64_t ld_path, int path_width, const int32_t *path_lens, void *ws, size_t ws_bytes,
                                void *stream);

/* Sequences with more than `budget` tokens (lens of the handle, its starts and
 * tree are not looked at) come down to that many, layer by layer and key head
 * by key head: the first `sinks` and the last `recent` tokens stay, and of the
 * others the budget - sinks - recent with the largest weights, of equal ones
 * the first (a NaN is below everything). Afterwards token i of the sequence is
 * the one that was token keep[layer, b, head, i]: what stays and stands at
 * sinks..budget-recent-1 is not moved, the others among the largest take the
 * free places there, first to first, and the recent ones follow in their
 * order; keys, values and weights move alike, columns and rows from budget on
 * keep what they hold. (Attention does not depend on the order of cached
 * tokens: their keys carry their positions.) A sequence with fewer tokens has
 * 0, 1, .. in keep, then -1; so has one without weights or with more tokens than
 * columns, but for the weights and rows, which stay. keep: int32 device
 * [layers, seqs, heads, budget], packed. Rows of pages that are none stay.
 * Sequences must not share pages below position budget. 0 <= sinks, recent;
 * sinks + recent <= budget. */
int kr_op_cache_evict(const kr_cache *cache, const kr_seqs *seqs, const kr_weights *weights, int budget, int sinks,
                      int recent, int32_t *keep, void *stream);

/* Drafted tokens and what the target model says to them. Row r of a launch
 * (rows starts[b].. of sequence b, as in kr_seqs) is a token; logits
 * [rows, vocab] (row stride ld_logits; KR_BF16, KR_F16 or KR_F32) are the
 * target's after it. The first row of a sequence is its last token, decided
 * before; the others are drafts: row i of the sequence is tokens[r], drawn to
 * follow row parents[r] of the sequence (an earlier one; otherwise it follows
 * nothing). parents == NULL: each row follows the one before it. draft
 * [rows, vocab] (row stride ld_draft, draft_dtype): the probabilities from
 * which the tokens that follow row r were drawn, each on its own; NULL: the
 * drafts were not drawn. A negative or NaN probability is 0, a NaN logit -infinity. Any
 * vocab and strides >= vocab; rows that are not 16-byte aligned are read more slowly. */
typedef struct kr_drafts {
    const void *logits;
    int64_t ld_logits;
    const void *draft;
    int64_t ld_draft;
    const int64_t *tokens;    /* device [rows] */
    const int32_t *parents;   /* device [rows], or NULL */
    const float *u;           /* device [rows]: uniform in [0, 1), one for each draft */
    const float *u_next;      /* device [seqs]: one for the token that follows */
    const float *temperature; /* device [seqs], or NULL: 1; <= 0 or NaN: the first of the largest logits has it all */
    int32_t dtype;
    int32_t draft_dtype;
    int32_t vocab;
    int32_t rows;
} kr_drafts;

/* Rejection sampling down the drafts of each sequence. At a row with
 * probabilities p = softmax(logits / temperature) its drafts are tried in
 * order: token x is accepted if u q(x) < p(x) (q = 1 where the drafts were
 * not drawn), and the walk goes on there; if not, p becomes max(p - q, 0)
 * over its sum (without q: p without x over its sum; where nothing is left, p
 * stays). Where none is accepted, the token that follows is the first v with
 * p(0) + .. + p(v) > u_next (p(0) + .. + p(vocab - 1)), or the last with p > 0.
 * The kept tokens are then distributed as the target's own. All of it in 64
 * bits. Out: path[b][..] int32 [seqs, width], row stride ld_path: the accepted
 * rows of the sequence from 0 on, then -1 (kr_op_cache_compact takes it; a
 * walk ends after `width` rows, with the p of the last one); path_lens
 * [seqs]; next [seqs]: -1 where a row has no logit above -infinity, or the
 * sequence no rows. max_new <= 1024; with draft and parents fewer than 2^21
 * sequences; of kr_seqs starts and max_new are looked at. ws: caller-owned
 * device memory of at least the sizes that kr_op_verify_drafts_workspace
 * reports (functions of host fields alone); counters zero before the first
 * call and left zero; calls sharing them must be ordered. */
int kr_op_verify_drafts_workspace(const kr_drafts *drafts, const kr_seqs *seqs, size_t *ws_bytes, int *counters);
int kr_op_verify_drafts(const kr_drafts *drafts, const kr_seqs *seqs, int32_t *path, int64_t ld_path, int width,
                        int32_t *path_lens, int64_t *next, void *ws, size_t ws_bytes, int32_t *counters,
                        int n_counters, void *stream);

/* Page dst[i] becomes a copy of page src[i], keys and values of every layer.
 * src and dst are HOST arrays, read during the call. Refused: ids outside the
 * cache, a page named twice in dst, a page in both src and dst. */
int kr_op_cache_copy_pages(const kr_cache *cache, const int32_t *src, const int32_t *dst, int n, void *stream);

/* After drafts have been accepted: for every layer's keys and values and each
 * sequence b, the rows at positions lens[b] + path[b][i], i < path_lens[b],
 * move to lens[b] + i, as if all were read before any is written. path:
 * device [seqs, width], row stride ld_path, width <= 256; entries below 0 and
 * rows off the table or the cache stay. Uses the handle's table and lens.
 * Sequences must not share the pages of these rows. */
int kr_op_cache_compact(const kr_cache *cache, const kr_seqs *seqs, const int32_t *path, int64_t ld_path, int width,
                        const int32_t *path_lens, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* KR_OPS_H */
