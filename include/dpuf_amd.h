/*
 * dpuf_amd.h -- entry points this build adds next to the dpuf_kernels.h ABI.
 * None of them has a counterpart in the reference; they exist for callers
 * that want device-side greedy sampling, for parity tests (per-layer residual
 * capture, KV injection) and for measurement.  The reference ABI does not
 * depend on any of them.
 */
#ifndef DPUF_AMD_H
#define DPUF_AMD_H

#include <stddef.h>
#include <stdint.h>
#include "dpuf_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest n_tokens a single forward call accepts (the reference caps at 256;
 * 512 is a compatible superset). */
#define DPUF_AMD_MAX_BATCH 512

/* 1 when a HIP device is usable, else 0. */
DPUF_EXPORT int32_t dpuf_amd_device_ok(void);

/* Text of the first HIP error recorded by the library ("" if none). */
DPUF_EXPORT const char* dpuf_amd_last_error(void);

/* forward_batch_ex plus greedy sampling on the device: *token_out receives the
 * first-max argmax (dpuf-cli.c:1997-2004 rule) of the last row's logits, so a
 * decode loop moves 4 bytes per token instead of V floats.  logits_out may be
 * NULL (no copy) or receive the last row's logits.  Same return codes as
 * dpuf_engine_forward_batch_ex. */
DPUF_EXPORT int32_t dpuf_amd_engine_forward_argmax(void* handle, int32_t n_tokens, const int32_t* token_ids,
                                                   int32_t pos0, const float* embeds_in, int32_t use_graph,
                                                   int32_t* token_out, float* logits_out);

/* Writes / reads positions [pos0, pos0+n) of (layer, kv head) of the active
 * slot, host pointers of n * head_dim floats.  0 ok, -1 bad arguments. */
DPUF_EXPORT int32_t dpuf_amd_engine_set_kv(void* handle, int32_t layer, int32_t kv_head, int32_t pos0, int32_t n,
                                           const float* k, const float* v);
DPUF_EXPORT int32_t dpuf_amd_engine_get_kv(void* handle, int32_t layer, int32_t kv_head, int32_t pos0, int32_t n,
                                           float* k, float* v);

/* Captures the residual stream after every layer ([num_layers][n][hidden])
 * for calls with n_tokens <= max_tokens (0 disables).  get_capture copies
 * num_layers * max_tokens * hidden floats.  0 ok, -1 error. */
DPUF_EXPORT int32_t dpuf_amd_engine_set_capture(void* handle, int32_t max_tokens);
DPUF_EXPORT int32_t dpuf_amd_engine_get_capture(void* handle, float* out, size_t n_floats);

/* Kernel timing with HIP events on the engine's stream.  Kinds:
 * 0 gate/up GEMV, 1 down GEMV, 2 QKV GEMV, 3 O GEMV, 4 LM head, 5 attention,
 * 6 norm+prep, 7 whole forward call.  get_timing returns total ms, launch
 * count and algorithmic bytes for a kind; enabling resets the counters. */
DPUF_EXPORT void dpuf_amd_engine_set_timing(void* handle, int32_t enable);
DPUF_EXPORT int32_t dpuf_amd_engine_get_timing(void* handle, int32_t kind, double* total_ms, int64_t* count,
                                               double* bytes);

/* Graph replay of one-token steps, on by default: the reference entry points
 * and dpuf_amd_engine_forward_argmax (use_graph set) replay a HIP graph
 * captured once per step shape.  0 enqueues every kernel of every step
 * instead (for per-kernel traces) and releases the graphs kept so far. */
DPUF_EXPORT void dpuf_amd_engine_set_graphs(void* handle, int32_t enable);

/* Mode 12 tile bytes resident in HBM (all layers + LM head). */
DPUF_EXPORT uint64_t dpuf_amd_engine_weight_bytes(void* handle);

/* Number of forward calls in which the LM-head early exit fired. */
DPUF_EXPORT int64_t dpuf_amd_engine_early_exit_count(void* handle);

/* Attention launches enqueued so far in this process, by path (which: 0 the
 * matrix-instruction kernels of several tokens, 1 the one-token long-context
 * kernels (scores, softmax once per row, wide P.V; one per session where they
 * serve several), 2 the split scores + LDS softmax / P.V kernels over the fp32
 * cache, 3 the one-pair-per-workgroup fallback, 4 the fused short-context
 * decode kernel, 5 every kernel over the int8 cache; 6 those of 0 whose rows
 * are streamed, 7 those of 5 with the softmax in memory); -1 for another
 * `which`.  Enqueued, not executed: a replayed graph counts at its capture
 * only.  For tests that check which path a shape takes. */
DPUF_EXPORT int64_t dpuf_amd_attn_path_count(int32_t which);

/* Times `iters` back-to-back launches of one GEMV kind over resident weights
 * (which: 0 q, 1 k, 2 v, 3 o, 4 gate, 5 up, 6 down, 7 LM head, 8 gate+up as
 * one launch, 9 q+k+v as one launch), cycling through layers
 * start..num_layers-1 so that consecutive launches read distinct weights.
 * Returns the mean ms per launch (or < 0 on error); *bytes gets the
 * algorithmic bytes of one launch (weight groups + activations + outputs). */
DPUF_EXPORT double dpuf_amd_gemv_bench(void* handle, int32_t which, int32_t M, int32_t iters, int32_t start_layer,
                                       double* bytes);

/* Copies `bytes` between two device buffers `iters` times (hipMemcpyAsync
 * device to device) and returns the mean ms per copy; a reference of known
 * traffic for calibrating hardware byte counters.  < 0 on error. */
DPUF_EXPORT double dpuf_amd_copy_bench(size_t bytes, int32_t iters);

/* Caps the workgroups of an M = 1 GEMV launch at n (n <= 0: no cap beyond
 * what the device holds at once), process-wide.  A smaller cap gives each
 * workgroup more 8-row groups to walk; results do not depend on it.  For
 * tests of the multi-group path and for tuning. */
DPUF_EXPORT void dpuf_amd_set_gemv_max_workgroups(int32_t n);

/* Runs the device logit reductions on n host floats placed `offset` floats
 * (0..3) past a 16-byte boundary: mode 1 returns the first-maximum index the
 * greedy sampler takes (dpuf-cli.c:1997-2004); mode 0 returns the Zone-A
 * early-exit flag, 1 when thr > 0 and top1 - top2 >= thr over the multiset
 * (dpuf_engine.c:2101-2110).  -1 on error.  For tests. */
DPUF_EXPORT int32_t dpuf_amd_reduce_check(const float* x, int32_t n, int32_t offset, int32_t mode, float thr);

/* dpuf_amd_reduce_check without allocating: the reduction of n floats
 * already in device memory (d_x) into one int32 in device memory (d_out),
 * enqueued on hip_stream (a hipStream_t; NULL is the default stream) without
 * synchronising.  mode and thr as in dpuf_amd_reduce_check.  The partials
 * live in a 512-byte array of the library's that each device holds until the
 * process ends; every call on a device shares it, so calls that overlap on
 * one device (two streams, two threads) race and must be serialised by the
 * caller.  n is at most DPUF_AMD_NOALLOC_MAX_N.  Returns 0 when enqueued, -1
 * bad pointer or mode, -2 n out of range, -6 device error
 * (dpuf_amd_last_error says which).
 * No counterpart in the reference: for callers that cannot allocate device
 * memory -- code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc -- and sample the greedy token on the device. */
#define DPUF_AMD_NOALLOC_MAX_N (1 << 30)
DPUF_EXPORT int32_t dpuf_amd_reduce_check_noalloc(const float* d_x, int32_t n, int32_t mode, float thr,
                                                  int32_t* d_out, void* hip_stream);

/* One next token for each of n sessions in one pass (serving several
 * conversations with one read of the weights): token_ids[i] is appended to
 * KV slot slot_ids[i] (distinct slots, allocated on demand) at positions[i]
 * (any position below max_seq_len, for either KV cache type); logits_out
 * [n][V] and/or tokens_out [n] (greedy ids), in the caller's order.  Per token
 * the results equal a one-token dpuf_engine_forward_batch on that slot (decode
 * keep-tiles setting, no Zone-A early exit).  The projections and the LM head
 * run once for all n tokens; the attention of sessions with at most 192 keys
 * (fp32 cache) is one launch, every other session's takes the one-token
 * launches of its own length.  0 on success; -1 bad arguments or a repeated
 * slot, -2 above DPUF_AMD_MAX_BATCH or out of memory, -3 position out of
 * range, -4 token id out of range, -5 head dim other than 64/128/256, -6
 * device error.  No counterpart in the reference,
 * whose forward serves one slot per call; for serving loops (dpuf-cli.c's
 * one-slot-per-call generation stays as it is). */
DPUF_EXPORT int32_t dpuf_amd_engine_forward_slots(void* handle, int32_t n, const int32_t* slot_ids,
                                                  const int32_t* token_ids, const int32_t* positions,
                                                  float* logits_out, int32_t* tokens_out);

/* dpuf_qr_verify_tiles_ex (reference dpuf_avx2.c:846-908) with the CRC32 of
 * every tile body computed on the GPU: same arguments, tile_ok_out and return
 * value (the number of bad tiles; -1 on error).  No counterpart in the
 * reference, which checks tiles on the CPU while binding tensors; for hosts
 * that verify multi-GB files before dpuf_engine_create. */
DPUF_EXPORT int32_t dpuf_amd_verify_tiles_device(int32_t mode, int32_t n_tiles, int32_t cols,
                                                 const uint8_t* tensor_base, const uint64_t* tile_offsets,
                                                 uint8_t* tile_ok_out);

/* ---- Paged serving -------------------------------------------------------
 * A KV cache in pages shared by many sequences, and the operators over it:
 * RoPE with the append of new rows, attention of new tokens, accumulation of
 * the attention weight each cached row receives, eviction by that weight, and
 * sampling.  All pointers inside the descriptors and all d_ arguments are
 * device memory of one device, which need not be the current one; work is
 * enqueued on hip_stream (a hipStream_t of that device; NULL: its default
 * stream) without synchronising and may be captured into a HIP graph: lengths,
 * tables and sampling settings are read on the device, so a replay takes their
 * current contents.  Nothing is allocated; calls that share a workspace must
 * not overlap.  No counterparts in the reference.
 *
 * Return codes: 0 enqueued; -1 NULL or misaligned pointer, host memory where
 * device memory is needed, pointers of different devices, or an output or
 * workspace that shares memory with anything else that the call reads or
 * writes (pools count from their first row to their last; k and v of one
 * allocation may interleave, and an operator says where it works in place);
 * -2 a size or setting out of range; -4 a stride that is not a multiple of 8
 * elements or too small; -5 a type or head dim that is not built; -6 device
 * error (dpuf_amd_last_error); -7 workspace too small. */

/* Element types. */
enum {
    DPUF_AMD_F32  = 0,
    DPUF_AMD_BF16 = 1,
    DPUF_AMD_F16  = 2
};

/* One layer's pages.  Row r of page p of kv head h starts at element
 * p * page_stride + h * head_stride + r * row_stride of k and of v (any order
 * of the three, each a multiple of 8 elements and at least head_dim,
 * row_stride at most 2^26; k and v on 16 bytes).  w holds one accumulated
 * weight per row, [n_pages][n_kv_heads][page_size], or is NULL where no
 * operator needs it. */
typedef struct {
    int32_t type;         /* DPUF_AMD_BF16 or DPUF_AMD_F16 */
    int32_t n_pages;
    int32_t page_size;    /* rows: a power of two, 16 to 1024 */
    int32_t n_kv_heads;   /* 1 to 256 */
    int32_t head_dim;     /* 64, 128 or 256 */
    int64_t page_stride;
    int64_t head_stride;
    int64_t row_stride;
    void* k;
    void* v;
    float* w;
} DpufAmdPages;

/* A ragged batch: sequence s has new rows row_start[s] .. row_start[s + 1] - 1
 * of the call's n_rows, which are the last of its ctx_len[s] cached rows
 * (new ones included); its cached row i is row i % page_size of page
 * page_table[s * table_stride + i / page_size].  A sequence may have no new
 * rows.  Lengths are clamped to the table and to n_rows; a cached row on a
 * page outside [0, n_pages) is absent: never read, written or attended to. */
typedef struct {
    int32_t n_seqs;              /* 1 to 16384 */
    int32_t n_rows;              /* 0 to 65536 */
    int32_t table_stride;        /* table entries per sequence; times page_size at most 2^30 */
    int32_t max_ctx;             /* about the longest ctx_len: how the work is split, not a bound */
    const int32_t* row_start;    /* [n_seqs + 1], ascending from 0 */
    const int32_t* ctx_len;      /* [n_seqs] */
    const int32_t* page_table;   /* [n_seqs][table_stride] */
} DpufAmdBatch;

/* How a model turns positions into angles. */
enum {
    DPUF_AMD_ROPE_PLAIN  = 0,
    DPUF_AMD_ROPE_LINEAR = 1,    /* every frequency / factor */
    DPUF_AMD_ROPE_LLAMA3 = 2,    /* / factor below low_freq turns over orig_max_pos, as is above high_freq */
    DPUF_AMD_ROPE_YARN   = 3     /* ramp between the dims of beta_fast and beta_slow turns; rotated columns scaled */
};
typedef struct {
    int32_t rot_dim;             /* rotated columns of each head, even, 2 to 256 */
    float   theta;
    int32_t scaling;
    float   factor;
    float   low_freq, high_freq; /* llama3 */
    float   beta_fast, beta_slow; /* yarn */
    int32_t orig_max_pos;        /* llama3, yarn: positions the model was trained on */
} DpufAmdRopeSpec;

/* Host only: turns[j] = turns per position of pair j (rot_dim / 2 of them)
 * and *scale, the factor on rotated columns (yarn: 0.1 ln factor + 1, else 1).
 * 0 ok, -1 NULL, -2 a setting out of range. */
DPUF_EXPORT int32_t dpuf_amd_rope_turns(const DpufAmdRopeSpec* spec, double* turns, float* scale);

/* A rotation as the device takes it: columns 0 .. rot_dim - 1 of a head in
 * pairs (j, j + rot_dim / 2), or (2j, 2j + 1) when interleaved; the other
 * columns stay as they are. */
typedef struct {
    const double* turns;         /* device, [rot_dim / 2] */
    int32_t rot_dim;             /* even, 2 to head_dim */
    int32_t interleaved;
    float   scale;
} DpufAmdRope;

/* New rows of q, k and v (elements of in_type; row strides in elements, each
 * head's head_dim columns contiguous, rows on 16 bytes): with d_q_norm /
 * d_k_norm set, the RMSNorm of each head with these head_dim weights; the
 * rotation by d_positions[row] (0 to 2^31 - 1); then q into d_q_out
 * [n_rows][n_q_heads][head_dim] (the pages' type; it may be d_q itself where
 * the types and strides agree) and k and v into the rows' places in the pages,
 * each rounded once; a written row's weight (pages->w set) becomes 0.  Rows
 * behind the last sequence's are left as they were.  d_q and d_q_out may both
 * be NULL (n_q_heads 0): the append alone. */
DPUF_EXPORT int32_t dpuf_amd_rope_append(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                         const DpufAmdRope* rope, const int32_t* d_positions, int32_t in_type,
                                         int32_t n_q_heads, const void* d_q, const void* d_k, const void* d_v,
                                         int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                         const float* d_q_norm, const float* d_k_norm, float eps, void* d_q_out,
                                         void* hip_stream);

/* Positions of several axes (time, height and width of a picture's or film's
 * patches; text has the same on all): pair j of the rotated columns turns by
 * the position on its axis.  Axes take sections[0], sections[1], ... pairs one
 * after the other, or in turn: axis a > 0 the pairs a, a + n_axes, ... as many
 * as its section says, axis 0 all others.  n_axes 1 to 4; sections 0 or more,
 * rot_dim / 2 together (entries past n_axes are not read), and in turn no more
 * than there are such pairs. */
typedef struct {
    int32_t n_axes;
    int32_t sections[4];
    int32_t in_turn;
} DpufAmdRopeAxes;

/* dpuf_amd_rope_append with a position on each axis: row's on axis a is
 * d_positions[a * pos_stride + row], pos_stride at least n_rows (with one axis
 * it is not read).  Everything else as above. */
DPUF_EXPORT int32_t dpuf_amd_rope_append_axes(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                              const DpufAmdRope* rope, const DpufAmdRopeAxes* axes,
                                              const int32_t* d_positions, int64_t pos_stride, int32_t in_type,
                                              int32_t n_q_heads, const void* d_q, const void* d_k, const void* d_v,
                                              int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                              const float* d_q_norm, const float* d_k_norm, float eps, void* d_q_out,
                                              void* hip_stream);

/* Attention of the new rows over the pages: row i of a sequence's n attends
 * to cached rows 0 .. ctx_len - n + i; query head j to kv head
 * j / (n_q_heads / n_kv_heads), at most 32 query heads per kv head.  d_q
 * [n_rows][n_q_heads][head_dim] of the pages' type, on 16 bytes; d_out of the
 * same shape, out_type that type or DPUF_AMD_F32; d_lse [n_rows][n_q_heads]
 * (or NULL) the logarithm of each row's sum of exp(scale q.k).  A row with no
 * cached row to attend to gives 0 and -infinity; rows behind the last
 * sequence's are left as they were.  Sums are fp32; probabilities enter the
 * product with V rounded to the pages' type, and in bf16 those of decoding
 * sequences (up to 16 new rows times query heads per kv head, 32 where a row
 * alone has more than 16) with the remainder beside them.  d_workspace of at
 * least dpuf_amd_paged_attn_workspace bytes, on 16 bytes (NULL when that is 0).
 * That is the need of these very arguments: fewer rows, sequences or keys are
 * split otherwise and may need more, so a program that keeps one workspace
 * takes the largest over the batches it makes, or asks before each call (the
 * host's arithmetic alone). */
DPUF_EXPORT size_t dpuf_amd_paged_attn_workspace(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                                 int32_t n_q_heads);
DPUF_EXPORT int32_t dpuf_amd_paged_attn(const DpufAmdBatch* batch, const DpufAmdPages* pages, int32_t n_q_heads,
                                        const void* d_q, float scale, int32_t out_type, void* d_out, float* d_lse,
                                        void* d_workspace, size_t workspace_bytes, void* hip_stream);

/* dpuf_amd_paged_attn with a sliding window and first tokens that stay visible:
 * the row at place p of its sequence (p = ctx_len - n + i) attends to cached
 * rows t <= p with t > p - window or t < sink.  window 1 to 2^30, itself
 * included; sink 0 to 2^30.  Table entries of pages with no row that a new row
 * attends to may hold anything, and pages that they still name may be other
 * sequences' by now: of the pool's, those beside a window's ends may be loaded,
 * but nothing of them reaches an output.  Probabilities that are rounded once
 * (all but bf16 ones of decoding sequences) count in their row's sum as they were
 * rounded, so that a row that sees one key alone gets its values bit for bit;
 * d_lse has them whole.  That holds for windows that reach everything too: such a
 * call differs from dpuf_amd_paged_attn by roundings (its keys may be split
 * otherwise as well), and the table's width does not change its outputs.  The
 * workspace is that of these arguments, window and sink among them.  Everything
 * else as above. */
DPUF_EXPORT size_t dpuf_amd_paged_attn_window_workspace(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                                        int32_t n_q_heads, int32_t window, int32_t sink);
DPUF_EXPORT int32_t dpuf_amd_paged_attn_window(const DpufAmdBatch* batch, const DpufAmdPages* pages, int32_t n_q_heads,
                                               const void* d_q, float scale, int32_t window, int32_t sink,
                                               int32_t out_type, void* d_out, float* d_lse, void* d_workspace,
                                               size_t workspace_bytes, void* hip_stream);

/* pages->w[row] = decay * d_w_in[row] + the probabilities exp(scale q.k - lse)
 * that the new rows of the row's sequence give it, summed over rows and over
 * the query heads of its kv head, for every cached row of the batch; d_w_in is
 * laid out as w, may be w itself, and counts as 0 when NULL.  d_q and d_lse
 * are what dpuf_amd_paged_attn took and gave.  No page may be in two of the
 * batch's sequences.  The same inputs give the same bits. */
DPUF_EXPORT int32_t dpuf_amd_paged_attn_weights(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                                int32_t n_q_heads, const void* d_q, float scale, const float* d_lse,
                                                float decay, const float* d_w_in, void* hip_stream);

/* Shortens every sequence longer than `keep` rows to keep rows, each kv head
 * on its own: its first `sink` and last `recent` rows stay, and of the others
 * the keep - sink - recent with the largest w (NaN and absent rows last; ties:
 * the earliest); shorter sequences stay whole.  The rows that stay, in order,
 * and their weights are copied to rows 0 .. of the sequence's pages in
 * d_dst_table [n_seqs][dst_table_stride] of dst (same type, heads and
 * head_dim; its w must be set), which must not be pages that any of the
 * batch's sequences reads (absent source rows copy as zeros).  d_kept
 * [n_seqs][n_kv_heads][keep] receives their old row numbers (entries past a
 * sequence's new length are left as they were), d_new_len [n_seqs] the new
 * lengths.  row_start and n_rows are not read. */
DPUF_EXPORT int32_t dpuf_amd_paged_evict(const DpufAmdBatch* batch, const DpufAmdPages* pages, int32_t keep,
                                         int32_t sink, int32_t recent, const DpufAmdPages* dst,
                                         const int32_t* d_dst_table, int32_t dst_table_stride, int32_t* d_kept,
                                         int32_t* d_new_len, void* hip_stream);

/* One token from each of n rows (1 to 65536) of V logits (1 to
 * DPUF_AMD_SAMPLE_MAX_VOCAB; rows row_stride elements apart).
 * Settings are arrays of n on the device; each may be NULL (off).  Row i:
 * weights exp((x - max) / temperature), NaN logits counting as -infinity and
 * +infinity leaving only its like;
 * top_k (0 or less, or V or more: off) keeps the k largest (ties: the lowest
 * indices); top_p (1 or more: off) of those the shortest run of largest ones
 * whose weights reach top_p of their sum, one at least; min_p (0 or less: off)
 * of those the ones whose weight is at least min_p times the largest.  The
 * token is the first, in index order, whose running sum of the weights kept
 * exceeds d_u[i] (in [0, 1); outside: clamped) times their sum; its
 * logarithmic share of that sum goes to d_logprobs (or NULL).  temperature 0
 * or less (or NaN): the first largest logit, and 0.  A row with no logit above
 * -infinity: -1, and -infinity.  Weights are held as integers of at least
 * 2^-38 of the largest, so sums do not depend on any order.  The workspace is
 * that of n rows of V: fewer rows are cut into more chunks and may need more. */
#define DPUF_AMD_SAMPLE_MAX_VOCAB (1 << 24)
DPUF_EXPORT size_t dpuf_amd_sample_workspace(int32_t n, int32_t V);
DPUF_EXPORT int32_t dpuf_amd_sample(int32_t type, int32_t n, int32_t V, int64_t row_stride, const void* d_logits,
                                    const float* d_temperature, const int32_t* d_top_k, const float* d_top_p,
                                    const float* d_min_p, const float* d_u, int32_t* d_tokens, float* d_logprobs,
                                    void* d_workspace, size_t workspace_bytes, void* hip_stream);

/* Scores of n rows (1 to 65536) of V logits (1 to DPUF_AMD_SAMPLE_MAX_VOCAB;
 * rows row_stride elements apart) as they are, at temperature 1, with
 * p = exp(x) / sum exp(x): NaN logits count as -infinity, +infinity leaves only
 * its like.  d_logprobs [n][n_targets] gets ln p (0 at most) of row i's tokens
 * d_targets[i * n_targets ...] (0 to DPUF_AMD_LOGPROBS_MAX_TARGETS of them; the
 * same one may be there twice; one outside [0, V) gets -infinity), d_entropy [n]
 * -sum p ln p (0 at least), d_top_tokens and d_top_logprobs [n][n_top] the n_top
 * (0 to DPUF_AMD_LOGPROBS_MAX_TOP) largest logits' tokens (ties: the lowest
 * indices) and ln p, in that order.  Fewer logits above -infinity than that
 * leave -1 and -infinity; a row without any gives -infinity and an entropy of
 * 0.  d_targets and d_logprobs may be NULL (n_targets 0), as may d_entropy, and
 * d_top_tokens and d_top_logprobs (n_top 0), not all three outputs.  Sums are
 * fp32.  The same inputs give the same bits.  The workspace (on 16 bytes) is
 * that of n rows of V: fewer rows are cut into more chunks and may need more. */
#define DPUF_AMD_LOGPROBS_MAX_TARGETS 1024
#define DPUF_AMD_LOGPROBS_MAX_TOP 64
DPUF_EXPORT size_t dpuf_amd_logprobs_workspace(int32_t n, int32_t V, int32_t n_top);
DPUF_EXPORT int32_t dpuf_amd_logprobs(int32_t type, int32_t n, int32_t V, int64_t row_stride, const void* d_logits,
                                      int32_t n_targets, const int32_t* d_targets, int32_t n_top, float* d_logprobs,
                                      float* d_entropy, int32_t* d_top_tokens, float* d_top_logprobs,
                                      void* d_workspace, size_t workspace_bytes, void* hip_stream);

/* ---- The engine over pages and with sampling ----------------------------- */

/* Sampling settings of an engine call: host arrays, entry i for token or
 * sequence i, with the meaning they have in dpuf_amd_sample; all but u may be
 * NULL (off). */
typedef struct {
    const float*   temperature;
    const int32_t* top_k;
    const float*   top_p;
    const float*   min_p;
    const float*   u;
} DpufAmdSampling;

/* dpuf_amd_engine_forward_argmax with the last row's token drawn by
 * dpuf_amd_sample (one entry of each setting) instead of its largest logit;
 * logprob_out (or NULL) its logarithmic share.  No Zone-A early exit, which
 * vouches for the largest logit alone.  Same return codes, -1 also without
 * sampling->u. */
DPUF_EXPORT int32_t dpuf_amd_engine_forward_sample(void* handle, int32_t n_tokens, const int32_t* token_ids,
                                                   int32_t pos0, const float* embeds_in, int32_t use_graph,
                                                   const DpufAmdSampling* sampling, int32_t* token_out,
                                                   float* logprob_out, float* logits_out);

/* dpuf_amd_engine_forward_slots with session i's token drawn from its logits
 * by entry i of the settings. */
DPUF_EXPORT int32_t dpuf_amd_engine_forward_slots_sample(void* handle, int32_t n, const int32_t* slot_ids,
                                                         const int32_t* token_ids, const int32_t* positions,
                                                         const DpufAmdSampling* sampling, float* logits_out,
                                                         int32_t* tokens_out, float* logprobs_out);

/* Gives the engine a KV cache of n_pages pages of page_size rows (2^30 rows at
 * most) per layer (type DPUF_AMD_BF16 or DPUF_AMD_F16; 2 x 2 x n_kv_heads x
 * head_dim bytes and 4 x n_kv_heads of weights per row and layer), next to its
 * slots, for dpuf_amd_engine_forward_pages; n_pages 0 frees it.  An earlier
 * one is replaced, its contents lost.  0 ok; -1 NULL handle, -2 a size out of range
 * or out of memory, -5 another type, or a rotation the config does not
 * describe, -6 device error. */
DPUF_EXPORT int32_t dpuf_amd_engine_pages_create(void* handle, int32_t n_pages, int32_t page_size, int32_t type);

/* Layer `layer`'s pages as the operators above take them.  0 ok, -1 no pages
 * or no such layer. */
DPUF_EXPORT int32_t dpuf_amd_engine_pages(void* handle, int32_t layer, DpufAmdPages* pages);

/* One forward pass over n sequences of any mix (prompts, chunks of prompts,
 * single tokens) on the engine's pages; host pointers.  Sequence i appends
 * rows[i] >= 1 tokens (token_ids: all sequences' one after the other, at most
 * DPUF_AMD_MAX_BATCH) whose rotary positions are positions[...] (any, not
 * bounded by max_seq_len); ctx_len[i] is its cached rows with them, in the
 * pages page_table[i * table_stride ...].  Which pages those are, and when
 * one is free, is the caller's affair: pages may be shared between sequences
 * as long as no new row goes into them and no weights are kept.  With
 * weight_decay >= 0 every cached row's weight becomes weight_decay times
 * itself plus the attention it receives in this pass (dpuf_amd_paged_attn_weights);
 * below 0 weights stay as they are.  Out, for each sequence's last row:
 * logits_out [n][V], and tokens_out [n] with logprobs_out [n] drawn by
 * sampling (tokens_out alone, the greedy token, when sampling is NULL); each
 * may be NULL, not all.  Attention runs on the pages' 16-bit type with fp32
 * sums, so results are close to, not bit-equal with, the slots'.
 * 0 ok; -1 NULL or contradicting arguments, no pages, a page used twice
 * where that is not allowed; -2 sizes; -3 a length or position out of range;
 * -4 a token id out of range; -6 device error. */
DPUF_EXPORT int32_t dpuf_amd_engine_forward_pages(void* handle, int32_t n, const int32_t* rows,
                                                  const int32_t* ctx_len, const int32_t* page_table,
                                                  int32_t table_stride, const int32_t* token_ids,
                                                  const int32_t* positions, float weight_decay,
                                                  const DpufAmdSampling* sampling, float* logits_out,
                                                  int32_t* tokens_out, float* logprobs_out);

/* The layers' sliding windows in dpuf_amd_engine_forward_pages and _score_pages
 * from now on, as in dpuf_amd_paged_attn_window: window [num_layers] (host), 0
 * for a layer that sees every cached row; NULL, or all 0, for none.  While any
 * layer has one, weight_decay has to be below 0, and where all have one, table
 * entries of pages that no new row sees in any layer may be anything.  0 ok; -1
 * NULL handle, -2 a window or sink outside 0 to 2^30. */
DPUF_EXPORT int32_t dpuf_amd_engine_pages_window(void* handle, const int32_t* window, int32_t sink);

/* dpuf_amd_engine_forward_pages whose every new row's logits are scored as
 * dpuf_amd_logprobs does, in the order of token_ids: with M rows in all, targets
 * [M][n_targets] (a prompt's next tokens, say) and logprobs_out of that size,
 * entropy_out [M], top_tokens_out and top_logprobs_out [M][n_top]; each may be
 * NULL (with a count of 0), not all three.  The cached rows' weights stay as they
 * are.  Codes as for dpuf_amd_engine_forward_pages, -2 also for the counts. */
DPUF_EXPORT int32_t dpuf_amd_engine_score_pages(void* handle, int32_t n, const int32_t* rows, const int32_t* ctx_len,
                                                const int32_t* page_table, int32_t table_stride,
                                                const int32_t* token_ids, const int32_t* positions, int32_t n_targets,
                                                const int32_t* targets, int32_t n_top, float* logprobs_out,
                                                float* entropy_out, int32_t* top_tokens_out, float* top_logprobs_out);

/* dpuf_amd_paged_evict on every layer of n sequences of the engine's pages
 * (host pointers): sequence i's min(ctx_len[i], keep) rows that stay go to the
 * pages dst_table[i * dst_stride ...], none of which any of the sequences
 * has, or has twice; new_len [n] receives the lengths.  Codes as for
 * dpuf_amd_engine_forward_pages. */
DPUF_EXPORT int32_t dpuf_amd_engine_evict_pages(void* handle, int32_t n, const int32_t* ctx_len,
                                                const int32_t* page_table, int32_t table_stride, int32_t keep,
                                                int32_t sink, int32_t recent, const int32_t* dst_table,
                                                int32_t dst_stride, int32_t* new_len);

#ifdef __cplusplus
}
#endif

#endif
