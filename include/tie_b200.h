/* tie_b200.h -- additive entry points of the B200 GPT-2 engine.
 *
 * Nothing here replaces a reference declaration; these are the additions that
 * the reference's single-sequence, host-logits API cannot express, listed in
 * the reference's own terms:
 *
 *   - a greedy step that keeps the logits on the device and returns only the
 *     argmax (the reference's greedy loop, src/main.c:274-287, copies a full
 *     vocabulary row to the host every step and scans it there);
 *   - batches of independent sequences sharing one model and one paged KV pool
 *     (the reference has exactly one sequence per model, src/model.c:216-245);
 *   - a whole greedy generation (prefill + every decode step) in one call, with
 *     the token ids staying on the device between steps;
 *   - access to the device and stream the model runs on, for callers that time
 *     or order work around it.
 *
 * All functions validate their arguments before launching any work and return
 * a model_status (include/model.h).
 */
#ifndef TIE_B200_TIE_H
#define TIE_B200_TIE_H

#include <stddef.h>
#include <stdint.h>

#include "model.h"

#ifdef __cplusplus
extern "C" {
#endif

/* model_load onto an explicit CUDA device ordinal (model_load uses the
 * calling thread's current device). */
model_status model_load_on_device(const char *weights_path, const char *inventory_path,
                                  const char *config_path, model_cproj_reading cproj_reading,
                                  int device, model **out);

/* The device ordinal and the cudaStream_t (as void*) every kernel of this model
 * is launched on. */
int   model_device(const model *m);
void *model_stream(const model *m);

/* Device bytes held by the weights (all layouts), and the number of kernels
 * this library has launched for the model since load (graph replays count each
 * node). */
size_t   model_weight_device_bytes(const model *m);
uint64_t model_kernel_launches(const model *m);

/* Cached decode step at context n_ids (same preconditions as
 * model_decode_step_cached) that returns only the greedy choice. */
model_status model_decode_step_greedy(model *m, const int32_t *ids, size_t n_ids, int32_t *next_id);

/* ---- batches of independent sequences --------------------------------------
 * model_batch_reserve sizes a paged KV pool and scratch for n_seq sequences of
 * up to `capacity` positions each (pages of KV_CACHE_PAGE_ROWS positions, page
 * tables on the device). It is separate from the single-sequence cache of
 * model_kv_reserve; the batch calls below use only the pool. Extends the
 * reference's kv_cache_create (src/kv_cache.c:150-190) to many sequences. */
model_status model_batch_reserve(model *m, size_t n_seq, size_t capacity);

/* The same pool over a bounded number of physical pages: n_pages pages of
 * KV_CACHE_PAGE_ROWS positions per layer (0: enough for every sequence's whole
 * capacity, which is what model_batch_reserve reserves), plus one scratch page.
 * No page belongs to a sequence until a batch call needs it: prefill assigns
 * the pages its prompt covers, each decode step the page its new position
 * opens, from a free list. A call that finds too few free pages returns
 * MODEL_ERR_CAPACITY before it launches the step (pages assigned by earlier
 * steps stay assigned). n_pages above n_seq * ceil(capacity / 16) is
 * MODEL_ERR_ARG. */
model_status model_batch_reserve_pages(model *m, size_t n_seq, size_t capacity, size_t n_pages);

/* Returns sequence `seq`'s pages to the pool's free list (a finished sequence,
 * so that others can grow into its pages). Its positions are then unmapped;
 * the next prefill that includes it assigns pages again. */
model_status model_batch_release(model *m, size_t seq);

/* Pages of the pool not assigned to any sequence (0 without a pool). */
size_t model_batch_free_pages(const model *m);

/* Prefill of n_seq sequences of n_ids tokens each (ids: host, n_seq * n_ids,
 * row-major). Writes every position's keys and values into the pool and sets
 * each sequence's length to n_ids. logits_out (host, n_seq * n_ids * vocab
 * floats, or NULL for none) receives all positions' logits; next_ids (host,
 * n_seq, or NULL) receives each sequence's greedy choice at its last position. */
model_status model_prefill_batch(model *m, const int32_t *ids, size_t n_seq, size_t n_ids,
                                 float *logits_out, size_t logits_cap, int32_t *next_ids);

/* One cached decode step for every sequence of the batch: token ids[s] is
 * appended at sequence s's current length, which then grows by one. logits_out
 * (host, n_seq * vocab floats, or NULL) and next_ids (host, n_seq, or NULL). */
model_status model_decode_step_batch(model *m, const int32_t *ids, size_t n_seq,
                                     float *logits_out, size_t logits_cap, int32_t *next_ids);

/* Greedy generation: prefill of n_prompt tokens for each of n_seq sequences,
 * then n_new greedy tokens each (n_new - 1 decode steps; the first new token
 * comes from the prefill's last row), all on the device. prompts: host,
 * n_seq * n_prompt; out_ids: host, n_seq * n_new. Requires a prior
 * model_batch_reserve covering n_seq sequences of n_prompt + n_new - 1
 * positions. The decode steps run as CUDA-graph replays. */
model_status model_generate_greedy(model *m, const int32_t *prompts, size_t n_seq,
                                   size_t n_prompt, size_t n_new, int32_t *out_ids);

/* Device-resident variant for timing the kernels alone: prompts and out_ids are
 * DEVICE buffers of the same shapes; no host copies, no synchronisation. */
model_status model_generate_greedy_device(model *m, const int32_t *d_prompts, size_t n_seq,
                                          size_t n_prompt, size_t n_new, int32_t *d_out_ids);

/* Appends n_ids tokens to each of the pool's sequences 0 .. n_seq - 1 behind
 * the positions it holds (ids: host, n_seq * n_ids, row-major): a prompt in
 * pieces, the next turn of a conversation, tokens to be scored. The new tokens
 * attend to everything cached and to one another, causally; their keys and
 * values go into the pool and its length grows by n_ids. As for
 * model_prefill_batch, logits_out (host, n_seq * n_ids * vocab floats, or NULL)
 * receives the new positions' logits and next_ids (host, n_seq, or NULL) each
 * sequence's greedy choice at its last position. A sequence that does not hold
 * the pool's length (never prefilled to it, released, or overwritten by a call
 * that failed) is MODEL_ERR_ARG. Attention statistics (model_collect_attn_stats)
 * do not cover this call. At most 4096 sequences. */
model_status model_extend_batch(model *m, const int32_t *ids, size_t n_seq, size_t n_ids,
                                float *logits_out, size_t logits_cap, int32_t *next_ids);

/* Beam search: for each of n_req (<= 4096) prompts of n_prompt tokens (host, n_req *
 * n_prompt) the `beams` (<= 16) continuations of n_new tokens that one beam
 * search step after the other keeps (tie_beam_select: largest sum of log
 * probabilities, ties to the lowest beam and token). A continuation that has
 * produced eos_id is kept with its score, filled up with eos_id; eos_id < 0:
 * none. out_ids (host, n_req * beams * n_new) and out_scores (host, n_req *
 * beams): each request's continuations, best first. Requires a prior
 * model_batch_reserve covering n_req * beams sequences of n_prompt + n_new - 1
 * positions. The pool then holds the continuations in the order of out_ids, all
 * but their last tokens: sequence r * beams + i is request r's prompt and its
 * i-th best continuation, ready for model_decode_step_batch on the last tokens. */
model_status model_generate_beam(model *m, const int32_t *prompts, size_t n_req, size_t n_prompt,
                                 size_t beams, size_t n_new, int32_t eos_id, int32_t *out_ids,
                                 float *out_scores);

/* ---- diagnostics --------------------------------------------------------
 * Times `iters` back-to-back launches of one kernel of the forward pass, alone,
 * on the model's stream with CUDA events, and stores the average milliseconds
 * per launch (the numbers a roofline is computed from). It runs on the batch
 * pool and scratch of model_batch_reserve, which must cover `rows` sequences of
 * `context` positions, and overwrites their contents and the decode state.
 *   TIE_KERNEL_DECODE_ATTENTION  one layer's decode attention (split + merge),
 *                                `rows` sequences at context `context`
 *   TIE_KERNEL_DECODE_QKV        the QKV matmul of a decode step, `rows` rows
 *   TIE_KERNEL_DECODE_FC         the MLP up-projection (+ GELU) of a decode step
 *   TIE_KERNEL_DECODE_MLP_PROJ   the MLP down-projection (+ residual)
 *   TIE_KERNEL_DECODE_HEAD       the tied head with its fused argmax
 *   TIE_KERNEL_PREFILL_ATTENTION causal attention over `context` tokens x `rows`
 *   TIE_KERNEL_PREFILL_FC        the MLP up-projection over rows * context tokens
 *   TIE_KERNEL_DECODE_STEP       one whole decode step of `rows` (<= 4) sequences
 *                                at context `context` as the persistent kernel */
enum {
    TIE_KERNEL_DECODE_ATTENTION = 0,
    TIE_KERNEL_DECODE_QKV = 1,
    TIE_KERNEL_DECODE_FC = 2,
    TIE_KERNEL_DECODE_MLP_PROJ = 3,
    TIE_KERNEL_DECODE_HEAD = 4,
    TIE_KERNEL_PREFILL_ATTENTION = 5,
    TIE_KERNEL_PREFILL_FC = 6,
    TIE_KERNEL_DECODE_STEP = 7
};
model_status model_time_kernel(model *m, int kernel, size_t rows, size_t context, int iters,
                               float *avg_ms);

/* ---- weight formats --------------------------------------------------------
 * The reference computes in fp32 only. These formats trade weight precision
 * for HBM traffic in the memory-bound decode:
 *   TIE_WEIGHTS_F32   the loaded weights (the default).
 *   TIE_WEIGHTS_BF16  each matrix element rounded to nearest-even bf16.
 *   TIE_WEIGHTS_INT8  per output channel (a row of each [out, in] matrix):
 *                     scale = absmax(row) / 127 in fp32, q = rint(w / scale)
 *                     (ties to even) clamped to +-127; the weight is q * scale.
 * The formats apply to the five matrix kinds -- qkv, attention proj, fc, mlp
 * proj, and the tied wte (head and embedding lookup alike); LayerNorm, biases
 * and wpe stay fp32. Accumulation is fp32 throughout. Decode steps of at most
 * 8 sequences stream the compact copies (2 or 1 byte per element); every other
 * path computes with the fp32 values the copies stand for, so the model is the
 * same model whichever kernels run. A format's copies are built on the device
 * on first selection and kept. */
enum { TIE_WEIGHTS_F32 = 0, TIE_WEIGHTS_BF16 = 1, TIE_WEIGHTS_INT8 = 2 };
model_status model_set_weight_format(model *m, int fmt);
int model_weight_format(const model *m);

/* The last CUDA failure behind a MODEL_ERR_DEVICE on the calling thread: the
 * error's name and text and the failing call, or "" if none yet. With the
 * environment variable TIE_DEBUG set, each such failure is also printed to
 * stderr. */
const char *tie_last_device_error(void);

/* The causal prefill attention of the engine (model.c:705-732, the step
 * between the QKV projection and the output projection) over HOST arrays, for
 * tests of the kernel alone: qkv is n_seq x T rows of 3 * n_head * 64 floats
 * (q, k, v of every head, the layout of the fused projection's output) and out
 * receives n_seq x T rows of n_head * 64. Runs on the current device; returns
 * MODEL_ERR_ARG for a null pointer or a non-positive size, MODEL_ERR_DEVICE on
 * a CUDA failure or an expired wait. */
model_status tie_attention_prefill(const float *qkv, int n_seq, int T, int n_head, float *out);

/* ---- how small decode steps run ------------------------------------------
 * A decode step of at most 8 sequences runs as a chain of per-layer kernels
 * linked by programmatic dependent launch: TIE_STEP_CHAINED, the default
 * (LayerNorm, QKV + the step's K/V rows, attention, projection + residual,
 * LayerNorm, FC + GELU, MLP projection + residual; each matmul's weights are
 * loaded into registers ahead of its dependency wait). TIE_STEP_STREAM runs
 * the same arithmetic as five kernels per layer: the weights are bulk-copied
 * into shared memory ahead of the wait, and LayerNorm, the embedding lookup
 * and the merge of attention chunk partials run in the matmuls' prologues. With
 * TIE_STEP_PERSISTENT a step of at most 4 sequences (fp32 weights, without
 * attention statistics) runs as ONE persistent kernel. All three form every
 * sum in the same order, so they return identical logits and tokens; the
 * switch exists to compare and time them. MODEL_ERR_ARG for any other value. */
enum { TIE_STEP_PERSISTENT = 0, TIE_STEP_CHAINED = 1, TIE_STEP_STREAM = 2 };

/* Failure drill for the bounded waits: the next decode step that runs on the
 * default chained path (at most 8 sequences, no attention statistics) has its
 * first matmul wait on a shared-memory barrier that nothing completes. The
 * wait gives up after limit_ns nanoseconds, the kernel records the expiry in
 * the model's device error flag and returns, and the step's call returns
 * MODEL_ERR_DEVICE with the cache length unchanged; the next step runs
 * normally. Every bounded wait of the engine's kernels reports through the
 * same flag. MODEL_ERR_ARG for a NULL model or a zero limit. No counterpart in
 * the reference (its CPU engine has no device waits). */
model_status model_debug_wait_drill(model *m, uint64_t limit_ns);

/* Trace of one decode step of `rows` (<= 8) sequences at context `context` on
 * the TIE_STEP_STREAM path (the batch pool must cover them; contents are
 * overwritten as for model_time_kernel): for each of its 4 * n_layer + 1
 * streaming matmul kernels in launch order, *per_kernel global-timer stamps
 * (ns) -- 256 CTA slots of 8 events: entry, dependency wait over, input rows
 * built, first weights landed, last stage done, exit, producer done (0 where
 * no CTA ran) -- written to out (host, cap >= *per_kernel * *n_kernels;
 * *per_kernel and *n_kernels are set even when the capacity is short, which
 * returns MODEL_ERR_CAPACITY). MODEL_ERR_ARG when the step would not take that
 * path. No counterpart in the reference. */
model_status model_stream_trace(model *m, size_t rows, size_t context, uint64_t *out, size_t cap,
                                size_t *per_kernel, size_t *n_kernels);

model_status model_set_step_kernel(model *m, int kind);

/* Trace of one persistent decode step of `rows` (<= 4) sequences at context
 * `context` on the batch pool (model_batch_reserve must cover them; contents
 * are overwritten as for model_time_kernel): per CTA, *per_cta global-timer
 * stamps in nanoseconds, *n_cta CTAs, written to out (host, cap >= per_cta *
 * n_cta, else MODEL_ERR_CAPACITY after filling the two counts). Stamp order per
 * CTA: [0] start; [1 + 3 * (5 * layer + stage) + k] for stage 0..4 (LN1+qkv,
 * attention, proj, LN2+fc, mlp) with k = 0 inputs ready, 1 rows staged, 2 done,
 * the head as stage 5 * n_layer; then the CTA's end; then, per weight matrix in
 * stream order (qkv, proj, fc, mlp per layer, then wte), when its last copy was
 * issued. */
model_status model_step_trace(model *m, size_t rows, size_t context, uint64_t *out, size_t cap,
                              size_t *per_cta, size_t *n_cta);

/* ---- the greedy head without allocation --------------------------------
 * No counterpart in the reference (its head is a CPU matmul over host memory).
 * For callers that cannot allocate device memory -- a serving framework whose
 * caching allocator already holds the GPU's memory, a plugin inside a runtime
 * that forbids allocations outside its own allocator, a latency-bound loop that
 * cannot take cudaMalloc's implicit device synchronisation.
 *
 * next[r] = argmax_j (x[r] . w[j]) for r < rows (lowest index on ties), and,
 * when `logits` is non-NULL, logits[r * ldl + j] = x[r] . w[j]. x (rows x k,
 * leading dimension ldx), w (vocab x k, ldw), logits and next are DEVICE
 * pointers; x and w 16-byte aligned, k, ldx and ldw multiples of 4. Work is
 * enqueued on `stream` (a cudaStream_t; NULL for the legacy default stream)
 * and not waited for.
 *
 * Limits: rows <= 16 and vocab <= 65536, else MODEL_ERR_CAPACITY. The per-block
 * partial maxima live in a fixed 512 KiB array inside the library, present on
 * every GPU that loads it until the process exits; nothing is allocated per
 * call. The array's device address is looked up on the first call made on each
 * device (with that device current); make that first call before any stream
 * capture. Every call shares the array, so calls that overlap on the GPU race
 * on it. */
model_status tie_head_argmax_noalloc(const float *x, int ldx, const float *w, int ldw, int rows,
                                     int vocab, int k, float *logits, int ldl, int32_t *next,
                                     void *stream);

/* ---- the paged cache and beams, over device memory -----------------------
 * No counterpart in the reference (one sequence, one contiguous cache:
 * src/kv_cache.c:150-190, src/model.c:826-850). For a caller that schedules
 * its own batches: pages are built, filled, attended to and reordered on the
 * GPU, without a copy of the lengths to the host.
 *
 * A pool is two arrays (keys, values) of n_pages pages of KV_CACHE_PAGE_ROWS
 * rows of n_kv_head * 64 elements, fp32 (TIE_KV_F32) or bf16 (TIE_KV_BF16),
 * contiguous. A page table has pages_per_seq int32 entries per sequence; an
 * entry outside [0, n_pages) is unmapped. A slot is page * KV_CACHE_PAGE_ROWS
 * + row, or -1 for none. New tokens of a batch form rows: those of sequence s
 * are row_start[s] .. row_start[s + 1] - 1, at positions ctx_lens[s], ...
 *
 * Pointers are DEVICE pointers of one device (made current for the call) and
 * `stream` a cudaStream_t of it (NULL: the legacy default stream); work is
 * enqueued and not waited for. Activations, workspaces and pages are 16-byte aligned
 * (pages that attention reads 32-byte), leading dimensions multiples of 4 floats. A workspace holds nothing
 * from one call to the next, but two calls that overlap on the GPU (streams,
 * replayed graphs) need one each. Nothing is allocated, and every call may be
 * captured into a graph. MODEL_ERR_ARG for a null or misaligned pointer, a
 * shape or format without meaning, or host memory; MODEL_ERR_CAPACITY for a
 * workspace too small or a limit below; MODEL_ERR_DEVICE for a CUDA failure.
 * Limits: 4096 sequences or requests, 2^27 pages (2^26 per sequence), 16 beams,
 * 2^30 logits a row. */
enum {
    TIE_KV_F32 = 0,
    TIE_KV_BF16 = 1,
    TIE_KV_INT8 = 2   /* pages with scales: the entry points that take scales */
};

/* Page table entries, row starts and slot maps from request lengths. Sequence
 * s has ctx_lens[s] positions cached and appends new_lens[s] (>= 0). Its
 * entries for the pages that start among the new positions are assigned from
 * the free list, a stack of max_free entries of which n_free[0] count: entry
 * n_free - 1 first, in the order of sequences and positions, as the engine's
 * own pool does. n_free_out[0] receives what is left (it may be n_free).
 * Without a free list (free_pages, n_free, n_free_out NULL) the table is taken
 * as complete; an empty one (max_free 0) needs no free_pages.
 * row_start[n_seq + 1] receives the row starts; seq_of, pos_of, slot_of
 * [max_rows] each row's sequence, position and slot (-1 where that entry is
 * unmapped), and -1 for rows behind the last sequence's.
 * status[0] receives MODEL_OK; MODEL_ERR_CAPACITY for too few free pages, a
 * sequence beyond pages_per_seq pages or more than max_rows rows; or
 * MODEL_ERR_ARG for a negative length or an n_free outside 0..max_free. With
 * either error nothing is assigned, row_start is 0 throughout and every row is
 * -1, so what follows in the stream does nothing. */
model_status tie_page_plan(const int32_t *ctx_lens, const int32_t *new_lens, int n_seq,
                           int32_t *page_table, int pages_per_seq, int n_pages,
                           const int32_t *free_pages, int max_free, const int32_t *n_free,
                           int32_t *n_free_out, int32_t *row_start, int32_t *seq_of,
                           int32_t *pos_of, int32_t *slot_of, int max_rows, int32_t *status,
                           void *stream);

/* Key and value rows into their slots: row r of k and v (n_kv_head * 64 floats,
 * ld floats apart) to slot slots[r] of the pool, rounded to nearest even for
 * bf16. A slot outside the pool stores nothing; of rows with one slot each
 * element is one or another's (which, may differ from element to element and
 * between keys and values). rows == 0 is allowed (k, v and slots may be NULL
 * then). */
model_status tie_kv_store(const float *k, const float *v, int ld, const int32_t *slots, int rows,
                          void *k_pages, void *v_pages, int kv_format, int n_pages, int n_kv_head,
                          void *stream);

/* Causal attention of new tokens over the cache that holds them: for row r of
 * sequence s at position p and query head h (n_head of them, a multiple of
 * n_kv_head; K/V head h / (n_head / n_kv_head)),
 *   out[r][h] = sum_j softmax_j(scale * q[r][h] . k[j]) v[j],  0 <= j <= p,
 * over the positions whose page is mapped; 0 where none is left. The new
 * tokens' own keys and values are read from the pages (tie_kv_store first).
 * q and out: `rows` rows of n_head * 64 floats, ldq and ldo apart, not
 * overlapping (rows == 0: nothing to do, q and out may be NULL). max_new bounds
 * the new tokens per sequence. A sequence without new tokens, with more than
 * max_new, with row_start outside 0..rows or beyond pages_per_seq pages is left
 * out: its rows of out stay as they were, and so do rows behind the last
 * sequence's. Sums and softmax statistics are fp32.
 * Operands of many rows are held in 22 bits of the largest element of their
 * query, of their 16 keys or of their 16 values (an element below 2^-17 of it
 * to 2^-40 of it), and values to 2^-106 at the least.
 * A value that is not finite makes the rows that see it not finite, a key that
 * is not finite may, and neither does it to any other row. The result of a row
 * depends, in its rounding, on how the batch splits its keys, and is the same
 * for the same call.
 * status, if not NULL, receives MODEL_ERR_DEVICE when a bounded wait in the
 * kernel expires (the output is then incomplete, and nothing else tells); it is
 * not written otherwise. */
size_t tie_attention_paged_workspace(void);
model_status tie_attention_paged(const float *q, int ldq, int n_head, const void *k_pages,
                                 const void *v_pages, int kv_format, int n_pages, int n_kv_head,
                                 const int32_t *page_table, int pages_per_seq,
                                 const int32_t *row_start, const int32_t *ctx_lens, int n_seq,
                                 int max_new, int rows, float scale, float *out, int ldo,
                                 void *workspace, size_t workspace_bytes, int32_t *status,
                                 void *stream);

/* One step of beam search. Row r * beams + b of logits (ldl floats apart) and
 * scores belongs to beam b of request r. A candidate (b, v) has the total
 *   scores[b] + logits[b][v] - logsumexp(logits[b]),
 * formed in double; a finished beam (done != 0; done may be NULL) has the one
 * candidate (b, eos_id) with its score unchanged. The `beams` largest totals
 * are kept, the lowest b * vocab + v first among equal ones (within one beam
 * logits are compared as they are). A NaN logit counts as -inf; a total that
 * is NaN counts as -inf, as do all of a row whose largest logit is infinite.
 * Places: a beam's best kept candidate stays in that beam's place; the others
 * take the places left, lowest first, best first. So a beam that has children
 * is its own first child, and tie_kv_reorder moves no row that others copy.
 * Per place: next (token), parent (row index r * beams + b), scores_out (may
 * be scores), done_out (may be done, may be NULL: parent finished, or token ==
 * eos_id). eos_id < 0: none, then done and done_out must be NULL. */
size_t tie_beam_select_workspace(int n_req, int beams, int vocab);
model_status tie_beam_select(const float *logits, int ldl, const float *scores,
                             const int32_t *done, int n_req, int beams, int vocab, int eos_id,
                             int32_t *next, int32_t *parent, float *scores_out, int32_t *done_out,
                             void *workspace, size_t workspace_bytes, void *stream);

/* The cached rows follow the beams: for every layer (layer_stride elements
 * apart in each of k_pages and v_pages) and every sequence s = r * beams + b
 * whose parent[s] is another beam of request r, the rows of positions first[r]
 * .. length[r] - 1 of s's pages become those of the parent's, as they were
 * before the call (any permutation). Positions before first[r] are taken to be
 * equal in all beams of the request (the prompt); pages that hold later ones
 * belong to one beam each. A parent outside the request, an unmapped page and
 * a page that both beams share move nothing. */
model_status tie_kv_reorder(void *k_pages, void *v_pages, int kv_format, int n_layer,
                            size_t layer_stride, int n_pages, int n_kv_head,
                            const int32_t *page_table, int pages_per_seq, const int32_t *parent,
                            const int32_t *first, const int32_t *length, int n_req, int beams,
                            void *stream);

/* ---- the cache in 8 bits --------------------------------------------------
 * A pool in 8 bits (TIE_KV_INT8) is, for keys and for values, n_pages pages of
 * KV_CACHE_PAGE_ROWS rows of n_kv_head * 64 int8 levels, and a scale per row and
 * head: fp32 [n_pages][n_kv_head][KV_CACHE_PAGE_ROWS]. An element is level *
 * scale; scale = max |x| / 127 of the head's 64 elements, level = x / scale to
 * the nearest integer, ties to even (of the exact quotient), 0 where the scale
 * is 0. A head's row with an element that is not finite gets a scale that is NaN
 * and levels 0. Pointers, streams and errors are those of the paged cache above;
 * rows * n_kv_head is below 2^31 (MODEL_ERR_CAPACITY). */

/* tie_kv_store into a pool in 8 bits. Rows with one slot leave levels and scales there that
 * may be of different ones: a slot is given once. */
model_status tie_kv_store_q8(const float *k, const float *v, int ld, const int32_t *slots, int rows,
                             void *k_pages, void *v_pages, float *k_scales, float *v_scales,
                             int n_pages, int n_kv_head, void *stream);

/* Rows of a pool of any format read back: row r of k and v (n_kv_head * 64
 * floats, ld floats apart) receives what slot slots[r] holds. A slot outside the
 * pool leaves its row as it was; a slot may be read by any number of rows.
 * k_scales and v_scales: those of TIE_KV_INT8, NULL for the other formats.
 * rows == 0 is allowed (k, v and slots may be NULL then). */
model_status tie_kv_load(const int32_t *slots, int rows, const void *k_pages, const void *v_pages,
                         const float *k_scales, const float *v_scales, int kv_format, int n_pages,
                         int n_kv_head, float *k, float *v, int ld, void *stream);

/* Attention of new tokens over their sequences' own pages and over pages that
 * groups of sequences share: beams and answers of one prompt, requests behind one
 * instruction. Group g is sequences group_start[g] .. group_start[g + 1] - 1
 * (group_start[n_group + 1], ascending); its first prefix_lens[g] positions lie in
 * the pages of prefix_table (n_group rows of pages_per_prefix entries). They are read for 8 to 32 of
 * its rows (tokens times query heads of a K/V head) together, or, where a group has 64 rows and more in the
 * mean and the products of rows and pages_per_prefix are many, by the tensor cores for 128. (The arguments
 * decide, not the lengths on the device: a table far wider than its prefixes, or one large group among many
 * small ones, may be better served by a table or a call of its own.) A sequence's own pages
 * (page_table, ctx_lens) hold what comes behind them, from a page's first row on. For row r of sequence s, its new
 * token i, and query head h,
 *   out[r][h] = sum_j softmax_j(scale * q[r][h] . k[j]) v[j]
 * over the group's shared positions and the sequence's own positions 0 ..
 * ctx_lens[s] + i whose page is mapped; 0 where none is left. A sequence in no
 * group has its own positions only, and so have those of a group whose range or
 * length has no meaning (outside 0..n_seq or pages_per_prefix pages). n_group 0:
 * no groups (prefix_table, prefix_lens and group_start NULL). kv_format may be
 * TIE_KV_INT8, with the pool's scales (NULL for the others).
 * All else is as for tie_attention_paged: rows, limits, what is left out, what is
 * not finite, and status. It is set where a wait of a long prefix's kernel ran out (2 s) and may
 * be NULL; rows whose shared positions were not finished then are NaN, the others as always. Sums
 * and softmax statistics are fp32. Over fp32 and bf16 pages products are of all of their operands' 24
 * bits. Over pages in 8 bits a row's scaled query is held
 * in 24 bits relative to its largest element (to 2^-126), and the products of a step
 * of 32 keys' weights (at most 1) with their values' scales in 23 bits relative to the
 * largest of the step (to 2^-95); its products with a key's levels are summed before the key's scale, so
 * such a sum has to be finite in fp32 too. The result of a row depends, in its rounding, on how
 * the batch splits its keys, and is the same for the same call. Where group_start does
 * not ascend, rows of a sequence in two groups' ranges hold no particular result.
 * workspace: tie_attention_shared_workspace(rows, n_head) bytes (on the current
 * device) or more. */
size_t tie_attention_shared_workspace(int rows, int n_head);

/* The failure drill of it: in the calling thread's next tie_attention_shared with a prefix long enough for
 * the tensor cores, waits last limit_ns (1 to 2,000,000,000) at most, and half of that kernel's CTAs
 * wait for what does not come. So a test sees NaN, MODEL_ERR_DEVICE in status, and then a clean next call. */
model_status tie_attention_shared_wait_drill(uint64_t limit_ns);
model_status tie_attention_shared(const float *q, int ldq, int n_head, const void *k_pages,
                                  const void *v_pages, const float *k_scales,
                                  const float *v_scales, int kv_format, int n_pages, int n_kv_head,
                                  const int32_t *page_table, int pages_per_seq,
                                  const int32_t *row_start, const int32_t *ctx_lens, int n_seq,
                                  int max_new, int rows, const int32_t *prefix_table,
                                  int pages_per_prefix, const int32_t *prefix_lens,
                                  const int32_t *group_start, int n_group, float scale, float *out,
                                  int ldo, void *workspace, size_t workspace_bytes,
                                  int32_t *status, void *stream);

/* ---- 4-bit weights --------------------------------------------------------
 * A weight matrix W of n rows (outputs) of k weights, cut along k into groups of
 * 32, 64 or 128. A group has a scale = max |w| / 7 in fp32, rounded to bf16, and
 * levels -7 .. 7 = w / scale to the nearest integer, ties to even (of the exact
 * quotient); a weight is level * scale. A group with a weight that is not finite
 * gets a scale that is NaN and levels 0, one whose scale is 0 levels 0.
 * packed: tie_q4_bytes(n, k) bytes, 16-byte aligned; a row is blocks of 128
 * weights in 64 bytes, the last one filled up with zeros. The 32-bit word 4 t + j
 * of a block (t, j = 0 .. 3) holds its weights 32 j + 8 t + i, i = 0 .. 7, as
 * level + 8 in bits 4 i .. 4 i + 3. scales: bf16 [n][ceil(k / group)].
 * Pointers are DEVICE pointers of one device; any k and leading dimension is
 * taken (fp32 rows that are 16-byte aligned are read faster). Streams and errors
 * are those of the paged cache above; MODEL_ERR_CAPACITY for k above 2^24 or more
 * than 2^31 - 1 blocks of 128 weights. */

/* Bytes of the packed levels (0 for sizes without meaning). */
size_t tie_q4_bytes(int n, int k);

/* fp32 weights (ldw floats from row to row) to levels and scales, and back. */
model_status tie_quantize_q4(const float *w, long long ldw, int n, int k, int group, void *packed,
                             void *scales, void *stream);
model_status tie_dequantize_q4(const void *packed, const void *scales, int n, int k, int group,
                               float *w, long long ldw, void *stream);

/* y[r] = act(x[r] W^T + bias) + residual[r] for `rows` rows of activations (ldx,
 * ldr, ldy floats apart): the matmul of a decode step with its epilogue (the
 * bias, GELU and residual forms of model.c:735-752). bias [n] and residual may be
 * NULL; gelu 1: act is GELU (model.c:615-623), 0: none. residual may be y itself, x
 * must not overlap y. An activation is held to 2^-30 of the largest of its 128
 * columns (and to 2^-128), its products with levels and their sums over a group are
 * exact, sums over groups fp32. A row's result does not depend on the rows beside
 * it, except by their number being above 2; a row with an element that is not finite
 * is not finite. The weights are read once for every 8 rows (every 2, where k is
 * above 6,400, 6,784 or 6,912 for groups of 32, 64 or 128). rows == 0 is allowed (x and y may be NULL then); at most 16,384
 * columns and 131,070 rows (MODEL_ERR_CAPACITY). */
model_status tie_matvec_q4(const float *x, long long ldx, int rows, const void *packed,
                           const void *scales, int n, int k, int group, const float *bias,
                           const float *residual, long long ldr, int gelu, float *y, long long ldy,
                           void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TIE_B200_TIE_H */
