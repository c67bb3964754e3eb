/*
 * rtr_b200.h - C ABI of the B200-native semantic-ID beam-search engine.
 *
 * One session = one model replica on one GPU serving sequential requests
 * (batch 1, 50 beams, 3 SID tokens + newline + EOS), which is how the
 * reference runs (rapidtinyrec/benchmark_inference.py:62-258; one model, one
 * stream, one isolated worker: docs/release-scope.md:41-44).
 *
 * Conventions
 *   - Every entry point returns an int status: RTR_OK (0) or an RTR_ERR_*
 *     code.  No exception crosses the ABI.  rtr_last_error() gives the text.
 *   - RTR_ERR_ARG mirrors the reference's ValueError (shape, capacity,
 *     aliasing: shared_prefix.py:71-73, prefix_replay.py:99-101);
 *     RTR_ERR_STATE its RuntimeError (call order, frozen pools:
 *     decode_replay.py:185, inference_precision.py:53-54).
 *   - Pointers are plain host or device addresses; sizes are element counts.
 *     "dev" parameters must be device memory of the session's GPU; "host"
 *     parameters are host memory (pinned memory makes the copies async).
 *   - The caller owns every buffer it passes; the session owns its device
 *     state (weights, constraint tables, prefix arena, beam state).
 *   - A session is not thread-safe; use one session per GPU per process.
 *     All device work is issued on the session's stream (rtr_set_stream).
 */
#ifndef RTR_B200_H
#define RTR_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RTR_OK 0
#define RTR_ERR_ARG 1     /* invalid argument, shape or capacity          */
#define RTR_ERR_STATE 2   /* wrong call order / missing weights or tables */
#define RTR_ERR_CUDA 3    /* CUDA runtime error                           */
#define RTR_ERR_DEVICE 4  /* a device-side check failed (see message)     */

#define RTR_DTYPE_F32 0
#define RTR_DTYPE_BF16 1

#define RTR_NUM_STEPS 5   /* prefill output + 4 decode forwards */

typedef struct rtr_session rtr_session;

/* Model shape.  Mirrors the Qwen2 config fields the reference reads from the
 * release (benchmark_inference.py:93-98) plus the runtime capacities of the
 * prefix arena (shared_prefix.py:53-65). */
typedef struct {
  int32_t layers, hidden, heads, kv_heads, head_dim, intermediate, vocab;
  int32_t tied_embeddings;  /* lm_head shares the embedding matrix */
  float rms_eps;
  float rope_theta;
  int32_t dtype;            /* RTR_DTYPE_F32 / RTR_DTYPE_BF16: weights, activations, KV */
  int32_t max_prefix;       /* prefix arena capacity in tokens (PrefixArena max_prefix_tokens) */
  int32_t num_beams;        /* 50 in the reference (benchmark_inference.py:139) */
} rtr_model_config;

/* Dense SID constraint tables, int32 copies of GpuSidConstraintTables
 * (gpu_constraints.py:31-60): offsets/sizes of the three SID levels, the
 * step-1 table [sizes[0] x width1], the step-2 table
 * [sizes[0]*sizes[1] x width2] (rows padded by repeating their first token),
 * the validity bitmap over sizes[0]*sizes[1]*sizes[2] (one byte each), the
 * root prefix and the sorted first tokens.  All pointers are host memory. */
typedef struct {
  int32_t offsets[3], sizes[3];
  const int32_t* table1; int32_t width1;
  const int32_t* table2; int32_t width2;
  const uint8_t* valid;
  int32_t root[3];
  const int32_t* first_tokens; int32_t n_first;
  int32_t newline, eos;
} rtr_constraint_tables;

/* Per-request result, host buffers sized by num_beams B (the reference's
 * per-user record, benchmark_inference.py:150-154 / 241-244):
 *   token_ids[B*5]       generated tokens of the ranked beams (int32)
 *   beam_indices[B*5]    parent beam row at every step
 *   sequence_logp[B]     FP32 sequence scores (sequences_scores)
 *   transition_logp[B*5] FP32 per-step scores (compute_transition_scores)  */
typedef struct {
  int32_t* token_ids;
  int32_t* beam_indices;
  float* sequence_logp;
  float* transition_logp;
} rtr_result;

/* ---- session lifecycle -------------------------------------------------- */

/* Replaces the model/compiler/arena/pool set-up of
 * benchmark_inference.py:93-121 (CompiledForward, PrefixArena,
 * PrefixReplayPool, ReorderSuffix).  Allocates all device state. */
int rtr_session_create(const rtr_model_config* cfg, int device, rtr_session** out);
/* The same session sized for up to max_users (1..8) users per request: each
 * user gets its own prefix arena, beam state and result; rtr_launch_batch runs
 * their decode steps together (no reference counterpart: the reference serves
 * one user per request). */
int rtr_session_create_batched(const rtr_model_config* cfg, int device, int32_t max_users, rtr_session** out);
int rtr_session_destroy(rtr_session* s);

/* Text of the last error of this session (when s is NULL: of this thread's last
 * failed call without a session).  Valid until the next call on the session. */
const char* rtr_last_error(const rtr_session* s);

/* Issue all work of the session on this cudaStream_t (NULL = session-owned
 * stream).  Invalidates captured graphs. */
int rtr_set_stream(rtr_session* s, void* stream);

/* Load weights in the canonical Qwen2 order: embed [V,H]; per layer
 * q_w [Hq*D,H], q_b, k_w [Hkv*D,H], k_b, v_w, v_b, o_w [H,Hq*D],
 * gate_w [I,H], up_w [I,H], down_w [H,I], input_norm [H], post_norm [H];
 * final_norm [H]; lm_head [V,H] unless tied.  n_tensors = 1 + 12*layers + 1
 * (+1 untied).  src_dtype is the element type of the given tensors
 * (converted with round-to-nearest-even when it differs from the session
 * dtype); src_on_device selects device or host pointers.
 * Replaces from_pretrained(...).to('cuda') (benchmark_inference.py:93-98). */
int rtr_load_weights(rtr_session* s, const void* const* tensors, int32_t n_tensors,
                     int32_t src_dtype, int32_t src_on_device);

/* RoPE cos/sin tables [n_positions, head_dim/2] float32, host memory
 * (Qwen2RotaryEmbedding, transformers modeling_qwen2.py:89-113).  Optional:
 * without it the session computes them on the host in double precision. */
int rtr_load_rope(rtr_session* s, const float* cos_host, const float* sin_host, int32_t n_positions);

/* Upload the constraint tables.  Replaces GpuSidConstraintTables(...,
 * device='cuda') (gpu_constraints.py:18-67, benchmark_inference.py:92). */
int rtr_load_constraints(rtr_session* s, const rtr_constraint_tables* t);

/* ---- one request ---------------------------------------------------------- */

/* Prefill one request of L tokens into the single shared prefix copy and run
 * step 0 (normalisation, mask, beam top-k).  ids may be host or device
 * (ids_on_device).  Replaces PrefillPrefix.forward + PrefixArena.start_request
 * + the first _beam_search iteration (prefix_prefill.py:27-63,
 * shared_prefix.py:67-89). */
int rtr_prefill(rtr_session* s, const int32_t* ids, int32_t L, int32_t ids_on_device);

/* Decode step t in 1..4: 50-row forward over the shared prefix and the beams'
 * suffixes, full-vocabulary double log-softmax, trie mask, beam top-k and the
 * suffix parent gather, all on device without a host round trip.  Replaces
 * one _beam_search iteration with PrefixReplayPool.__call__,
 * GpuSidConstrainedLogitsProcessor.__call__ and ReorderSuffix.reorder
 * (decode_replay.py:180-191, gpu_constraints.py:95-101,
 * prefix_replay.py:95-117). */
int rtr_decode_step(rtr_session* s, int32_t t);

/* Copy the finished ranking to host buffers (blocking on the stream).  Fails
 * with RTR_ERR_DEVICE when the beam loop would not have stopped after five
 * steps or a device-side bound check fired.  Replaces unpack
 * (benchmark_inference.py:150-154). */
int rtr_read_results(rtr_session* s, const rtr_result* out);

/* Whole request: prefill + steps 1..4 (one CUDA graph) + result copy.
 * Replaces benchmark_inference.generate (:123-148). */
int rtr_generate(rtr_session* s, const int32_t* ids_host, int32_t L, const rtr_result* out);

/* Batched requests (sessions from rtr_session_create_batched): n_users prompts
 * ids[u] of lengths L[u]; every user's prefill runs on its own, then one decode
 * graph runs steps 1-4 for all n users, each projection GEMM at n x beams rows.
 * Each user's ranking equals its batch-1 result (same kernels and, up to two
 * users, the same split-K partition; beyond that the GEMM partition can change
 * the last bits).  out points to n_users results.  One status word covers the
 * batch: a device check that fails for one user fails the batch. */
int rtr_launch_batch(rtr_session* s, const int32_t* const* ids, const int32_t* L, int32_t n_users,
                     int32_t ids_on_device);
int rtr_wait_batch(rtr_session* s, const rtr_result* out);
int rtr_generate_batch(rtr_session* s, const int32_t* const* ids_host, const int32_t* L, int32_t n_users,
                       const rtr_result* out);

/* The two halves of rtr_generate for callers that overlap requests with host
 * work: rtr_launch enqueues prefill + the decode graph + the result copy on the
 * session stream and returns without waiting (ids host or device);
 * rtr_wait blocks until the last launched request finished, checks it and
 * fills out (NULL out: check only).  Requests with device ids may be queued
 * back to back (the stream orders them; only the last one's result is kept);
 * a launch with host ids first waits for the request in flight, because the
 * prompt is staged through one pinned buffer. */
int rtr_launch(rtr_session* s, const int32_t* ids, int32_t L, int32_t ids_on_device);
int rtr_wait(rtr_session* s, const rtr_result* out);

/* Counters of the session, the counterpart of the reference's report()
 * records (PrefixReplayPool.report, PrefixArena.report, ReorderSuffix.report:
 * decode_replay.py:193-202, shared_prefix.py:110-116, prefix_replay.py:242-244). */
typedef struct {
  int64_t requests;               /* requests launched                         */
  int64_t kernel_launches;        /* kernels issued, graph nodes included      */
  int64_t launches_per_request;   /* kernels one request issues                */
  int64_t graph_kernel_nodes;     /* kernel nodes of the decode graph          */
  int64_t prefix_bytes_written;   /* prefix K/V written by the last prefill    */
  int64_t prefix_bytes_reordered; /* always 0: the prefix is shared in place   */
  int64_t suffix_bytes_written;   /* suffix K/V written per request            */
  int64_t suffix_bytes_gathered;  /* 0: parents are followed through anc rows  */
  int64_t weight_bytes;           /* resident weight bytes                     */
  int64_t device_bytes;           /* all device memory the session holds       */
  int64_t h2d_bytes_per_request;  /* prompt ids + length                       */
  int64_t d2h_bytes_per_request;  /* the result record                         */
  int64_t tensor_core_gemm;       /* 2: tcgen05 fp16-pair projections (fp32
                                     default), 1: tcgen05 3xTF32, 0: FFMA      */
  int64_t norm_fold;              /* 1: RMSNorms folded into the GEMMs         */
  int64_t decode_attention;       /* 0: per-head kernel (fp32 default,
                                     RTR_ATTN=rows), 1: tensor-core folded
                                     kernel (bf16 default, fp32 RTR_ATTN=tc),
                                     2: folded FFMA kernel (RTR_ATTN=folded)   */
  int64_t prefill_attention;      /* 0: FFMA kernel, 1: tensor-core kernel
                                     (default; RTR_PREFILL_ATTN=ffma)          */
} rtr_report;
int rtr_get_report(const rtr_session* s, rtr_report* out);

/* Measurement hook (no reference counterpart): run every projection GEMM of
 * one forward pass over M rows (q/k/v, o, gate/up, down per layer, then the
 * LM head) `reps` times on the session stream and return the average device
 * milliseconds of one pass, timed with CUDA events.  Activations are
 * scratch; the session must not have a request in flight. */
int rtr_profile_gemms(rtr_session* s, int32_t M, int32_t reps, float* ms_per_pass);

/* Test hook (no reference counterpart): C[M, N] = X[M, K] . W[N, K]^T (fp32,
 * row-major, device pointers) through one projection-GEMM kernel: 0 the
 * engine's fp32 dispatch (= 5), 1 the 64-row tcgen05 3xTF32 kernel, 2 the
 * 128-row one, 3 the bf16 kernel (X and W rounded to bf16 first; C holds the
 * bf16-rounded products as fp32), 4 the FFMA kernel, 5 the tcgen05 fp16-pair
 * kernel (X and W as fp16 (hi, lo) pairs; 64-row CTAs for M <= 64, else
 * 128-row).  N must be a multiple of 4 and K of 4 (8 for the bf16 and
 * fp16-pair kernels, 32 for FFMA).  Scratch is allocated per call; blocks
 * until done. */
int rtr_gemm_check(int32_t device, const float* x_dev, const float* w_dev, float* c_dev, int32_t M, int32_t N,
                   int32_t K, int32_t kernel);

/* Test hook (no reference counterpart): causal prefill attention of one layer
 * of one user, out[L, heads, D] = softmax(q k^T / sqrt(D), causal) v with the
 * query heads of KV group g = h / (heads / kv_heads) reading k, v [g] (fp32,
 * row-major, device pointers; k and v [kv_heads, L, D]) through one kernel:
 * 0 the FFMA kernel, 1 the tensor-core fp16-pair kernel, 2 the bf16 FFMA
 * kernel and 3 the bf16 tensor-core kernel (2 and 3: q, k, v rounded to bf16
 * first, out holds the bf16 results).  head_dim 64 or 128.  Builds the arena
 * and copies the kernel reads; scratch is allocated per call; blocks until
 * done. */
int rtr_attention_check(int32_t device, const float* q_dev, const float* k_dev, const float* v_dev, float* out_dev,
                        int32_t L, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t kernel);

/* Test hook (no reference counterpart; the reference's failure handling is
 * Python exceptions): on `device`, bound every pipeline wait of the
 * fp16-pair and bf16 tensor-core GEMMs to wait_cycles (default 2e9, ~1 s) and,
 * with withhold_activation_copies = 1, make their activation producers issue
 * no copy.  Those waits then run out: each CTA stops issuing, drains what it
 * issued, frees its tensor memory, keeps the split-K tickets whole and sets the
 * timeout bit of the session's status word, so the request fails with
 * RTR_ERR_DEVICE and the next request runs normally.  Applies to kernels
 * launched (or graph nodes replayed) after the call; wait_cycles >= 1000.
 * The 8-bit KV cache's attention is bounded and fails the same way (its tiles of many rows
 * then withhold the last K of a block's keys; the bit is set in the cache's status
 * word); a captured call keeps the setting it was captured with.
 * Blocks until the setting is on the device. */
int rtr_debug_wait_control(int32_t device, int64_t wait_cycles, int32_t withhold_activation_copies);

/* Processed scores of step t (0..4) as a dense [B, V] float32 device matrix:
 * the double-normalised log-probabilities at allowed columns and -inf
 * elsewhere, i.e. GenerateBeamOutput.scores[t] (the --save-full-scores
 * payload, benchmark_inference.py:160-172). */
int rtr_step_scores(rtr_session* s, int32_t t, float* out_dev);

/* ---- plugin-level entry points (the reference's LogitsProcessor API) ---- */

/* GpuSidConstraintTables.lookup (gpu_constraints.py:75-87): allowed columns
 * for input_ids [rows, cols] (int64, device) at step; out_dev [rows, width]
 * int32 where width = n_first at steps 0/3, width1 / width2 at steps 1/2 and 1
 * afterwards (rtr_lookup_width). */
int rtr_lookup_width(const rtr_session* s, int32_t step, int32_t* width);
int rtr_constraint_lookup(rtr_session* s, int32_t step, const int64_t* input_ids_dev,
                          int32_t rows, int32_t cols, int32_t* out_dev);

/* GpuSidConstrainedLogitsProcessor.__call__ (gpu_constraints.py:95-101):
 * out = log_softmax(scores) + mask(lookup(step, input_ids)); scores and out
 * are [rows, V] float32 device matrices (out may not alias scores). */
int rtr_constraint_process(rtr_session* s, int32_t step, const int64_t* input_ids_dev,
                           int32_t rows, int32_t cols, const float* scores_dev, float* out_dev);

/* Allocation-free rtr_constraint_process.  No counterpart in the reference.
 * For callers that must not allocate device memory per call - a plugin whose
 * host framework owns the GPU allocator and has reserved the memory, or a
 * serving loop whose latency budget rules out the allocator's synchronisation.
 * It computes the same scores with the same kernels, but keeps the per-row
 * reduction scratch in a fixed static device array of the library instead of
 * session memory, and it calls no cudaMalloc, cudaFree or allocating routine.
 * Limits and caveats:
 *   - rows <= 256 (the array's size: 256 rows x 16 slices x 2 floats = 32 KiB,
 *     held by every GPU that loads the library until the process exits);
 *     larger requests fail with RTR_ERR_ARG;
 *   - the first call on a device looks the array's device address up once
 *     (cudaGetSymbolAddress) and keeps it; do not call cudaDeviceReset on
 *     that device afterwards (the kept address would be stale);
 *   - all calls share the one array, so calls whose work overlaps on the GPU
 *     (other streams, other sessions on the same device) race on it; nothing
 *     needs clearing between calls, because each call writes every slot it
 *     reads before reading it;
 *   - blocks until the scores are written. */
int rtr_constraint_process_static(rtr_session* s, int32_t step, const int64_t* input_ids_dev,
                                  int32_t rows, int32_t cols, const float* scores_dev, float* out_dev);

/* ---- 8-bit KV cache --------------------------------------------------------
 * K and V of many sequences (users' histories) kept beside or between requests
 * in a quarter of the fp32 bytes: e4m3 codes in pages, with one float32 scale for
 * each page and KV head.  No counterpart in the reference, whose prefix lives for
 * one request (shared_prefix.py:67-89).  These calls need no session: they take
 * the buffers, a device and a cudaStream_t (NULL: the default stream), enqueue
 * their kernels and return; every buffer is the caller's and must live until
 * they ran.  They may be captured into a CUDA graph.  rtr_last_error(NULL) has
 * the text of a refusal.
 *
 * A value is code * scale.  Code [page][head][token][dim] lies at
 * page * page_stride + head * head_stride + token * head_dim + dim, its scale at
 * page * scale_stride + head.  head_dim 64 or 128, page 16, 32, 64 or 128 tokens;
 * strides of codes and their addresses are multiples of 16, and either a page's last head
 * ends before the next page or a head's last page before the next head.  `status` is a device
 * word that the kernels set bits in (never clear): 1 << 5 a length or row range
 * that does not fit, 1 << 8 a bounded wait that ran out (its call's rows are undefined),
 * 1 << 9 a page number outside [0, pages), 1 << 10 an old scale that is not positive and
 * finite.  The work concerned is left out (attention:
 * rows of NaN; where starts itself is at fault the whole call is left out and no row written),
 * memory outside the buffers is never touched. */
typedef struct {
  void *k, *v;
  float *k_scale, *v_scale;
  int64_t page_stride, head_stride, scale_stride; /* elements */
  int32_t pages, kv_heads, page, head_dim;
  uint32_t* status;
} rtr_kv_cache;

/* Sequences of one call and their rows (device arrays).  Sequence b's i-th page is
 * table[b * table_stride + i], i < table_width; it holds lens[b] tokens.  Rows
 * starts[b] .. starts[b + 1] - 1 of the call's `rows` are its rows (starts has
 * seqs + 1 entries, not decreasing); without starts each has rows / seqs.  Rows
 * before starts[0] and from starts[seqs] on belong to none and are not touched. */
typedef struct {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int64_t table_stride;
  int32_t table_width, seqs, rows;
} rtr_kv_batch;

/* Quantise k and v rows (row r, head h, dim d at r * token_stride + h * head_stride
 * + d; RTR_DTYPE_*; addresses and strides multiples of 16 bytes) into the cache as
 * the last positions of their sequences: lens already counts them.  A page's scale
 * is the least power of two in [2^-48, 2^48] at which its largest magnitude is at
 * most 448; a page that already holds older tokens of the sequence keeps its scale
 * if that is larger, and has their codes rounded again if it is smaller.  Codes are
 * rounded to nearest even; NaN, infinities and magnitudes above 448 * 2^48 become
 * NaN.  Codes behind a sequence's last token stay.  The pages that a call writes
 * must be different ones: where two sequences write into one page, its codes and scale
 * are some of either's. */
int rtr_kv_write(const rtr_kv_cache* cache, const rtr_kv_batch* batch, const void* k_dev, const void* v_dev,
                 int32_t dtype, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                 int64_t v_head_stride, int32_t device, void* stream);

/* The reverse: each sequence's last starts[b + 1] - starts[b] tokens as dense rows,
 * rounded once to dtype. */
int rtr_kv_read(const rtr_kv_cache* cache, const rtr_kv_batch* batch, void* k_dev, void* v_dev, int32_t dtype,
                int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                int32_t device, void* stream);

/* out[r][h] = softmax(scale * q[r][h] . K^T) V, K and V [h / (heads / kv_heads)] of
 * the row's sequence.  causal: a sequence's n rows stand at its last n positions and
 * see what is not behind them; otherwise each sees all lens[b] tokens.  Rows that see
 * nothing are 0.  q: row r, head h at r * q_token_stride + h * head_dim; out
 * [rows][heads][head_dim], same dtype, q itself or apart from it; lse_dev (optional, float32
 * [rows][heads]): log of the softmax's sum, minus infinity for rows that see nothing.  fp32 q and
 * weights enter the tensor cores as fp16 pairs: 22 bits, or for small ones half a step of 2^-37
 * of the largest q of the row, of 2^-39 of the largest weight (times V scale) among 128 keys.
 * bf16 rows' weights are one fp16 value: 11 bits, or half a step of 2^-34 of the row's largest.
 * Sums are fp32.  A row that sees a page whose V scale is outside [2^-48, 2^48], whose K scale
 * is negative or NaN or whose number is outside the cache is NaN.  The workspace must hold
 * rtr_kv_attention_workspace bytes (the same batch, dtype and heads), aligned to 16, and is
 * free again when the call's kernels ran: calls that may overlap need one each.  A table row wider than the
 * sequences need costs idle blocks. */
int rtr_kv_attention_workspace(const rtr_kv_cache* cache, const rtr_kv_batch* batch, int32_t dtype, int32_t heads,
                               int32_t device, int64_t* bytes);
int rtr_kv_attention(const rtr_kv_cache* cache, const rtr_kv_batch* batch, const void* q_dev, int32_t dtype,
                     int32_t heads, int64_t q_token_stride, int32_t causal, float scale, void* out_dev, float* lse_dev,
                     void* workspace_dev, int64_t workspace_bytes, int32_t device, void* stream);

/* A request's prefix kept beyond the request, for users who come back (no counterpart in
 * the reference: its prefix arena holds one request, shared_prefix.py:67-100).
 * rtr_keep_prefix, between rtr_prefill and the first decode step: quantises the prefix of
 * every layer into pages of a cache with layers x kv_heads heads (head l * kv_heads + g is
 * layer l's group g), table_dev [table_width] its page numbers, and copies the final hidden
 * state of the prompt's last token (hidden elements of the session's type) to hidden_dev.
 * Blocks until done; a prefill that failed on the device is refused (RTR_ERR_DEVICE) and nothing
 * written; a page number outside the cache sets the cache's status word.
 * rtr_prefill_kept takes rtr_prefill's place for that user: step 0 from the hidden state
 * (the same scores as at first), then rtr_decode_step 1 - 4 and rtr_read_results as ever,
 * the prefix's K and V now the 8-bit values.  in_place: the decode steps attend over the
 * pages (they must stay until rtr_read_results; a page number outside the cache fails the
 * request); otherwise the pages are read back into the arena first, which needs a decode
 * attention that reads the arena alone (fp32: the default kernel).  ids: host. */
int rtr_keep_prefix(rtr_session* s, const rtr_kv_cache* cache, const int32_t* table_dev, int32_t table_width,
                    void* hidden_dev);
int rtr_prefill_kept(rtr_session* s, const rtr_kv_cache* cache, const int32_t* table_dev, int32_t table_width,
                     const int32_t* ids, int32_t L, const void* hidden_dev, int32_t in_place);

/* ---- pages of sequences that grow and shrink -------------------------------
 * The page numbers of a paged cache (the 8-bit one above or a caller's own) handed out and taken
 * back on the GPU.  No counterpart in the reference, whose prefix arena holds one request
 * (shared_prefix.py:67-89).  `free` [pages] is a stack of page numbers, `count` its height (device
 * word), `marks` [pages] 1 for a page that a sequence holds and 0 for a free one, `status` a device word that the
 * kernels set bits in, `ticket` a device word that is 0 between calls.  Calls on one pool must follow
 * one another (one stream, or streams that wait); they may be captured into a CUDA graph.
 * What is read from device memory is checked, and a call that does not fit as a whole changes
 * nothing but the status word: 1 << 5 a length or row count that does not fit (negative, more
 * tokens than a table row holds, more rows than the call has), 1 << 9 a page number outside
 * [0, pages), 1 << 11 fewer free pages than are needed, 1 << 12 a page given back that no sequence holds. */
typedef struct {
  int32_t *free, *count, *marks;
  uint32_t *status, *ticket;
  int32_t pages, page; /* page: tokens, a power of two from 1 to 1024 */
} rtr_page_pool;

/* Sequence b holds held[b] tokens and gets fresh[b] more (fresh NULL: `each`): table row b gets the page
 * numbers that it needs for them, the call's j-th page (sequences in order, then pages in order)
 * free[count - 1 - j].  lens[b] = held[b] + fresh[b]; starts [seqs + 1]: running sum of the fresh tokens.  Row
 * starts[b] + i has positions held[b] + i (its place in the sequence) and slots table[b][position / page] * page +
 * position % page; a row whose page number is outside the pool, and rows from starts[seqs] to `rows`,
 * have -1 in both.  A call that does not fit: lens = held, starts 0, every row -1.  At most 16384 sequences.  lens, starts,
 * positions and slots must not overlap the inputs. */
int rtr_pages_grow(const rtr_page_pool* pool, int32_t* table, int64_t table_stride, int32_t table_width, const int32_t* held,
                   const int32_t* fresh, int32_t each, int32_t seqs, int32_t rows, int32_t* lens, int32_t* starts,
                   int32_t* positions, int64_t* slots, int32_t device, void* stream);

/* The reverse: of held[b] tokens the sequence keeps keep[b] (keep NULL: none), and the pages that those do not need go
 * back: page j of m (in the same order) to free[count + m - 1 - j], so that growing again by as much takes
 * the same pages in the same places.  The table stays as it is. */
int rtr_pages_release(const rtr_page_pool* pool, const int32_t* table, int64_t table_stride, int32_t table_width,
                      const int32_t* held, const int32_t* keep, int32_t seqs, int32_t device, void* stream);

/* ---- rotary positions ------------------------------------------------------
 * The rotation that the engine fuses into its q/k/v projection (Qwen2RotaryEmbedding: pairs half a
 * head apart), for rows of a caller's own and with the other layouts: pairs (2 i, 2 i + 1) where
 * `interleaved`, the first rotary_dim dimensions of a head alone, scaled frequencies.  Pair i of row r becomes
 *   factor * (a cos t - b sin t, b cos t + a sin t),  t = 2 pi * fraction(positions[r] * turns[i] / 2^64)
 * with turns [rotary_dim / 2] the frequencies in turns a position, times 2^64 (device array): the
 * product modulo 2^64 is the angle itself, as exact at position 2^31 as at 1 (turns rounded to half a unit: off by
 * positions * 2^-65 turns).  back: -t, which takes the rotation back and is its transpose (the
 * gradient of a rotated row gives that of the row).  Rows may be strided; out is the input itself or apart
 * from it, and holds all head_dim dimensions.  fp32 arithmetic, one rounding to dtype. */
typedef struct {
  const void* in;
  void* out;
  int64_t in_row, in_head, out_row, out_head; /* strides in elements; dimensions are contiguous */
  int32_t heads;
} rtr_rotary_rows;

/* k may be NULL.  head_dim 2 to 512, rotary_dim even and at most head_dim.  positions: int32 or (wide) int64, of any
 * sign. */
int rtr_rotary(const rtr_rotary_rows* q, const rtr_rotary_rows* k, int64_t rows, int32_t head_dim, int32_t rotary_dim,
               int32_t interleaved, int32_t dtype, const void* positions, int32_t wide, const uint64_t* turns, float factor,
               int32_t back, int32_t device, void* stream);

/* ---- beam search over whole vocabularies -----------------------------------
 * One step of a beam search that no catalog constrains to a few columns (rtr_decode_step's beam update has
 * at most 256 allowed tokens a beam and five steps; this replaces the log_softmax, top-k and
 * bookkeeping of HF GenerationMixin._beam_search, generation/utils.py:3252-3352, for callers with a
 * model of their own).  Item b has n beams: rows b * n .. of logits [items * n][logits_stride], scores [items][n].  The candidate
 * (i, v) is worth logits[i][v] - log sum_u exp logits[i][u] + scores[i] where allowed (bytes [items * n][allowed_stride],
 * NULL: everywhere; an allowed_stride of 0 is one row for all) is not 0, and minus infinity elsewhere.  all_* [items][k]: the k best, in
 * descending order, equal ones by i * vocab + v: token v, parent i, value.  next_* [items][beams]: the first
 * `beams` of those whose token is not eos (eos < 0: none is).  A row whose score is minus infinity is not read.  A row
 * with a NaN or plus infinity among its logits, or such a score, is worth minus infinity throughout and sets 1 << 7 in `status` (a
 * device word).  The order is that of values computed in 64 bits: rows are summed in 32, and again in 64 where two candidates are
 * closer than that may be off by.  The values are float32; those of rows that were not summed again are off by 1.4e-6 at most besides,
 * and may differ in their last bits with the call's other rows.  A value below float32's range counts as minus infinity.
 * n 1 to 128, vocab 1 to 2^20, k 1 to 256 and at most n * vocab, beams at most k (with eos: k at least beams + n).  dtype float32 or bfloat16; the workspace (rtr_beam_select_workspace bytes, aligned to 16) is free again when the call's
 * kernels ran. */
typedef struct {
  const void* logits;
  const float* scores;
  const uint8_t* allowed;
  int64_t logits_stride, allowed_stride;
  int32_t dtype, items, n, vocab, k, beams, eos;
  int32_t *all_tokens, *all_parents, *next_tokens, *next_parents;
  float *all_scores, *next_scores;
  uint32_t* status;
} rtr_beam_step;
int rtr_beam_select_workspace(const rtr_beam_step* step, int32_t device, int64_t* bytes);
int rtr_beam_select(const rtr_beam_step* step, void* workspace_dev, int64_t workspace_bytes, int32_t device, void* stream);

/* The states of the beams in the order that a step's parents give: row b * beams + i of every state becomes what row
 * b * beams + parents[b][i] was, in place (the reference's ReorderSuffix copies every row into new tensors,
 * prefix_replay.py:95-117; here only rows that move are written, and their parents read once).  A state has rows at
 * data + r * row_bytes and in each of them up to three outer dimensions of sizes[] at strides[] bytes and `inner` contiguous
 * bytes; no two bytes of the states may be the same.  A parent outside [0, beams) sets 1 << 1 in `status`
 * (a device word), and its row stays.  At most 128 beams. */
typedef struct {
  void* data;
  int64_t row_bytes, inner, strides[3];
  int32_t sizes[3];
} rtr_beam_state;
int rtr_beam_reorder(const rtr_beam_state* states, int32_t count, const int32_t* parents, int32_t items, int32_t beams,
                     uint32_t* status, int32_t device, void* stream);

/* ---- synthetic workload --------------------------------------------------- */

/* Deterministic synthetic tensor values: element i of stream (seed, tid) is
 * (k - 2^23) * (scale * 2^-23) + offset, k = top 24 bits of
 * splitmix64(key(seed, tid) + i * golden).  Host (multi-threaded) and device
 * fills are bit-identical.  No reference counterpart: it generates the
 * stand-in for the unavailable release checkpoint. */
int rtr_synth_fill_host(float* dst, int64_t n, uint64_t seed, uint64_t tid, float scale, float offset);
int rtr_synth_fill_device(float* dst_dev, int64_t n, uint64_t seed, uint64_t tid, float scale,
                          float offset, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RTR_B200_H */
