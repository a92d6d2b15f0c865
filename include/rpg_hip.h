/* rpg_hip.h -- token-level and kernel-level C entry points of the MI355X
 * engine, below the chat ABI of rpg_engine.h.
 *
 * These replace the reference's internal C++ seams for this path, which its
 * own parity tools and benchmarks drive (reference src/qwen3.h:83-142,
 * src/sampler.h:35-65, src/quant.h, src/matmul.h:35-64). Plain pointers and
 * sizes, no C++ types; host buffers in and out unless a name says "dev".
 * Return: >= 0 success (handles, counts), < 0 failure with the message in
 * rpg_hip_last_error(). Handles are int32 from 1, never reused.
 */
#ifndef RPG_HIP_H
#define RPG_HIP_H

#include <stdint.h>

#if defined(__GNUC__)
#define RPG_HIP_API __attribute__((visibility("default")))
#else
#define RPG_HIP_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

RPG_HIP_API const char* rpg_hip_last_error(void);

/* Number of visible GPUs (0 when none; never fails). */
RPG_HIP_API int32_t rpg_hip_device_count(void);

/* ---- model: reference Model::Load (src/model.cc:147-281) */
RPG_HIP_API int32_t rpg_hip_model_load(const char* gguf_path, int32_t max_pos);
RPG_HIP_API void rpg_hip_model_free(int32_t model);
/* out[9] = n_layers, hidden, n_heads, n_kv_heads, head_dim, intermediate,
 *          vocab, context_length, eos_id */
RPG_HIP_API int32_t rpg_hip_model_config(int32_t model, int32_t* out);
/* Bytes read from HBM for weights per decode token (all matrices incl.
 * lm_head, norms, one embedding row). */
RPG_HIP_API int64_t rpg_hip_model_decode_bytes(int32_t model);
/* RoPE table row of position pos: hd floats = cos(hd/2) | sin(hd/2)
 * (reference src/model.cc:122-145). */
RPG_HIP_API int32_t rpg_hip_model_rope_row(int32_t model, int64_t pos, float* out);

/* ---- session: KV cache + token loop (reference src/kv_cache.h, src/qwen3.h) */
RPG_HIP_API int32_t rpg_hip_session_new(int32_t model, int64_t max_seq);
RPG_HIP_API void rpg_hip_session_free(int32_t session);
RPG_HIP_API int64_t rpg_hip_session_len(int32_t session);
RPG_HIP_API int32_t rpg_hip_session_set_len(int32_t session, int64_t len);

/* ForwardFull with a cache (reference src/qwen3.cc:208-290): append n ids at
 * positions len..len+n-1. last_logits[vocab] and all_logits[n*vocab] may be
 * NULL. */
RPG_HIP_API int32_t rpg_hip_prefill(int32_t session, const int32_t* ids, int64_t n, float* last_logits,
                                    float* all_logits);

/* Generate (reference src/qwen3.cc:302-355). first_logits == NULL continues
 * from the last device logits. temperature <= 0 is greedy; top_k / top_p /
 * seed as SampleOptions (reference src/sampler.h:35-45). step_logits
 * (optional) receives [returned, vocab]. Returns the number of ids written to
 * out_ids (capacity max_tokens). */
RPG_HIP_API int32_t rpg_hip_generate(int32_t session, const float* first_logits, int32_t max_tokens,
                                     float temperature, int32_t top_k, float top_p, uint64_t seed,
                                     const int32_t* stop_ids, int32_t n_stop, int32_t* out_ids,
                                     float* step_logits);

/* Generate for n sessions of one model at once (1 <= n <= 8): each session
 * continues from its device logits with its own temperature[i], top_k[i],
 * top_p[i], seed[i] and produces max_tokens ids into out_ids[i * max_tokens
 * ...], the tokens it would produce alone (reference src/qwen3.cc:302-355 per
 * session); one decode step forwards all n tokens, each weight matrix read
 * once. No stop ids: every session needs room for max_tokens positions.
 * step_logits (optional, [n][max_tokens][vocab]) receives each session's
 * logits after each generated token (parity probe); decode_ms (optional)
 * the device time of the steps. Returns max_tokens. */
RPG_HIP_API int32_t rpg_hip_generate_batch(const int32_t* sessions, int32_t n, int32_t max_tokens,
                                           const float* temperature, const int32_t* top_k, const float* top_p,
                                           const uint64_t* seed, int32_t* out_ids, float* step_logits,
                                           double* decode_ms);

/* Teacher-forced decode (parity probes; no reference counterpart): like
 * rpg_hip_generate without stop ids, except that step i forwards
 * force_ids[i] instead of the id the sampler drew, which goes to
 * drawn_ids[i]. Every step then decides on the logits of the forced history,
 * so a caller holding another engine's ids and per-step logits can compare
 * every step. Returns max_tokens. */
RPG_HIP_API int32_t rpg_hip_generate_forced(int32_t session, const float* first_logits, int32_t max_tokens,
                                            float temperature, int32_t top_k, float top_p, uint64_t seed,
                                            const int32_t* force_ids, int32_t* drawn_ids, float* step_logits);

/* rpg_hip_generate_batch with teacher forcing: session i forwards
 * force_ids[i * max_tokens + t] at step t; drawn_ids[i * max_tokens + t]
 * receives the id drawn. No reference counterpart (parity probe). */
RPG_HIP_API int32_t rpg_hip_generate_batch_forced(const int32_t* sessions, int32_t n, int32_t max_tokens,
                                                  const float* temperature, const int32_t* top_k,
                                                  const float* top_p, const uint64_t* seed,
                                                  const int32_t* force_ids, int32_t* drawn_ids,
                                                  float* step_logits);

/* Failure injection for the out-of-memory contract (test hook; no reference
 * counterpart): after n more successful device allocations in this process,
 * the next one fails as a failed hipMalloc would, without calling it
 * (models, sessions, batches and the token-level buffers allocate this way);
 * n < 0 switches injection off. One failure per call. Returns 0. */
RPG_HIP_API int32_t rpg_hip_fail_alloc_after(int64_t n);

/* Which decode path the session runs: 0 = one launch per projection and
 * attention stage (the default), 1 = one persistent launch per token (only
 * when RPG_DECODE_STEP=1 was set at session creation and every projection is
 * Q4_K / Q6_K with a tile-major copy). No reference counterpart: a test
 * probe. */
RPG_HIP_API int32_t rpg_hip_session_decode_path(int32_t session);

/* Copy K (which = 0) or V (1) of (layer, kv_head, positions [0, n)), fp32. */
RPG_HIP_API int32_t rpg_hip_kv_read(int32_t session, int32_t which, int32_t layer, int32_t head, int64_t n,
                                    float* out);

/* Device milliseconds of the session's last prefill / generate call. */
RPG_HIP_API int32_t rpg_hip_session_timing(int32_t session, double* prefill_ms, double* decode_ms);

/* Roofline probe of the decode step's largest launch: `iters` back-to-back
 * gate+up (SwiGLU) matvecs on the session's stream, layers layer+1,
 * layer+2, ... (mod n_layers, so no launch re-reads cached weights), timed
 * with HIP events. out[0] = mean microseconds per launch, out[1] =
 * algorithmic bytes per launch (both weight matrices, input, norm gain,
 * output). No reference counterpart: measurement only. */
RPG_HIP_API int32_t rpg_hip_session_bench_gate_up(int32_t session, int32_t layer, int32_t iters, double* out);

/* The same launches where the decode step runs them: `tokens` greedy decode
 * steps from the session's state through the per-launch path, each layer's
 * gate+up launch bracketed by HIP events on the session stream (the interval
 * includes its dispatch after the previous kernel). out[0] = mean
 * microseconds per launch, out[1] = algorithmic bytes per launch. The session
 * must be prefilled and advances by `tokens`. Measurement only. */
RPG_HIP_API int32_t rpg_hip_session_instep_gate_up(int32_t session, int32_t tokens, double* out);

/* Device-to-device copy of `bytes` (a multiple of 16) by a plain grid-stride
 * kernel, `iters` times between two buffers: *us = mean microseconds per
 * copy. The measured stream bandwidth, and a kernel of known read and write
 * volume for calibrating byte counters. Measurement only. */
RPG_HIP_API int32_t rpg_hip_bench_copy(int64_t bytes, int32_t iters, double* us);

/* ---- kernels on host buffers (parity tests and microbenchmarks) */

/* DequantizeRow on the GPU, bit-exact (reference src/quant.cc:416-436). */
RPG_HIP_API int32_t rpg_hip_dequant(uint32_t type, const uint8_t* src, int64_t n, float* dst);

/* Y[t*rows + r] = X[t] . W[r] for t < n: the fused dequant matvec / blocked
 * matmul (reference src/matmul.h:35-64, QuantMatrix::MatMulBatch
 * src/model.cc:39-69). */
RPG_HIP_API int32_t rpg_hip_matmul(uint32_t type, const uint8_t* w, int64_t rows, int64_t cols, const float* X,
                                   int64_t n, float* Y);

/* The few-token matvec the batched decode step runs (1 <= n <= 8 tokens,
 * Q4_K / Q6_K, cols % 256 == 0, cols <= 10240), on a tile-major copy it
 * makes: with norm_w (a [cols] gain) each row of X is RMS-normalised first
 * (reference src/qwen3.cc:131-134: double sum of squares, float scale,
 * (x * scale) * w); with `up` the output is silu(X[t] . W[r]) * (X[t] .
 * U[r]) (reference src/kernels.h:82-92); with add != 0, Y[t*rows + r] +=
 * X[t] . W[r] (the residual add, reference src/qwen3.cc:186-188), else
 * Y = X . W^T (reference src/matmul.h:35-64). Returns 0, or -1 on error. */
RPG_HIP_API int32_t rpg_hip_matvec_few(uint32_t type, const uint8_t* w, const uint8_t* up, int64_t rows, int64_t cols,
                                       const float* X, int64_t n, const float* norm_w, float eps, int32_t add,
                                       float* Y);

/* Y[t*rows + r] = silu(X[t] . G[r]) * (X[t] . U[r]) for t < n (n >= 2): the
 * prefill's gate/up projection with SwiGLU (reference src/kernels.h:82-92,
 * src/qwen3.cc:191-199). Returns 1 when the single fused GEMM launch ran, 0
 * when the two products and the SwiGLU pass ran, -1 on error. */
RPG_HIP_API int32_t rpg_hip_matmul_swiglu(uint32_t type, const uint8_t* gate, const uint8_t* up, int64_t rows,
                                          int64_t cols, const float* X, int64_t n, float* Y);

/* SampleToken (reference src/sampler.cc:96-112) with
 * u = CounterUniform(seed, counter) computed on the GPU; probs (optional,
 * [n]) receives FilterToProbs. Returns the token id. */
RPG_HIP_API int32_t rpg_hip_sample(const float* logits, int32_t n, float temperature, int32_t top_k, float top_p,
                                   uint64_t seed, int64_t counter, float* probs);

/* Number of sampler draws so far that took the sequential fallback. */
RPG_HIP_API int64_t rpg_hip_sampler_fallbacks(void);

/* Number of rpg_hip_sample draws so far whose top-p cut split a set of equal
 * probabilities, resolved by replaying the reference's std::sort order
 * (reference src/sampler.cc:72-82). Test probe. */
RPG_HIP_API int64_t rpg_hip_sampler_tie_orders(void);

/* rpg_hip_sample without any allocation. No counterpart in the reference: it
 * is for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops). Device buffers in and out: logits_dev [n]
 * fp32, token_dev [1], probs_dev [n] (optional, FilterToProbs); u =
 * CounterUniform(seed, counter). The work is enqueued on `stream` (a
 * hipStream_t; NULL = the null stream) and is complete when the stream is.
 * Scratch is a static device array of 8 MiB + 4 KiB per GPU (held until the
 * process ends): n must be at most 262144. Calls that overlap on one GPU
 * race on it. Returns 0 when enqueued, -1 on error. */
RPG_HIP_API int32_t rpg_hip_sample_noalloc(const float* logits_dev, int32_t n, float temperature, int32_t top_k,
                                           float top_p, uint64_t seed, int64_t counter, int32_t* token_dev,
                                           float* probs_dev, void* stream);

/* Causal GQA attention of a segment (the prefill kernel; reference
 * src/qwen3.cc:79-117): q [seq][n_heads][128] (QK-normed, rotated), the cache
 * contents k, v [n_kv][pos0 + seq][128], query t at position pos0 + t sees
 * positions 0 .. pos0 + t; out [seq][n_heads][128]. */
RPG_HIP_API int32_t rpg_hip_attention(const float* q, const float* k, const float* v, int32_t seq, int32_t n_heads,
                                      int32_t n_kv, int32_t pos0, float* out);

/* Where the GEMM operands of a segment of `tokens` x k inputs and the partial
 * sums of its products (columns: of the widest launch; q8: Q8_0 weights among them) lie in their
 * buffer: out = {operands' begin, end, partials' begin, end, buffer size}, bytes. Host
 * only. */
RPG_HIP_API int32_t rpg_hip_split_layout(int32_t tokens, int32_t k, int32_t columns, int32_t q8,
                                         int64_t* out);

/* glibc-exact expf on the GPU over n inputs (parity probe). */
RPG_HIP_API int32_t rpg_hip_expf(const float* x, int64_t n, float* out);

/* Microbenchmark: for each token count ns[i], time `iters` launches of the
 * matmul y[n][rows] = x[n][cols] . W^T over `copies` device copies of W
 * (rotated so the weights stream from HBM; one upload, then device copies).
 * n = 1 takes the decode path (tile-major copies where the type has one).
 * out[i] = average milliseconds per launch at ns[i]. */
RPG_HIP_API int32_t rpg_hip_bench_matmul(uint32_t type, const uint8_t* w, int64_t rows, int64_t cols,
                                         const int32_t* ns, int32_t n_count, int32_t copies, int32_t iters,
                                         double* out);

/* ---- serving operators on device buffers: a paged key-value cache that many
 * sequences share, the attention that reads it, and a sampler of many rows. No
 * counterpart in the reference, whose cache belongs to one session
 * (src/kv_cache.h:19-34) and whose sampler draws its own numbers; for hosts
 * that schedule sessions themselves.
 *
 * Every pointer is a device pointer of the current GPU. The work is enqueued
 * on `stream` (a hipStream_t; NULL = the null stream), without allocation or
 * synchronisation, so calls may be captured into a graph; it is complete when
 * the stream is. Lengths, pages, starts and sampling parameters are read on
 * the device, so a replayed graph takes the values of that moment. Return 0
 * when enqueued, -1 with a message in rpg_hip_last_error() and nothing
 * enqueued when the arguments are refused.
 *
 * Element types are ggml ids: 0 = f32, 1 = f16, 30 = bf16. Rows of head_dim
 * elements are contiguous; pointers and strides are multiples of 16 bytes,
 * strides are counted in elements. */

/* A pool of n_pages pages, each of page_size positions (a power of two, 16 to
 * 65536) of n_kv heads of head_dim (64 or 128) elements: position r of head h of
 * page p at p * page_stride + h * head_stride + r * row_stride, alike in k and v. */
typedef struct {
  void* k;
  void* v;
  int64_t page_stride, head_stride, row_stride;
  int32_t n_pages, page_size, n_kv, head_dim, type;
} rpg_hip_paged_cache;

/* n_seqs sequences. Sequence s holds lens[s] positions (at most pages *
 * page_size, which is at most 2^30; 0 and less: none), the new tokens among
 * them; position p lies in page table[s * table_stride + p / page_size]. A page
 * number outside [0, n_pages) is never followed: its positions take no part.
 * The new tokens of sequence s are the packed rows starts[s] .. starts[s + 1]
 * (n_seqs + 1 of them, not decreasing), at its last positions; rows of no
 * sequence are left as they are. starts is not read by rpg_hip_paged_decode
 * (one token each). Without sequences a call does nothing. */
typedef struct {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* starts;
  int32_t pages, n_seqs, n_tokens;
} rpg_hip_sequences;

/* [token][head] rows of head_dim elements of the cache's type */
typedef struct {
  void* data;
  int64_t token_stride, head_stride;
} rpg_hip_rows;

/* Stores the new tokens' keys and values in their pages. Keys, and queries
 * from q into q_out (which may be q, with its strides; q->data NULL: no
 * queries), are RMS-normed per head with the gains k_norm and q_norm (f32 [head_dim]; NULL: not normed)
 * and rotated by row `position` of rope (f32 [rope_rows][head_dim], cos |
 * sin, as rpg_hip_model_rope_row; NULL: not rotated), as the engine's own
 * QK-norm and RoPE (reference src/qwen3.cc:139-167), computed in f32 and
 * rounded once. A token whose position is below 0 (more new tokens than
 * positions) or at or past rope_rows is left out: no key, value or query of
 * it is written. Two new tokens whose tables lead to one place leave nothing
 * defined there. */
RPG_HIP_API int32_t rpg_hip_paged_append(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs,
                                         const rpg_hip_rows* k, const rpg_hip_rows* v, const rpg_hip_rows* q,
                                         const rpg_hip_rows* q_out, int32_t n_heads, const float* q_norm,
                                         const float* k_norm, float eps, const float* rope, int64_t rope_rows,
                                         void* stream);

/* Attention of one token per sequence, row s of q, over all of the sequence's
 * positions: out = softmax(scale q . k) v per head, heads kv * (n_heads / n_kv)
 * .. sharing key head kv (reference src/qwen3.cc:79-117). scale > 0. Sums and
 * softmax in f32, weights up to 1 (in prompts 256) before the division by their
 * sum: a float has to hold the keys' number times the largest value times that.
 * For 16-bit types the weights multiply the values in two parts of that type,
 * which together keep 16 (bf16) or 22 bits. A sequence without positions gives
 * zeros. out may be q, with its strides. work: rpg_hip_paged_work bytes, read
 * and written by this call alone until it is complete (any contents; may be
 * NULL when that is 0). */
RPG_HIP_API int32_t rpg_hip_paged_decode(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs,
                                         const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_heads, float scale,
                                         void* work, int64_t work_bytes, void* stream);

/* Causal attention of the packed new tokens: as rpg_hip_paged_decode, the token
 * at position p over positions 0 .. p; for 16-bit types the weights are rounded
 * to that type before they multiply the values. */
RPG_HIP_API int32_t rpg_hip_paged_prompt(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs,
                                         const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_heads, float scale,
                                         void* work, int64_t work_bytes, void* stream);

/* Bytes of work memory that rpg_hip_paged_decode (prompt = 0) or
 * rpg_hip_paged_prompt (prompt = 1) takes for these sizes; -1 when they are
 * refused; 0 for batches with nothing to do. Host only; reads the sizes of *cache and *seqs, no pointers. */
RPG_HIP_API int64_t rpg_hip_paged_work(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs,
                                       int32_t n_heads, int32_t prompt);

/* ---- a cache held in 8 bits. Position r of head h of page p is a row of
 * head_dim codes (k, v: one byte each, strides in bytes, multiples of 16) and a
 * scale (k_scale, v_scale: f32 at p * scale_page_stride + h * scale_head_stride + r,
 * strides in elements, multiples of 4): element = code * scale. code:
 * RPG_HIP_I8 = whole numbers up to 127 either way, RPG_HIP_E4M3 = 8-bit floats of
 * 4 exponent and 3 mantissa bits, up to 448, without infinities. As
 * rpg_hip_paged_cache in all else; the rows that go in and come out are f32, f16 or
 * bf16 (`type`, a ggml id), all of a call alike. */
enum { RPG_HIP_I8 = 0, RPG_HIP_E4M3 = 1 };
typedef struct {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t page_stride, head_stride, row_stride;
  int64_t scale_page_stride, scale_head_stride;
  int32_t n_pages, page_size, n_kv, head_dim, code;
} rpg_hip_quant_cache;

/* rpg_hip_paged_append into such a cache. A row y (keys: as normed and rotated in
 * f32; values: as they are) with the largest magnitude a is held as scale a / M, M
 * the largest code, and codes y M / a in f32, to the nearest, even at ties. Where a is below
 * 2^-112 scale and codes are 0; where y is not finite the scale is NaN, the codes 0:
 * the whole row reads as NaN. */
RPG_HIP_API int32_t rpg_hip_quant_append(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                                         const rpg_hip_rows* k, const rpg_hip_rows* v, const rpg_hip_rows* q,
                                         const rpg_hip_rows* q_out, int32_t n_heads, const float* q_norm,
                                         const float* k_norm, float eps, const float* rope, int64_t rope_rows,
                                         void* stream);

/* The last positions of each sequence as rows: those of sequence s go to the packed
 * rows starts[s] .. starts[s + 1] of k and v ([token][n_kv] rows), computed in f32 and
 * rounded once. Positions of pages that the table does not name give zeros; rows of no
 * sequence and of positions below 0 are left as they are. */
RPG_HIP_API int32_t rpg_hip_quant_read(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                                       const rpg_hip_rows* k, const rpg_hip_rows* v, void* stream);

/* rpg_hip_paged_decode and rpg_hip_paged_prompt over such a cache, q and out rows of
 * `type`. Scales are applied in f32 to scores and weights, codes are multiplied as
 * they are; weights times scales go to the product in two parts of 8 bits, for f32
 * rows in three. Queries are finite; a row whose scale is
 * NaN makes NaN of what sees it, and of nothing else. In places that no query sees codes and scales may be
 * anything, but for the NaN codes of e4m3 (which rpg_hip_quant_append never writes)
 * behind a prompt's token in its own sequence. work: rpg_hip_quant_work bytes. */
RPG_HIP_API int32_t rpg_hip_quant_decode(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                                         const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_heads, float scale,
                                         void* work, int64_t work_bytes, void* stream);
RPG_HIP_API int32_t rpg_hip_quant_prompt(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                                         const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_heads, float scale,
                                         void* work, int64_t work_bytes, void* stream);
RPG_HIP_API int64_t rpg_hip_quant_work(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                                       int32_t n_heads, int32_t prompt);

/* Groups of sequences whose first positions lie in the same pages (a prompt that
 * many sessions share): group g is sequences starts[g] .. starts[g + 1] (n_groups + 1
 * starts, not decreasing), and the tables of those of them that have positions name
 * the same pages for the first shared[g] positions. A sequence may belong to no group.
 * Where tables differ there, it is not defined whose pages are read for which
 * sequence of the group. */
typedef struct {
  const int32_t* starts;
  const int32_t* shared;
  int32_t n_groups;
} rpg_hip_groups;

/* rpg_hip_paged_decode (rpg_hip_quant_decode) that reads what a group has in common
 * once. Group starts and shared positions are read on the device. work:
 * rpg_hip_paged_shared_work (rpg_hip_quant_shared_work) bytes. */
RPG_HIP_API int32_t rpg_hip_paged_shared(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs,
                                         const rpg_hip_groups* groups, const rpg_hip_rows* q, const rpg_hip_rows* out,
                                         int32_t n_heads, float scale, void* work, int64_t work_bytes, void* stream);
RPG_HIP_API int64_t rpg_hip_paged_shared_work(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs,
                                              int32_t n_groups, int32_t n_heads);
RPG_HIP_API int32_t rpg_hip_quant_shared(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs,
                                         const rpg_hip_groups* groups, int32_t type, const rpg_hip_rows* q,
                                         const rpg_hip_rows* out, int32_t n_heads, float scale, void* work,
                                         int64_t work_bytes, void* stream);
RPG_HIP_API int64_t rpg_hip_quant_shared_work(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs,
                                              int32_t n_groups, int32_t type, int32_t n_heads);

/* Edits of logits before a draw. All device pointers; arrays of one element per
 * row unless a stride (in elements) is given.
 *
 * history: the tokens of each row so far ([rows][history_size], of which
 * history_lens counts the first ones that are there; NULL: all), the first
 * prompts[row] of them its prompt (NULL: none). Tokens outside [0, vocab) count for
 * nothing. x being a token's logit and c the times that it was made behind the prompt:
 *   x = x > 0 ? x / repetition : x * repetition   where the history holds it
 *   x = x - frequency c - presence                where c > 0
 *   x = x + bias                                  where bias_ids lists it
 *   x = -inf                                      where its mask's bit is 0
 * in f32, rounded once. repetition, presence, frequency may be NULL: none of it; a
 * repetition that is not above 0 counts as 1. bias_ids, bias: [rows][n_biases];
 * numbers outside [0, vocab) are no entries, of several for one token the last
 * counts. mask: [n_masks] rows of ceil(vocab / 32) words, bit t % 32 of word t / 32
 * set where token t may come; row r goes by mask mask_rows[r] (NULL: r), by none
 * where that is outside [0, n_masks). */
typedef struct {
  const int32_t* history;
  int64_t history_stride;
  const int32_t* history_lens;
  const int32_t* prompts;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const int32_t* bias_ids;
  int64_t bias_ids_stride;
  const float* bias;
  int64_t bias_stride;
  const int32_t* mask;
  int64_t mask_stride;
  const int32_t* mask_rows;
  int32_t history_size, n_biases, n_masks;
} rpg_hip_edits;

/* logits [rows][vocab], row_stride elements apart, edited into out (which may be
 * logits, with its stride: then rows without a mask are touched only where tokens
 * change; and else lies apart from them). Any alignment of the type; vocab <= 2^24, rows <= 65535, history_size
 * <= 2^20, n_biases <= 1023. No work memory. */
RPG_HIP_API int32_t rpg_hip_edit_logits(int32_t type, const void* logits, int64_t rows, int64_t vocab,
                                        int64_t row_stride, const rpg_hip_edits* edits, void* out,
                                        int64_t out_stride, void* stream);

/* One token per row of logits ([rows][vocab], row_stride elements apart, any
 * alignment of the type): weights exp((x - max) / temperature), tokens ranked
 * by value, equal ones by index; kept are the first top_k of them, of those
 * the shortest head that holds top_p of their weight, and of those the ones
 * whose weight is at least min_p times the largest. The token is the first, by
 * index, at which the kept weights' running sum passes u times their sum
 * (u in [0, 1), brought there from outside); logprobs (may be NULL) receives
 * the log of its weight over the kept ones' sum. temperature <= 0: the first
 * largest value, log 1. top_k <= 0 or >= vocab, top_p outside (0, 1) and min_p
 * <= 0 set no limit; each of the four [rows] arrays may be NULL: temperature
 * 1, no limit. NaN counts as -inf; a row with nothing above -inf gives token
 * -1 and log 0 = -inf. Other than rpg_hip_sample, top_k keeps exactly that many,
 * top_k = 1 keeps one, and the weights are exact to 2^-45 of the largest, in
 * any order of summation. vocab <= 262144, rows <= 65535. work:
 * rpg_hip_sample_rows_work bytes. */
RPG_HIP_API int32_t rpg_hip_sample_rows(int32_t type, const void* logits, int64_t rows, int64_t vocab,
                                        int64_t row_stride, const float* temperature, const int32_t* top_k,
                                        const float* top_p, const float* min_p, const float* u, int32_t* tokens,
                                        float* logprobs, void* work, int64_t work_bytes, void* stream);
RPG_HIP_API int64_t rpg_hip_sample_rows_work(int64_t rows, int64_t vocab);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* RPG_HIP_H */
