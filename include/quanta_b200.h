/* quanta_b200.h -- C ABI of the B200 (sm_100a) engine for Quanta.cpp's quantized-transformer hot path.
 *
 * Plain C: pointers, sizes and int status codes; no C++ or CUDA types cross this boundary (streams are void*).
 * Every entry point returns QNT_OK (0) or a negative QNT_ERR_*; qnt_last_error() gives the message of the
 * calling thread's last failure.  Exceptions never cross the ABI.
 *
 * Each declaration names the reference interface it replaces (paths inside the Quanta.cpp tree).
 */
#ifndef QUANTA_B200_H
#define QUANTA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QNT_OK 0
#define QNT_ERR_INVALID (-1)     /* bad argument / shape */
#define QNT_ERR_CUDA (-2)        /* CUDA runtime error */
#define QNT_ERR_IO (-3)          /* file open / parse error */
#define QNT_ERR_UNSUPPORTED (-4) /* valid for the reference, not implemented on the device */
#define QNT_ERR_RANGE (-5)       /* position / context overflow (reference: std::out_of_range) */
#define QNT_ERR_DEVICE (-6)      /* a kernel reported an error bit (bad token id, bounded wait timed out...) */

/* dtypes of engine/src/model_file.h:16 */
#define QNT_F32 0
#define QNT_F16 1
#define QNT_Q8_0 2
#define QNT_Q4_0 3
/* activations only (the qnt_kv_*, norm, rope and beam entries); no .qnt tensor has this type */
#define QNT_BF16 4

const char* qnt_last_error(void);
int qnt_version(void);          /* 100 * major + minor */
int qnt_device_count(void);
int qnt_set_device(int device); /* cudaSetDevice for the calling thread */

/* ---------------------------------------------------------------- ops level (engine/src/ops.h) */

typedef struct qnt_dtensor qnt_dtensor;

/* Uploads a quantized weight matrix given in the .qnt layout (quants, then fp16 scales: engine/src/model_file.h:25-38,
 * scripts/export.py:10-13) to device memory.  Replaces passing `const Tensor& W` (engine/src/ops.h:57,68).
 * When cols % 128 == 0 it also keeps what the tensor-core matmul reads: a K-step-major copy of the scales and, for
 * Q4_0, an int8 copy of q - 8 (rows * cols bytes). */
int qnt_tensor_upload(int dtype, int rows, int cols, const void* host_data, qnt_dtensor** out);
int qnt_tensor_free(qnt_dtensor* t);
int qnt_tensor_shape(const qnt_dtensor* t, int* dtype, int* rows, int* cols);

/* quantize_q8 (engine/src/ops.h:52, ops_ref.cpp:69-83) on device memory: x [n_tok][n] -> q [n_tok][n],
 * d [n_tok][n/32].  stream: a cudaStream_t or NULL. */
int qnt_quantize_q8(const float* x, int n_tok, int n, int8_t* q, float* d, void* stream);

/* MatvecQFn (engine/src/ops.h:57): out[r] = sum_b float(sum_i qW*qx) * dW * dx for r in [r0, r1); device pointers.
 * Bit-identical to matvec_q_ref (engine/src/ops_ref.cpp:85-120) built without FMA contraction. */
int qnt_matvec(const qnt_dtensor* W, const int8_t* qx, const float* dx, int r0, int r1, float* out, void* stream);

/* MatmulQFn (engine/src/ops.h:68): n activations (q [n][cols], d [n][cols/32]), out[t * ldo + r]; device pointers.
 * Per (row, token) bit-identical to qnt_matvec.  impl: 0 auto, 1 CUDA cores, 2 tensor cores (tcgen05; q and d
 * 16-byte aligned; the call makes a stream-ordered block-major copy of d with cudaMallocAsync). */
int qnt_matmul(const qnt_dtensor* W, const int8_t* qx, const float* dx, int n, int r0, int r1, float* out, int ldo,
               int impl, void* stream);

/* No reference counterpart: waits for `stream`, then reports (and clears) the status bits that the calling thread's
 * earlier qnt_matmul calls left -- QNT_ERR_DEVICE when a tensor-core wait gave up.  The host forms check it themselves. */
int qnt_ops_check(void* stream);

/* Synchronous host-pointer forms of the three calls above: the drop-in for the reference's function pointers
 * (a MatvecQFn / MatmulQFn shim passes QuantVec::q / QuantVec::d and the caller's output buffer).  Re-entrant like the
 * reference's kernels, which Model::linear calls from its thread pool on disjoint row ranges (engine/src/model.cpp:
 * 150-157): each calling thread keeps its own stream, staging buffers (device and pinned host, grown on demand, so a
 * call allocates nothing once its sizes have been seen) and kernel status word, and waits only for its own stream. */
int qnt_quantize_q8_host(const float* x, int n, int8_t* q, float* d);
int qnt_matvec_host(const qnt_dtensor* W, const int8_t* qx, const float* dx, int r0, int r1, float* out);
int qnt_matmul_host(const qnt_dtensor* W, const int8_t* qx, const float* dx, int n, int r0, int r1, float* out, int ldo,
                    int impl);

/* ---------------------------------------------------------------- around a decoder layer's products
 *
 * For models that a caller composes of the operators of this file: the engine's own layers fuse the reference's forms of these
 * (engine/src/ops_ref.cpp:69-83, 194-199), whose sums are in element order, bit for bit.  Device pointers; work is queued on `stream` (a
 * cudaStream_t, NULL = legacy default); nothing is allocated, so the calls can be captured into a graph. */

/* RMS norm with the residual's addition, 8-bit rows out (the operand of qnt_matvec / qnt_matmul):
 *   h = x + residual (f32; residual := h, rounded to its type; NULL: h = x),  y = h / sqrt(mean h^2 + eps) * weight,
 *   per 32 values: d = max |y| / 127,  q = y / d to the nearest integer, halves away from zero.
 * x [n_tok][n] at x_stride, of dtype QNT_F32, QNT_F16 or QNT_BF16; residual [n_tok][n] at residual_stride, of x's dtype or
 * QNT_F32, which does not overlap x; weight f32 [n]; q [n_tok][n] and d [n_tok][n / 32], 16-byte aligned; n a multiple of 32, at most 32768.
 * Sums are in f32.  A row reads as NaN where a value of h, or its sum of squares, is not finite (the sum is, for a root mean square
 * below 1.8e19 / sqrt(n), which is 10^17 or more), a block where a weight is not; a block whose d is below 2^-126 reads as zeros.
 * Squares below 2^-126 lose bits: with eps = 0 the root mean square should be 10^-18 or more. */
int qnt_rms_norm_q8(const void* x, int dtype, long long x_stride, void* residual, int residual_dtype, long long residual_stride,
                    const float* weight, float eps, int n_tok, int n, int8_t* q, float* d, void* stream);

/* The values q * d of 8-bit rows (the inverse of qnt_quantize_q8 and qnt_rms_norm_q8): out [n_tok][n] of dtype, 16-byte aligned
 * like q; one rounding of the f32 product. */
int qnt_dequantize_q8(const int8_t* q, const float* d, int n_tok, int n, void* out, int dtype, void* stream);

/* Rotary positions of query and key heads (either may be NULL with 0 heads): pair i of a head's first rotary_dim dims, (i, i +
 * rotary_dim / 2) or, interleaved, (2 i, 2 i + 1), turns by positions[t] * turns[i] revolutions and is multiplied by `scale`; the
 * dims behind are copied.  Token t, head h, dim i at t * stride + h * head_dim + i (elements) of dtype QNT_F32, QNT_F16 or QNT_BF16; an
 * output may be its input (with one stride), and must not overlap it otherwise, nor the other output or input.  turns: f64
 * [rotary_dim / 2] = frequency / (2 pi), with whatever scaling for long contexts; the revolution count is formed in f64, so that far
 * positions keep their angles.  positions int32 [n_tok], of any sign.  head_dim even, at most 1024. */
int qnt_rope(const void* q, long long q_stride, void* q_out, long long q_out_stride, int n_heads, const void* k, long long k_stride,
             void* k_out, long long k_out_stride, int n_kv_heads, int dtype, int head_dim, int rotary_dim, int interleaved,
             const double* turns, float scale, const int* positions, int n_tok, void* stream);

/* The selection of a beam search's next step: of each group's candidates (b, t), beam b < beams and token t < vocab,
 *     s(b, t) = scores[group][b] + logit(b, t) - log sum_u exp(logit(b, u))
 * the k best: out_scores, tokens and parents (the beams) [groups][k], best first, equal ones by the lowest b * vocab + t.
 * logits: row group * beams + b at that times stride (elements), of dtype QNT_F32, QNT_F16 or QNT_BF16.  ended (may be NULL)
 * [groups][beams]: such a beam has one candidate, its own score with token end_id.  Candidates that are -inf or no numbers (a
 * forbidden token, a row with NaN or +inf, a score that is not finite) come behind all others, with score -inf, in order of their
 * places.  Scores are formed and compared in f64.  k <= 64, beams <= 1024, vocab <= 2^30, beams * vocab < 2^31.
 * workspace: qnt_beam_workspace bytes, 16-byte aligned, contents irrelevant.  Results overlap neither the inputs nor each other. */
size_t qnt_beam_workspace(int groups, int beams, int vocab, int k);
int qnt_beam_select(const void* logits, int dtype, long long stride, const float* scores, const uint8_t* ended, int end_id,
                    int groups, int beams, int vocab, int k, float* out_scores, int* tokens, int* parents, void* workspace,
                    size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------- model level (engine/src/model.h) */

typedef struct qnt_model qnt_model;

/* HeadQuery (engine/src/model.h:20-29). */
typedef struct qnt_head_query {
    int top_k;        /* 0 = full head */
    int n_valid;      /* ids >= n_valid are padding (0 = whole vocab) */
    const int* must;  /* ids whose logits must also be exact (e.g. penalized history) */
    int n_must;
} qnt_head_query;

/* HParams (engine/src/model_file.h:40-45). */
typedef struct qnt_hparams {
    int vocab_size, dim, n_layers, n_heads, n_kv_heads, head_dim, ffn_dim, max_seq;
    float rope_theta, norm_eps;
    int tied_embeddings, qkv_bias;
    uint32_t flags;
    int n_tokens;  /* tokenizer vocabulary (Tokenizer::n_tokens, engine/src/tokenizer.h:24) */
    int ctx_len;   /* KV cache positions of this model handle */
    int has_shortlist;
} qnt_hparams;

/* Model::load (engine/src/model.h:35): mmaps the .qnt, uploads every tensor once to HBM in the device layout and
 * allocates one sequence's f16 KV cache for ctx_len positions (<= 0: the file's max_seq).  flags: 0, or
 * QNT_OPEN_NIBBLE_SCREEN: the Exact Shortlist Head screens with the high nibble plane of the Q8 output head (built at
 * load: rows * cols / 2 bytes, plus an f16 norm per row and 32-block of the dropped low nibbles) instead of the
 * file's quanta.head_q4 / quanta.head_err (not uploaded), and a file
 * without those tensors gets a shortlist head too.  Exact rows, tau and the sampled ids are those of the full head
 * either way; the coarse / upper scores and the count of exact rows differ.  No reference counterpart (the
 * reference's research notes, docs/PROGRESS.md:121-130, describe the screen). */
#define QNT_OPEN_NIBBLE_SCREEN 1
int qnt_model_open(const char* path, int ctx_len, int flags, qnt_model** out);
void qnt_model_close(qnt_model* m);
int qnt_model_hparams(const qnt_model* m, qnt_hparams* out);

/* Model::forward (engine/src/model.h:39): one token at pos (positions fed in order), then the head for hq (NULL or
 * top_k <= 0: full head).  logits: host buffer of vocab_size floats or NULL.  QNT_ERR_RANGE if pos >= ctx_len. */
int qnt_model_forward(qnt_model* m, int token, int pos, const qnt_head_query* hq, float* logits);

/* Model::forward_batch (engine/src/model.h:44): n tokens at pos0..pos0+n-1 (device chunks of up to 512 tokens; the
 * results do not depend on the chunking); logits of the last. */
int qnt_model_forward_batch(qnt_model* m, const int* tokens, int n, int pos0, const qnt_head_query* hq, float* logits);

/* Model::head (engine/src/model.h:47) for the last token; coarse / upper (may be NULL) receive the shortlist pass's
 * 4-bit scores and upper bounds (Model::head_coarse / head_upper, model.h:50-51). */
int qnt_model_head(qnt_model* m, const qnt_head_query* hq, float* logits, float* coarse, float* upper);

/* The sum behind the CLI's `ppl` (tools/cli/main.cpp:261-282): Model::forward of ids[0..n-2] in order from position 0
 * (full head), and for each p the full-vocabulary -log softmax of ids[p + 1] over ids < n_tokens, summed in f64 into
 * *nll; perplexity = exp(*nll / (n - 1)).  Leaves the KV cache holding those positions. */
int qnt_model_nll(qnt_model* m, const int* ids, int n, double* nll);

/* Model::last_head_rows / has_shortlist_head / kv_cache_bytes (engine/src/model.h:48-49,58). */
int qnt_model_last_head_rows(const qnt_model* m);
int qnt_model_has_shortlist(const qnt_model* m);
size_t qnt_model_kv_cache_bytes(const qnt_model* m);
size_t qnt_model_weight_bytes(const qnt_model* m);

/* A copy of the .qnt at in_path, written to out_path, with the device's fused matrices stored pre-packed beside the
 * original tensors (which stay byte for byte, so the reference's ModelFile reads the copy as it reads the original:
 * engine/src/model_file.cpp:189-211 looks tensors up by name and ignores the rest).  Added, per layer l:
 * b200.layers.<l>.qkv (q|k|v rows pair-interleaved per head), b200.layers.<l>.gate_up (gate|up interleaved per 32
 * rows), b200.layers.<l>.qkv_bias (files with q|k|v biases), and the marker b200.layout (f32 [1], the layout
 * version).  qnt_model_open uploads those tensors as they are instead of reordering rows on the host.  The writer of
 * the format is scripts/export.py:290-315; this is its extension point (no reference counterpart).  QNT_ERR_IO if
 * in_path does not open or out_path cannot be written. */
int qnt_export_device_layout(const char* in_path, const char* out_path);
/* How many fused tensors the last qnt_model_open took pre-packed from the file (0 for a plain .qnt).  A pre-packed
 * tensor counts only when it holds the file's own rows in the fused order (shape and a sample of rows checked; the
 * q|k|v bias in full); otherwise that layer's rows are fused at load. */
int qnt_model_packed_tensors(const qnt_model* m);

/* ---------------------------------------------------------------- session + sampling (engine/src/session.h, sampler.h) */

/* SamplerParams (engine/src/sampler.h:9-18). */
typedef struct qnt_sampler_params {
    float temperature; /* <= 0: greedy */
    int top_k;         /* 0 = disabled (every candidate), as in the reference */
    float top_p, min_p;
    float repeat_penalty;
    int repeat_window; /* 0 = whole history */
    uint64_t seed;     /* 0 = fixed default seed (the reference uses the clock) */
} qnt_sampler_params;

typedef struct qnt_gen_stats {
    double prefill_ms, decode_ms;  /* device time (CUDA events) */
    long long head_rows, head_calls;
    int kernels_per_step;
} qnt_gen_stats;

#define QNT_GEN_SHORTLIST 1     /* Session::set_sampler: use the Exact Shortlist Head when the file has one */
#define QNT_GEN_BATCH_PREFILL 2 /* Session::set_batch_prefill(true) */
#define QNT_GEN_KEEP_RNG 4      /* qnt_session_begin: keep the previous session's xorshift state (a Chat::reset keeps
                                   its Sampler) instead of starting from the seed */

/* Session::feed + Session::generate (engine/src/session.cpp:13-52) with Sampler::sample (sampler.cpp:22-85) on the
 * device: prefill the prompt, then n_gen steps of sample -> append -> forward without host round trips.
 * Writes the sampled ids to out_ids and returns how many (or < 0). */
int qnt_generate(qnt_model* m, const int* prompt, int n_prompt, const qnt_sampler_params* sp, int flags, int n_gen,
                 int* out_ids, qnt_gen_stats* stats);

/* The same loop in pieces, for callers that drive decoding step by step (and for timing exactly K steps):
 * qnt_session_begin = Session::feed of the prompt (engine/src/session.cpp:13-31) with the sampler configured;
 * qnt_session_step  = n iterations of Session::generate's loop body (session.cpp:45-53), queued on the model's stream
 *                     (returns without waiting; at most ctx_len - 1 positions in total);
 * qnt_session_read  = waits for the queued steps and copies the sampled ids (returns how many). */
int qnt_session_begin(qnt_model* m, const int* prompt, int n_prompt, const qnt_sampler_params* sp, int flags);
int qnt_session_step(qnt_model* m, int n);
int qnt_session_read(qnt_model* m, int* out_ids, int max_ids, qnt_gen_stats* stats);

/* The rest of Session (engine/src/session.cpp:13-52) for multi-turn use (Chat::reply, session.cpp:94-118):
 *   qnt_session_feed    Session::feed after the first: appends n ids to the history and prefills them at the next
 *                       positions (the same results as feeding them with the first prompt); the sampler state carries on.
 *   qnt_session_rewind  forgets the last n_drop history tokens -- a sampled stop token, which the reference never
 *                       appends (session.cpp:41-42); the next call on the session must be a feed.
 *   qnt_session_last    waits for the queued steps; *token = the last sampled id, *length = the history length. */
int qnt_session_feed(qnt_model* m, const int* ids, int n);
int qnt_session_rewind(qnt_model* m, int n_drop);
int qnt_session_last(qnt_model* m, int* token, int* length);

/* Text <-> ids (engine/src/tokenizer.h:15-39): byte-level BPE over the .qnt's tokenizer section, on the host (no GPU).
 *   qnt_tokenizer_open  Tokenizer(ModelFile::tokenizer()): QNT_ERR_IO for an unreadable file or a vocabulary without
 *                       all 256 byte tokens
 *   qnt_tokenize        Tokenizer::encode (special literals such as "<|im_start|>" recognised): returns the id count and
 *                       writes at most max_ids of them
 *   qnt_token_piece     Tokenizer::decode(id): the raw bytes (possibly part of a UTF-8 sequence); returns their count and
 *                       writes at most cap of them (an unknown id has none)
 *   qnt_token_id        Tokenizer::token_id: a special token's id, or -1 */
typedef struct qnt_tokenizer qnt_tokenizer;
int qnt_tokenizer_open(const char* path, qnt_tokenizer** out);
void qnt_tokenizer_free(qnt_tokenizer* t);
int qnt_tokenizer_n_tokens(const qnt_tokenizer* t);
int qnt_tokenize(const qnt_tokenizer* t, const char* text, size_t len, int* ids, int max_ids);
int qnt_token_piece(const qnt_tokenizer* t, int id, char* buf, int cap);
int qnt_token_id(const qnt_tokenizer* t, const char* literal);

/* Batched serving of many independent sequences on one model (the multi-sequence API qnt_prefill_batch /
 * qnt_decode_batch of the drop-in boundary; the reference serves one Session at a time, engine/src/session.cpp:13-52).
 * Each sequence has its own f16 KV cache; a decode step advances n distinct sequences by one token each through the
 * tensor-core matmul (tokens as the matmul's N), and the greedy head is one tensor-core pass over the Q8 lm_head with
 * the argmax fused (Sampler::sample at temperature 0: the first maximum over ids < n_valid).
 *   qnt_batch_init     allocates the caches of max_seqs sequences of ctx_len positions (lengths reset to 0)
 *   qnt_prefill_batch  feeds n prompt tokens to sequence seq; *next_id = its greedy next token (may be NULL)
 *   qnt_decode_batch   n <= 512 distinct sequences, tokens[i] appended to seq_ids[i]; next_ids[i] its greedy next token
 *   qnt_batch_reset    forgets sequence seq (length 0) */
int qnt_batch_init(qnt_model* m, int max_seqs, int ctx_len);
int qnt_prefill_batch(qnt_model* m, int seq, const int* tokens, int n, int* next_id);
int qnt_decode_batch(qnt_model* m, const int* seq_ids, const int* tokens, int n, int* next_ids);
int qnt_batch_reset(qnt_model* m, int seq);
/* Batched serving from the paged 8-bit KV cache (qnt_kv_cache): sequences take pages of page_tokens positions from one pool
 * of n_pages as they grow, at a bit more than half of the f16 caches' bytes per position, and share a common prefix.
 *   qnt_batch_init_paged  instead of qnt_batch_init; prefill, decode and reset are the same calls.  A call that would need
 *                         more pages than are free returns QNT_ERR_RANGE and leaves its sequences as they were (a prefill
 *                         of more than 512 tokens: with those of its 512-token chunks that found room).  A token id outside
 *                         the embedding is QNT_ERR_DEVICE as above, and changes nothing.  After any other QNT_ERR_DEVICE or
 *                         QNT_ERR_CUDA the call's sequences have its positions without their values: reset them
 *   qnt_batch_fork        the empty sequence dst takes over src's positions: full pages are shared, a part-filled last page
 *                         is copied
 *   qnt_batch_resize      the pages in use are moved together and into a pool of n_pages, which replaces the old one
 *                         (QNT_ERR_RANGE: more are in use) */
int qnt_batch_init_paged(qnt_model* m, int max_seqs, int ctx_len, int n_pages, int page_tokens);
int qnt_batch_fork(qnt_model* m, int src, int dst);
int qnt_batch_resize(qnt_model* m, int n_pages);

/* Beam search from the paged cache (qnt_batch_init_paged; sequences 0 .. beams - 1 empty, before and after the call; no
 * counterpart in the reference): the prompt, then up to n_gen steps of qnt_beam_select over all beams' logits, qnt_kv_reorder and
 * one batched decode step.  A beam that takes end_id (-1: none) ends with it and stays with its score; the search stops when all
 * have.  ids [beams][n_gen], lens and scores (sums of log-probabilities) [beams], best first.  beams <= 64; n + n_gen - 1 positions. */
int qnt_beam_search(qnt_model* m, const int* prompt, int n, int beams, int n_gen, int end_id, int* ids, int* lens, float* scores);

/* Sampler (engine/src/sampler.h:20-38): Sampler::sample (sampler.cpp:22-85) on logits that are already in device
 * memory -- repetition penalty -> greedy argmax (first max) or top-k -> softmax(T) -> min-p -> top-p -> xorshift64*
 * draw, with the reference's float operations, so the same logits, history and seed give the same ids.
 *   qnt_sampler_create  = Sampler(const SamplerParams&): the xorshift state starts at (seed ? seed : fixed) | 1, on the
 *                         current device.  Any top_k: up to 32 the candidates come from per-CTA lists; top_k 0 (disabled)
 *                         or above 32 sorts every logit below n_valid on the device (scratch of 16 B per id, allocated
 *                         on first use and kept by the sampler).
 *   qnt_sampler_sample  = Sampler::sample(float* logits, int n_valid, const std::vector<int>& history): `logits` is a
 *                         DEVICE array of at least n_valid floats and is edited in place like the reference's (the
 *                         penalised ids); `history` is a host array of n_history ids.  Work is queued on `stream`
 *                         (a cudaStream_t, NULL = legacy default); the call waits for it and writes the id to *token.
 *   qnt_sampler_free    = ~Sampler. */
typedef struct qnt_sampler qnt_sampler;
int qnt_sampler_create(const qnt_sampler_params* sp, qnt_sampler** out);
int qnt_sampler_sample(qnt_sampler* s, float* logits, int n_valid, const int* history, int n_history, int* token,
                       void* stream);
void qnt_sampler_free(qnt_sampler* s);

/* No counterpart in the reference: qnt_sampler_sample without a sampler object and without allocating memory, for
 * callers that cannot allocate -- a serving process whose device memory is reserved up front by its own pool (weights
 * and KV pages), where a cudaMalloc fails or fragments that pool, and a token loop that must not stall other streams,
 * as cudaMalloc / cudaFree can synchronise the device.  Same kernels and results as qnt_sampler_sample.
 *   *rng_state: the xorshift64* state, in/out; start it at (seed ? seed : any nonzero) | 1 as Sampler's constructor
 *               does (sampler.cpp:10-13); each call advances it exactly like the sampler object's.
 *   Limits: n_valid <= 262144, n_history <= 32768, 1 <= top_k <= 32 when temperature > 0; larger sizes return
 *           QNT_ERR_INVALID with the limit in qnt_last_error().
 *   Scratch: one static device array of 459,008 bytes per device (sampler state, candidate lists, history copy and
 *            penalty marks) plus a static 4 MiB copy of the host exp table.  The marks must be all zero when a call
 *            starts: they start zeroed, every completed call clears the ones it set, and a call that fails after
 *            setting them clears them (a stream-ordered memset) before it returns its error.  Calls whose GPU work
 *            overlaps (other host threads, or other streams) share that scratch and race: serialise them.
 *   The first call on each device does the set-up, with that device current: cudaGetSymbolAddress of the scratch and
 *            of the table, and a synchronous copy of the exp table into it.  Make that first call before any stream
 *            capture begins.  Every call copies its parameters and history through pageable host memory, waits for
 *            its stream (cudaStreamSynchronize) and writes the id to *token. */
int qnt_sampler_sample_noalloc(const qnt_sampler_params* sp, uint64_t* rng_state, float* logits, int n_valid,
                               const int* history, int n_history, int* token, void* stream);

/* ---------------------------------------------------------------- paged 8-bit KV cache
 *
 * No counterpart in the reference (its cache is one dense f16 array per sequence, engine/src/model.h:58): a cache of many
 * sequences in pages, int8 codes with one f32 scale for each block of 16 tokens, K or V, layer and kv head, in device
 * memory that the caller owns.  value = code * scale.
 *   codes   [n_pages][n_layers][2: K, V][n_kv_heads][page_tokens * head_dim], 16-byte aligned; within a page the K tile is
 *           [head_dim / 16][page_tokens][16 dims] and the V tile [page_tokens / 16][head_dim][16 tokens]
 *   scales  [n_pages][n_layers][2][n_kv_heads][page_tokens / 16]
 *   refs    [n_pages]: how many sequences use the page (0: free)
 *   table   [max_seqs][max_pages]: the page of positions k * page_tokens .. of a sequence, -1 past its pages
 *   lens    [max_seqs]: positions of the sequence; it holds ceil(len / page_tokens) pages
 *           (refs, table and lens change through the calls below: a length lowered by hand would lose its pages)
 *   status  one word of error bits that kernels set (qnt_kv_check reports and clears them)
 * An empty cache: refs and lens 0, table -1, status 0; codes and scales need no initial values.  An append makes scales of 0 and
 * above; the caller may write scales of either sign.
 * Limits: head_dim 64 or 128; page_tokens 16, 32, 64 or 128; n_pages <= 1048576; max_seqs <= 8192.
 *
 * Every call queues its work on `stream` (a cudaStream_t, NULL = legacy default) and returns.  All pointers are device
 * pointers, sequence lists included.  Calls that write a cache must be ordered against every other call on it (one stream,
 * or events); workspaces belong to one call at a time.  Nothing is allocated, so the calls can be captured into a graph. */
typedef struct qnt_kv_cache {
    int n_layers, n_kv_heads, head_dim, page_tokens;
    int n_pages, max_seqs, max_pages;
    int8_t* codes;
    float* scales;
    int* refs;
    int* table;
    int* lens;
    unsigned* status;
} qnt_kv_cache;

/* Page operations.  Free pages are taken from the lowest index up, in the order of the list.  A call whose list is not
 * valid, or that needs more pages than are free, changes nothing and sets an error bit.
 *   qnt_kv_reserve  lens[seqs[i]] += extra[i] and the pages for it (distinct sequences)
 *   qnt_kv_fork     sequence dst[i] (empty) becomes a copy of src[i]: full pages are shared (refs + 1), a part-filled last
 *                   page is copied in every layer, so that both can go on; distinct dst, none of them also a src
 *   qnt_kv_free     the sequences give back their pages (refs - 1) and become empty (distinct sequences)
 *   qnt_kv_reorder  sequence seqs[i] becomes what sequence seqs[i - i % group + parents[i]] was before the call (n distinct
 *                   sequences in whole groups; 0 <= parents[i] < group): a beam search's step.  Full pages are shared; a
 *                   part-filled last page goes to one child (the parent itself if it goes on, else the first), the others
 *                   get copies of its filled blocks of 16 positions, in every layer; pages that nothing uses any more
 *                   are given back, to this call's copies first.  Its workspace: qnt_kv_reorder_workspace bytes.
 *   qnt_kv_compact  the n pages in use move to indices 0 .. n - 1 (only those at or past n move); table and refs follow
 *   qnt_kv_copy     page src[i]'s codes and scales, all layers, over page dst[i]'s (no dst twice, none also a src)
 * workspace: qnt_kv_page_workspace bytes, 16-byte aligned, contents irrelevant. */
size_t qnt_kv_page_workspace(const qnt_kv_cache* cache);
int qnt_kv_reserve(const qnt_kv_cache* cache, const int* seqs, const int* extra, int n, void* workspace, size_t workspace_bytes,
                   void* stream);
int qnt_kv_fork(const qnt_kv_cache* cache, const int* src, const int* dst, int n, void* workspace, size_t workspace_bytes,
                void* stream);
size_t qnt_kv_reorder_workspace(const qnt_kv_cache* cache);
int qnt_kv_reorder(const qnt_kv_cache* cache, const int* seqs, const int* parents, int n, int group, void* workspace,
                   size_t workspace_bytes, void* stream);
int qnt_kv_free(const qnt_kv_cache* cache, const int* seqs, int n, void* stream);
int qnt_kv_compact(const qnt_kv_cache* cache, void* workspace, size_t workspace_bytes, void* stream);
int qnt_kv_copy(const qnt_kv_cache* cache, const int* src, const int* dst, int n, void* stream);

/* Rows of a call: n distinct sequences, tokens starts[j] .. starts[j + 1] - 1 (of n_tok) belong to sequence seqs[j]
 * (starts: n + 1 ascending ints from 0 to n_tok).
 *   qnt_kv_append     quantizes rows into one layer.  A sequence's m new tokens are its last m positions (reserve first;
 *                     then append in every layer): token i goes to position lens[seq] - m + i.  k, v: token t, head h,
 *                     dim d at t * stride + h * head_dim + d, of dtype QNT_F32, QNT_F16 or QNT_BF16; max_new bounds m.
 *                     Per block of 16 tokens, K or V, and head: d = max(the block's scale if it holds earlier tokens,
 *                     max |x| * (1 / 127), in f32); earlier codes are rounded to the new scale, new codes are round(x / d).  A
 *                     non-finite value makes its block read as NaN.
 *   qnt_kv_read       values of positions first[j] + i of sequence seqs[j] to rows starts[j] + i of k_out and v_out,
 *                     [n_tok][n_kv_heads][head_dim] of dtype (16-byte aligned)
 *   qnt_kv_attention  out[t][h] = softmax attention of query row t, head h over its sequence's cache in one layer: query i
 *                     of a sequence's m sits at p = lens[seq] - m + i and sees positions max(0, p - window + 1) .. p
 *                     (window 0: 0 .. p).  scores are scaled by `scale`; head h reads kv head h / (n_heads /
 *                     n_kv_heads).  q: token t, head h, dim d at t * q_stride + h * head_dim + d; out [n_tok][n_heads]
 *                     [head_dim] of the same dtype, 16-byte aligned; lse (may be NULL) [n_tok][n_heads] f32: log of the
 *                     sum of exp(score).  A query that sees nothing gets out 0 and lse -inf.  max_q bounds m; max_len
 *                     bounds lens (a longer sequence is still read whole, only less evenly spread).  lse is of the scores
 *                     alone; a V scale that is not finite makes out NaN where it is seen, a query that is not finite
 *                     makes out NaN.  (Weights carry up to 2^64 in f32: V below 2^40 in magnitude cannot overflow on the
 *                     way.)
 *                     workspace: qnt_kv_attention_workspace bytes for the same counts, 16-byte aligned, contents
 *                     irrelevant. */
int qnt_kv_append(const qnt_kv_cache* cache, int layer, const void* k, const void* v, int dtype, long long k_stride,
                  long long v_stride, const int* seqs, const int* starts, int n, int n_tok, int max_new, void* stream);
int qnt_kv_read(const qnt_kv_cache* cache, int layer, const int* seqs, const int* first, const int* starts, int n, int n_tok,
                void* k_out, void* v_out, int dtype, void* stream);
size_t qnt_kv_attention_workspace(const qnt_kv_cache* cache, int n_heads, int n, int n_tok, int max_q, int max_len);
int qnt_kv_attention(const qnt_kv_cache* cache, int layer, const void* q, int dtype, long long q_stride, int n_heads,
                     const int* seqs, const int* starts, int n, int n_tok, int max_q, int max_len, float scale, int window,
                     void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream);

/* Waits for `stream`, then reports (and clears) the error bits of earlier calls on this cache: QNT_ERR_DEVICE with the
 * reason in qnt_last_error(). */
int qnt_kv_check(const qnt_kv_cache* cache, void* stream);

/* Diagnostics (no reference counterpart): copies an internal buffer of the last forward as floats -- 0 roped q,
 * 1 attention output, 2 residual x (of the last layer, before the final norm), 3 quantized SwiGLU output, 4 its block
 * scales, 5 the head's quantized input.  Returns the element count. */
int qnt_model_debug_buffer(qnt_model* m, int what, float* out);

/* The cudaStream_t (as void*) every call on this model is queued on: lets a caller record CUDA events around
 * qnt_session_step for device timing. */
void* qnt_model_stream(const qnt_model* m);

/* Diagnostics (no reference counterpart): the dense int8 tensor-core rate of the current GPU, measured -- every SM
 * issues 4 * iters back-to-back tcgen05.mma.kind::i8 (M 128, N 256, K 32) on operands resident in shared memory;
 * *tops = int8 TOP/s over the slowest SM.  The roofline denominator of the tensor-core matmul. */
int qnt_bench_mma_i8(int iters, double* tops);

/* Diagnostics (no reference counterpart): runs the tensor-core matmul's bounded wait on an mbarrier that nothing
 * completes, with `limit` tries (1..2^20; each try may sleep up to 20 us), on `stream`.  The wait runs out, the kernel
 * records the timeout in the calling thread's status word and returns, and the call reports it as QNT_ERR_DEVICE --
 * the path a real timeout takes, shown without a fault; the context stays usable. */
int qnt_wait_probe(unsigned limit, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QUANTA_B200_H */
