/*
 * tgsample.h -- C ABI of the B200 batched logits-processing and sampling engine.
 *
 * Drop-in boundary for the sarthak-fleet/tinygpt sampling step: the step that
 * turns the last-position logits of a batch into one token id per row.  Every
 * entry point takes plain pointers and sizes, returns an int32 status
 * (TG_OK = 0, negative on error), never throws and never exits the process.
 * A SwiftPM target binds it through a module map, Python through ctypes.
 *
 * Reference interfaces this ABI replaces (paths are inside sarthak-fleet/tinygpt):
 *   tg_sample        <- TinyGPT.generate sampling block   python_ref/model.py:213-224
 *                    <- tg_generate sampling tail         wasm/src/model.cpp:489-517
 *                       (C ABI declared at wasm/src/model.h:39-43)
 *                    <- sampleToken                       native-mac/Sources/TinyGPTServe/Serve.swift:1483-1506
 *                    <- repetition penalty + top-k        native-mac/Sources/TinyGPTApp/ModelController.swift:262-304
 *                    <- LogitsMasker.mask (as a bitmask)  native-mac/Sources/TinyGPTModel/ConstrainedGen.swift:775-837
 *   tg_spec_verify   <- SpeculativeDecode.stepStochastic  native-mac/Sources/TinyGPT/SpeculativeDecode.swift:121-210
 *                    <- SpeculativeDecode.step (greedy)   native-mac/Sources/TinyGPT/SpeculativeDecode.swift:41-98
 *
 * Beyond the reference (it keeps one sequence's contiguous cache and samples only):
 *   tg_cache_*, tg_tree_attention, tg_tree_masks   a paged key/value cache and the
 *                       attention of drafted trees over it
 *   tg_beam_*           beam search's selection over beams and vocabulary
 *
 * Memory: all array arguments of tg_sample / tg_spec_verify are DEVICE pointers
 * on the sampler's device, owned by the caller.  The *_host variants take host
 * pointers and stage through buffers the handle owns.  Threading: one handle
 * per device; a handle is not shared between threads without external locking,
 * and serves one stream at a time: its candidate buffer, status word, counters
 * and statistics are per handle, so calls on one handle from two streams that
 * can overlap on the GPU race (use one handle per stream).
 * Allocation: tg_sample allocates nothing (its buffers are made by
 * tg_sampler_create); tg_spec_verify and tg_sample_sharded use buffers made by
 * tg_sampler_reserve and return TG_ERR_UNSUPPORTED for calls beyond them.
 *
 * Semantics (bit-exact definition, restated by the CPU oracle):
 *   y[v]   = logits[v] (bf16 widened exactly to fp32)
 *   penalties, for each distinct id t in the row's history (count c_t):
 *            if repetition_penalty > 1: y = y > 0 ? y / rp : y * rp
 *            if presence or frequency != 0: y = y - (frequency * c_t + presence)
 *   mask   : state_id >= 0 and bit v of mask_table[state_id] clear -> y = -inf
 *   greedy : temperature <= 0 -> first index of max y (-1 if every y is -inf)
 *   s[v]   = y[v] / temperature
 *   top-k  : 0 < top_k < vocab -> keep s >= k-th largest s (ties kept)
 *   mass   : q[v] = trunc(tg_exp(s[v] - max s) * 2^44) as uint64 (exact sums)
 *   top-p  : top_p < 1 -> order survivors by (s desc, id asc), keep the shortest
 *            prefix whose mass reaches top_p * total mass
 *   min-p  : min_p > 0 -> keep q >= min(min_p, 1) * 2^44 (the top survivor has q = 2^44)
 *   draw   : r = trunc(u * S) over the final mass S; first id in INDEX order whose
 *            inclusive running mass exceeds r.
 */
#ifndef TGSAMPLE_H
#define TGSAMPLE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---------------------------------------------------------- */
#define TG_OK                 0
#define TG_ERR_INVALID_ARG   -1  /* bad pointer, size, dtype or parameter         */
#define TG_ERR_CUDA          -2  /* a CUDA runtime call failed                    */
#define TG_ERR_UNSUPPORTED   -3  /* size beyond a compiled limit                  */
#define TG_ERR_NO_DEVICE     -4  /* device index not present                      */
#define TG_ERR_DEVICE_STATUS -5  /* a kernel reported a data error (see below)    */
#define TG_ERR_COLLECTIVE    -6  /* a collective missed its deadline; the communicator was aborted */

/* ---- dtypes of the logits and caches --------------------------------------------------- */
#define TG_DTYPE_F32   0
#define TG_DTYPE_BF16  1
#define TG_DTYPE_F16   2  /* caches only */

/* ---- per-row sampling parameters (32 bytes, POD) ---------------------------
 * temperature <= 0 selects greedy.  top_k <= 0 or >= vocab disables top-k.
 * top_p >= 1 disables top-p.  min_p <= 0 disables min-p.
 * repetition_penalty <= 1 disables the CTRL penalty; presence / frequency
 * penalties of 0 disable them.  flags is reserved and must be 0.            */
typedef struct tg_row_params {
  float   temperature;
  float   top_p;
  float   min_p;
  float   repetition_penalty;
  float   presence_penalty;
  float   frequency_penalty;
  int32_t top_k;
  int32_t flags;
} tg_row_params;

/* Compiled limits. */
#define TG_MAX_VOCAB    (1 << 20)  /* ids must fit in 20 bits                  */
#define TG_MAX_HISTORY  4096       /* history entries per row                  */

typedef struct tg_sampler tg_sampler;

/* Version of this ABI: (major << 16) | minor. */
int32_t tg_abi_version(void);

/* Message for the last error raised on the calling thread ("" if none). */
const char* tg_last_error_string(void);

/* Create a sampler bound to CUDA device `device` for rows of `vocab` logits and
 * at most `max_batch` rows per call.  Allocates the device scratch and the host
 * staging used by the *_host variants; when vocab > 2816 and max_batch >= 1024
 * also the candidate buffer of the two-kernel mode (used for calls of 1024 rows
 * or more), min(max_batch, 2048) rows of
 * 22,536 bytes (46 MB at 2048 rows; environment TG_SAMPLE_SPLIT=0 at creation
 * turns the mode and the buffer off).  Replaces tg_model_create's role as the
 * owner of sampling state (wasm/src/model.h:21-23); returns TG_OK and *out. */
int32_t tg_sampler_create(int32_t device, int32_t vocab, int32_t max_batch,
                          tg_sampler** out);
int32_t tg_sampler_destroy(tg_sampler* s);

/* Sample one token per row.  Device pointers:
 *   logits       [batch, row_stride] of dtype (row_stride >= vocab, in elements)
 *   params       [batch] tg_row_params
 *   history      [batch, history_stride] int32 ids (may be NULL if history_len is NULL)
 *   history_len  [batch] int32, 0..min(history_stride, TG_MAX_HISTORY) (NULL: no history)
 *   mask_table   [num_states, ceil(vocab/32)] uint32, bit set = token allowed (NULL: no masks)
 *   state_id     [batch] int32, -1 = unmasked row (NULL: no masks)
 *   uniforms     [batch] float in [0,1) (ignored for greedy rows)
 *   out_ids      [batch] int32; -1 where no token is admissible
 *   out_probs    [batch] float probability of the chosen id under the final
 *                distribution (1 for greedy rows), may be NULL
 * Asynchronous on `stream` (a cudaStream_t, NULL = legacy default stream);
 * allocates nothing.  The launch shape depends on the batch and never changes
 * a result: 8..148 rows run one 1024-thread CTA per row; 1024 rows or more run
 * two kernels (the stream to the handle's candidate buffer, then selection);
 * other batches run one 256-thread CTA per row.
 * Replaces: python_ref/model.py:213-224, wasm/src/model.cpp:489-517,
 *           Serve.swift:1483-1506, ModelController.swift:262-304. */
int32_t tg_sample(tg_sampler* s, const void* logits, int32_t dtype,
                  int64_t row_stride, int32_t batch, const tg_row_params* params,
                  const int32_t* history, const int32_t* history_len,
                  int32_t history_stride, const uint32_t* mask_table,
                  int32_t num_states, const int32_t* state_id,
                  const float* uniforms, int32_t* out_ids, float* out_probs,
                  void* stream);

/* Same as tg_sample with every array in HOST memory (pinned or pageable).
 * Copies the inputs into the handle's device staging, samples, copies the ids
 * (and probabilities) back and synchronizes before returning.  This is the call
 * a host-side caller with no device memory of its own makes (the Swift serve
 * loop's per-token sampleToken, Serve.swift:1483-1506). */
int32_t tg_sample_host(tg_sampler* s, const void* logits, int32_t dtype,
                       int64_t row_stride, int32_t batch,
                       const tg_row_params* params, const int32_t* history,
                       const int32_t* history_len, int32_t history_stride,
                       const uint32_t* mask_table, int32_t num_states,
                       const int32_t* state_id, const float* uniforms,
                       int32_t* out_ids, float* out_probs);

/* Speculative-decoding verification (rejection sampling), one call per batch.
 * Device pointers:
 *   target_logits [batch, K+1, vocab] of dtype (position K is the bonus position)
 *   draft_logits  [batch, K, vocab] of dtype
 *   draft_ids     [batch, K] int32 proposals
 *   temperature   [batch] float; <= 0 selects greedy verification
 *                 (SpeculativeDecode.swift:41-98), > 0 stochastic with
 *                 T = max(temperature, 1e-5) (SpeculativeDecode.swift:121-210)
 *   u_accept      [batch, K] float uniforms for the accept tests
 *   draft_logits and u_accept may both be NULL (greedy verification without a
 *   draft distribution: Medusa / EAGLE heads, MedusaHeads.swift:186-265,
 *   EagleDraft.swift:216-290); a stochastic row then ends without a token
 *   (out_n = 0) and sets device status bit 4
 *   u_draw        [batch] float uniform for the residual / bonus draw
 *   out_ids       [batch, K+1] int32: accepted proposals then the final token;
 *                 entries past out_n are set to -1
 *   out_n         [batch] int32: number of valid entries (1..K+1)
 * Accept iff u <= min(1, pT(tok) / max(pD(tok), 1e-10)).  On the first reject
 * the final token is drawn from max(0, pT - pD) renormalised when its mass
 * exceeds 1e-10, else from pT; after K accepts it is the bonus drawn from pT at
 * position K.  Probabilities are q / sum(q) with q the exact masses above.
 * Needs statistics reserved by tg_sampler_reserve(s, >= K, ...). */
int32_t tg_spec_verify(tg_sampler* s, const void* target_logits,
                       const void* draft_logits, int32_t dtype, int32_t batch,
                       int32_t K, const int32_t* draft_ids,
                       const float* temperature, const float* u_accept,
                       const float* u_draw, int32_t* out_ids, int32_t* out_n,
                       void* stream);

/* Grammar-masked verification: tg_spec_verify under the constraint of a
 * grammar (mask table as in tg_sample, rows from tg_grammar_state_row).
 * state_ids [batch, K+1] int32 device array: the grammar state before the token
 * of each position (position i's state follows the draft tokens 0..i-1; -1 =
 * unmasked position).  At position i an element whose bit is clear counts as
 * -inf in both the target and the draft rows, so both distributions are
 * renormalised over the allowed tokens, and a disallowed proposal is rejected.
 * A position with no allowed token ends the row without a token (greedy rows:
 * id -1).  A state id >= num_states leaves its position unmasked and sets
 * device status bit 0.  No counterpart in the reference: its speculative paths
 * verify without the grammar mask (docs/constrained_generation.md:243-246). */
int32_t tg_spec_verify_masked(tg_sampler* s, const void* target_logits,
                              const void* draft_logits, int32_t dtype, int32_t batch,
                              int32_t K, const int32_t* draft_ids, const float* temperature,
                              const float* u_accept, const float* u_draw,
                              const uint32_t* mask_table, int32_t num_states,
                              const int32_t* state_ids, int32_t* out_ids, int32_t* out_n,
                              void* stream);

/* Allocation-free variant of tg_spec_verify.  No counterpart in the reference.
 * For callers that cannot call cudaMalloc: for example a serving process that
 * reserved all free HBM for its KV cache at start-up (a cudaMalloc would fail),
 * or a decode loop that must not pay the device-wide synchronization cudaMalloc
 * and cudaFree may cause.  It takes no handle and allocates nothing: the
 * per-position statistics live in a fixed array inside the library, sized for
 * batch * (2K + 1) <= TG_STATIC_SPEC_MAX_ROWS vocab rows (larger calls return
 * TG_ERR_UNSUPPORTED).  Every GPU that loads the library holds that array
 * (about 128 KiB) until the process exits.  The first call on a device looks up
 * the array's device address with that device current; make that first call
 * before any stream capture.  All calls on a device share the array, so calls
 * that overlap on the GPU (different streams without ordering) race.
 * Arguments and results are those of tg_spec_verify, on CUDA device `device`;
 * data errors (bits 1 and 4 of the device status word) are kept in a status
 * word inside the same array, cleared at the start of every call and read by
 * tg_spec_verify_static_status. */
#define TG_STATIC_SPEC_MAX_ROWS 8192
int32_t tg_spec_verify_static(int32_t device, int32_t vocab, const void* target_logits,
                              const void* draft_logits, int32_t dtype, int32_t batch,
                              int32_t K, const int32_t* draft_ids,
                              const float* temperature, const float* u_accept,
                              const float* u_draw, int32_t* out_ids, int32_t* out_n,
                              void* stream);

/* Status bits of the last tg_spec_verify_static call on `device` (meaning as
 * tg_sampler_device_status); synchronizes the device, clears the word,
 * allocates nothing.  No counterpart in the reference. */
int32_t tg_spec_verify_static_status(int32_t device, uint32_t* out_bits);

/* Makes the buffers of the calls that need more than tg_sampler_create's:
 * verification statistics for max_batch rows of up to max_K proposals
 * (tg_spec_verify, tg_spec_verify_masked) and, when max_ranks > 0, the record
 * storage of tg_sample_sharded for communicators of up to max_ranks ranks
 * ((max_ranks + 1) x max_batch x 10,256 bytes).  Buffers only grow.  Call it
 * before the hot loop (and before any stream capture); the hot calls then
 * allocate nothing.  No counterpart in the reference (its C ABI has no
 * device buffers, wasm/src/model.h:39-43). */
int32_t tg_sampler_reserve(tg_sampler* s, int32_t max_K, int32_t max_ranks);

/* ---- vocab-sharded mode (one process per GPU, each owning a vocab slice) ----
 * For vocabularies or batches where one GPU should not hold whole rows: rank r
 * holds ids [vocab_offset, vocab_offset + vocab) of every row (vocab = the
 * handle's vocab).  tg_sample_shard_local writes one record per row: the local
 * survivors of top-k (every local value >= the local k-th, ties kept, global
 * ids) or, for greedy rows, the local first maximum.  The caller all-gathers the
 * records of all ranks (e.g. ncclAllGather / torch.distributed over NVLink) into
 * [nshards][batch] order and every rank calls tg_sample_shard_merge, which
 * returns exactly what tg_sample returns on the whole rows.  Supported rows:
 * greedy, or 0 < top_k <= 1024 (others: id -1 and device status bit 2).
 * No counterpart call exists in the reference (its sampler is single-device);
 * the semantics are those of tg_sample. */
#define TG_SHARD_CAP 1280
typedef struct tg_shard_cand { float value; int32_t id; } tg_shard_cand;
typedef struct tg_shard_record {
  int32_t count;   /* entries in cand; -1: row not supported in sharded mode */
  int32_t flags;   /* bit 0: more than TG_SHARD_CAP local survivors        */
  float absent_max; /* an upper bound of the local values not in cand     */
  int32_t reserved;
  tg_shard_cand cand[TG_SHARD_CAP];
} tg_shard_record;

/* Local half: arguments as tg_sample for this rank's slice (history ids and
 * mask bit positions are global; mask_table rows span full_vocab bits).
 * out_records: [batch] device records. */
int32_t tg_sample_shard_local(tg_sampler* s, int32_t vocab_offset, int32_t full_vocab,
                              const void* logits, int32_t dtype, int64_t row_stride,
                              int32_t batch, const tg_row_params* params,
                              const int32_t* history, const int32_t* history_len,
                              int32_t history_stride, const uint32_t* mask_table,
                              int32_t num_states, const int32_t* state_id,
                              tg_shard_record* out_records, void* stream);

/* Merge half: records [nshards][batch] (gathered), the same params and
 * uniforms on every rank; writes ids / probabilities as tg_sample.  The handle
 * needs max_batch >= batch (its vocab is not used). */
int32_t tg_sample_shard_merge(tg_sampler* s, const tg_shard_record* records, int32_t nshards,
                              int32_t full_vocab, int32_t batch, const tg_row_params* params,
                              const float* uniforms, int32_t* out_ids, float* out_probs,
                              void* stream);

/* Vocab-sharded sampling in one call: the local half (this handle's vocab is the
 * slice [vocab_offset, vocab_offset + vocab) of rows of full_vocab ids), one
 * ncclAllGather of the per-row records over `nccl_comm` (an ncclComm_t of
 * nranks ranks, this rank's slice in rank order), and the merge, all on
 * `stream`; every rank gets the same ids.  Arguments otherwise as tg_sample,
 * for this rank's slice of every row.  NCCL is not linked: ncclAllGather is
 * looked up in the NCCL the process has loaded (TG_ERR_UNSUPPORTED if none).
 * Record storage comes from tg_sampler_reserve(s, ..., >= nranks); nranks must
 * equal the communicator's size (checked with ncclCommCount).  With a collective
 * timeout set (tg_sampler_set_collective_timeout) the call waits on the host for
 * the all-gather and, when it misses the deadline (a rank that left), aborts the
 * communicator (ncclCommAbort) and returns TG_ERR_COLLECTIVE; with none (the
 * default) it only enqueues.  Limits as the two halves
 * (tg_sample_shard_local / tg_sample_shard_merge).  No counterpart in the
 * reference, which samples every row on one device. */
int32_t tg_sample_sharded(tg_sampler* s, void* nccl_comm, int32_t nranks, int32_t vocab_offset,
                          int32_t full_vocab, const void* logits, int32_t dtype, int64_t row_stride,
                          int32_t batch, const tg_row_params* params, const int32_t* history,
                          const int32_t* history_len, int32_t history_stride,
                          const uint32_t* mask_table, int32_t num_states, const int32_t* state_id,
                          const float* uniforms, int32_t* out_ids, float* out_probs, void* stream);

/* Deadline of tg_sample_sharded's all-gather in milliseconds (0: no host wait,
 * the default).  The reference has no collective (single device). */
int32_t tg_sampler_set_collective_timeout(tg_sampler* s, int32_t timeout_ms);

/* Device error word of the last completed call on this handle (synchronizes
 * the handle's device).  Bit 0: a state_id outside [0, num_states);
 * bit 1: a draft id outside [0, vocab); bit 2: a row the vocab-sharded mode
 * could not resolve (unsupported parameters, more than TG_SHARD_CAP local
 * survivors, or a top-k threshold tie between shards); bit 3: a bounded wait
 * of the opt-in fused sampling kernel (TG_FUSED=1) gave up (its rows are
 * unreliable); bit 4: a stochastic row in a verification called without
 * draft logits (it ends without a token).  Cleared by this call. */
int32_t tg_sampler_device_status(tg_sampler* s, uint32_t* out_bits);

/* Per-handle path counters of tg_sample (diagnostics, the device-side analogue
 * of the reference's per-token constraint timing, Serve.swift:1489-1491):
 *   [0] rows finished from the shared-memory candidate list
 *   [1] rows whose candidate list overflowed      -> full-row path
 *   [2] rows with fewer than k candidates         -> full-row path
 *   [3] rows whose top-k threshold fell below the candidate bound -> full-row path
 *   [4] rows processed by the full-row path (any reason)
 *   [5] candidates appended (sum over rows; single-kernel mode)
 *   [6] rows of [0] finished by the warp-group finisher (calls of >= 1024 rows)
 *   [7] rows the warp-group finisher left because its shared-memory pool was full
 * Copies min(n, TG_PATH_COUNTERS) counters (synchronizes the device); zeroes
 * them when reset != 0. */
#define TG_PATH_COUNTERS 8
int32_t tg_sampler_path_counters(tg_sampler* s, uint64_t* out, int32_t n, int32_t reset);

/* Kernel timing of tg_sample (diagnostics): with enable != 0 every later
 * tg_sample call on this handle records CUDA events around its kernels.  Each
 * call of this function first reports the last recorded call (synchronizing on
 * it): *out_kernels = 2 with out_ms[0] the streaming and out_ms[1] the
 * finishing kernel of the two-kernel mode, 1 with out_ms[0] the whole call, 0
 * if none was recorded; then applies `enable`.  out_ms ([2]) and out_kernels
 * may be NULL. */
int32_t tg_sampler_profile(tg_sampler* s, int32_t enable, float* out_ms, int32_t* out_kernels);

/* ---------------------------------------------------------------------------
 * Grammar compiler (host only; no GPU needed): grammar text -> byte-level
 * automaton -> per-state token bitmasks, the rows of tg_sample's mask_table.
 * Replaces the reference's constrained-decoding stack:
 *   ServeGrammarSpec.parse / ServeConstraint / ServeTokenMasker
 *     (native-mac/Sources/TinyGPTServe/Serve.swift:1903-2056),
 *   JSONSchemaNode (native-mac/Sources/TinyGPTModel/JSONSchema.swift:1-117),
 *   JSONSchemaFSM / LogitsMasker (native-mac/Sources/TinyGPTModel/ConstrainedGen.swift:35-837),
 *   PaceToolTagFSM (Serve.swift:2057-2233, grammars/pace-tool-tags.gbnf).
 * Grammar text: after trimming whitespace, text starting with '{' is a JSON
 * Schema (minified JSON only; object keys limited to the declared properties
 * not yet emitted; required keys before '}'; string enum / minLength /
 * maxLength; integer vs number; no trailing commas); a GBNF text holding
 * `root ::=` and `[POINT:` is the tool-tag grammar; anything else is
 * TG_ERR_UNSUPPORTED.
 *
 * Vocabulary: token i is bytes token_bytes[token_offsets[i] .. token_offsets[i+1]).
 * A token is allowed iff the automaton accepts all of its bytes; empty tokens
 * never are.  Once the document is complete only eos_id is allowed (none if
 * eos_id is -1, as in the serve masker). */
#define TG_GRAMMAR_JSON_SCHEMA 0
#define TG_GRAMMAR_TOOL_TAGS 1
typedef struct tg_grammar tg_grammar;
typedef struct tg_grammar_state tg_grammar_state;

const char* tg_grammar_last_error(void);
int32_t tg_grammar_create(const char* grammar_text, int64_t text_len, int32_t vocab,
                          const uint8_t* token_bytes, const int64_t* token_offsets,
                          int32_t eos_id, tg_grammar** out);
int32_t tg_grammar_destroy(tg_grammar* g);
int32_t tg_grammar_kind(tg_grammar* g, int32_t* kind);
/* A fresh automaton at the document start (one per generated sequence). */
int32_t tg_grammar_state_create(tg_grammar* g, tg_grammar_state** out);
int32_t tg_grammar_state_clone(const tg_grammar_state* s, tg_grammar_state** out);
int32_t tg_grammar_state_destroy(tg_grammar_state* s);
/* Feed raw bytes, all or nothing (JSONSchemaFSM.acceptBytes). */
int32_t tg_grammar_accept_bytes(tg_grammar_state* s, const uint8_t* bytes, int64_t n,
                                int32_t* accepted);
/* Advance by a sampled token's bytes (LogitsMasker.commit); *accepted = 0
 * leaves the state unchanged. */
int32_t tg_grammar_commit(tg_grammar_state* s, int32_t token, int32_t* accepted);
int32_t tg_grammar_is_complete(const tg_grammar_state* s, int32_t* out);
/* The state's mask into out_words[ceil(vocab/32)] (bit i%32 of word i/32 = token i). */
int32_t tg_grammar_mask(const tg_grammar_state* s, uint32_t* out_words);
/* The state's row in the grammar's mask table: automaton states with equal
 * futures share a row; the row is computed and appended the first time such a
 * state is seen (*is_new = 1).  The value to put in tg_sample's state_id. */
int32_t tg_grammar_state_row(const tg_grammar_state* s, int32_t* row, int32_t* is_new);
/* The host table (rows x ceil(vocab/32) words, row-major) to upload as
 * tg_sample's mask_table; valid until the next tg_grammar_state_row. */
int32_t tg_grammar_table(tg_grammar* g, const uint32_t** words, int32_t* rows);

/* ---------------------------------------------------------------------------
 * Paged key/value cache: what a decoder keeps between the calls of tg_sample,
 * tg_spec_verify and tg_beam_select.  No counterpart in the reference, whose
 * cache is one sequence's contiguous array (its KVCache).
 *
 * Keys and values live in two pools [layers, num_pages, kv_heads, page_size,
 * head_dim] that the caller owns; the handle owns the bookkeeping, all of it in
 * device memory: per sequence slot a length, a number of pages and a row of page
 * ids (-1 past that number), per page the number of rows that hold it.  Every call
 * is asynchronous on `stream`, reads its row arguments from device memory,
 * allocates nothing and never waits for the host, so a decode step whose lengths
 * are decided on the device (tg_cache_accept) needs no round trip and can be
 * captured in a CUDA graph.  Results do not depend on timing: a call that needs
 * pages takes the lowest-numbered free ones, row after row.
 *
 * A call's `seqs` hold slots in [0, max_seqs), each at most once (tg_cache_fork's
 * `src` may repeat).  A row that cannot be served is left as it was and sets a
 * bit of the handle's status word (tg_cache_device_status):
 *   bit 0: a slot outside [0, max_seqs), or twice in a call that forbids it
 *   bit 1: not enough free pages (extend: rows are served in order until one
 *          does not fit; that row and the later ones that need pages get none)
 *   bit 2: a length past max_pages_per_seq pages, or a negative count or length
 *   bit 3: keys and values past the pages reserved by tg_cache_extend, or into a
 *          page that a fork still shares (not stored), or an advance past them
 *   bit 4: a bounded wait of tg_tree_attention gave up (its output is unreliable)
 *   bit 5: a tree whose node count is outside [0, nodes]
 * Threading and streams: as tg_sampler, one handle serves one stream at a time. */
#define TG_MAX_TREE_NODES 64

typedef struct tg_cache tg_cache;

typedef struct tg_cache_config {
  int32_t layers;
  int32_t kv_heads;
  int32_t head_dim;           /* a multiple of 8, 8..128                          */
  int32_t page_size;          /* tokens per page: a power of two, 8..256          */
  int32_t num_pages;
  int32_t max_seqs;           /* sequence slots                                   */
  int32_t max_pages_per_seq;
  int32_t dtype;              /* TG_DTYPE_BF16 or TG_DTYPE_F16                    */
} tg_cache_config;

/* Device addresses of the bookkeeping, to read (int32): lens [max_seqs], counts
 * [max_seqs] (pages held), tables [max_seqs, max_pages_per_seq], refs [num_pages]. */
typedef struct tg_cache_state {
  const int32_t* lens;
  const int32_t* counts;
  const int32_t* tables;
  const int32_t* refs;
} tg_cache_state;

/* k_pool, v_pool: device memory, 16-byte aligned, owned by the caller and kept
 * while the handle lives.  Every slot starts empty.  The handle's own memory: about
 * 16 bytes a page, 8 a table entry, 1.1 KB a slot, and 39 MB in which
 * tg_tree_attention joins what its blocks leave. */
int32_t tg_cache_create(int32_t device, const tg_cache_config* config, void* k_pool, void* v_pool,
                        tg_cache** out);
int32_t tg_cache_destroy(tg_cache* c);
int32_t tg_cache_get_state(tg_cache* c, tg_cache_state* out);

/* Status bits since the last call; synchronizes the device and clears them. */
int32_t tg_cache_device_status(tg_cache* c, uint32_t* out_bits);

/* Reserves pages so that row i can store counts[i] tokens past its length.  Where
 * those would start in a page that other rows hold too, the row gets a copy of
 * its part of that page, in every layer (of several such rows in one call that
 * are the page's only holders, the first keeps the page, and is served only if
 * all the others are).  seqs, counts: [n]. */
int32_t tg_cache_extend(tg_cache* c, int32_t n, const int32_t* seqs, const int32_t* counts, void* stream);

/* Slot dst[i] becomes a copy of slot src[i] as it was before the call (src[i] = -1:
 * empty), sharing its pages; pages that dst[i] alone held are freed.  All rows at
 * once: src may repeat, and src and dst may overlap, as when a beam search's
 * parents replace the beams.  dst's slots are distinct.  Tokens reserved but not
 * committed are not taken along; a row of the pair that stores tokens next reserves
 * them again (tg_cache_extend), since its last page may now be shared. */
int32_t tg_cache_fork(tg_cache* c, int32_t n, const int32_t* src, const int32_t* dst, void* stream);

/* Sets row i's length back to lens[i] (NULL: to 0) and frees its pages past it,
 * reserved ones included. */
int32_t tg_cache_truncate(tg_cache* c, int32_t n, const int32_t* seqs, const int32_t* lens, void* stream);

/* Advances row i's length by counts[i] tokens, already stored in reserved pages (a
 * slot that is given more than once, by each of its rows that still fits). */
int32_t tg_cache_commit(tg_cache* c, int32_t n, const int32_t* seqs, const int32_t* counts, void* stream);

/* Stores tokens' keys and values in one layer at row i's positions length ..
 * length + counts[i] - 1 (counts NULL: `tokens` for every row); the length stays
 * (tg_cache_commit).  k, v: [n, tokens, kv_heads, head_dim] of the cache's dtype with
 * the given strides in elements (row, token, head); the last dimension is contiguous. */
int32_t tg_cache_append(tg_cache* c, int32_t layer, int32_t n, const int32_t* seqs, const int32_t* counts,
                        int32_t tokens, const void* k, int64_t k_row, int64_t k_token, int64_t k_head,
                        const void* v, int64_t v_row, int64_t v_token, int64_t v_head, void* stream);

/* Attention of each row's drafted nodes over its cached tokens and over the nodes
 * themselves, in one layer; stores the nodes' keys and values at the row's positions
 * length + node (reserved by tg_cache_extend; the length stays).
 *   nodes     nodes per row in the arrays, 1..TG_MAX_TREE_NODES
 *   n_nodes   [n] nodes of each row (NULL: all); the others' outputs are 0 and
 *             nothing of them is read
 *   masks     [n, nodes] uint64: bit j of node i set = node i sees node j (its
 *             ancestors and itself, as the caller says; NULL: j <= i, a chain or
 *             a single token)
 *   q         [n, nodes, q_heads, head_dim], k, v [n, nodes, kv_heads, head_dim] of the
 *             cache's dtype; strides in elements (row, node, head)
 *   out       [n, nodes, q_heads, head_dim] contiguous, of the cache's dtype
 *   out_lse   [n, nodes, q_heads] float: log of the sum of exp(score) (NULL: none)
 * q_heads is a multiple of kv_heads, at most 256 times; query head h reads key head h /
 * (q_heads / kv_heads).  score = scale * q.k; softmax and sums in 32 bits, the weights rounded
 * to the cache's dtype for the product with the values.  A node that sees
 * nothing has output 0 and out_lse -inf.  A node's key or value influences only the
 * nodes that see it, infinities and NaN included. */
int32_t tg_tree_attention(tg_cache* c, int32_t layer, int32_t n, const int32_t* seqs, int32_t nodes,
                          const int32_t* n_nodes, const uint64_t* masks, int32_t q_heads,
                          const void* q, int64_t q_row, int64_t q_node, int64_t q_head,
                          const void* k, int64_t k_row, int64_t k_node, int64_t k_head,
                          const void* v, int64_t v_row, int64_t v_node, int64_t v_head,
                          float scale, void* out, float* out_lse, void* stream);

/* Settles a step over drafted trees.  Walks each tree from node 0 (the root, whose
 * token was accepted before): ids[node] is the token that the target model gives
 * after that node (tg_sample over all nodes' logits); the lowest-numbered child
 * with that token is taken next, until there is none.  The taken nodes' keys and
 * values, in every layer, move to positions length, length + 1, ...; the length
 * grows by their number and the pages past it are freed.
 *   parents   [n, nodes] int32: a node's parent (before the node; ignored for node 0)
 *   tokens    [n, nodes] int32: the drafted tokens (ignored for node 0)
 *   ids       [n, nodes] int32
 *   n_nodes   [n] (NULL: all)
 *   out_ids   [n, nodes] int32: the step's new tokens, ids along the path (the
 *             accepted ones, then the target's own); -1 past out_n
 *   out_n     [n] int32: their number, also the number of nodes taken
 * Needs the nodes' positions reserved (tg_cache_extend) and stored. */
int32_t tg_cache_accept(tg_cache* c, int32_t n, const int32_t* seqs, int32_t nodes, const int32_t* n_nodes,
                        const int32_t* parents, const int32_t* tokens, const int32_t* ids, int32_t* out_ids,
                        int32_t* out_n, void* stream);

/* masks[i] of tg_tree_attention from parents: bit i, and the bits of i's ancestors.
 * parents [n, nodes] as above; nodes past n_nodes (NULL: all) get 0. */
int32_t tg_tree_masks(int32_t n, int32_t nodes, const int32_t* n_nodes, const int32_t* parents,
                      uint64_t* masks, void* stream);

/* ---------------------------------------------------------------------------
 * Beam search: the selection of the next beams over beams and vocabulary, with
 * the reordering of their histories (tg_cache_fork reorders the caches).  The
 * reference has no beam search.
 *
 * For beam w of batch row b, row r = b * beams + w:
 *   x      = logits[r] (bf16 widened); a clear mask bit, or NaN: -inf; +inf: FLT_MAX
 *   lse    = max x + log(sum exp(x - max x)), rounded to fp32
 *   score  = fl(scores[r] + fl(x - lse)), for a finished beam scores[r] for the
 *            token pad_id alone; NaN counts as -inf
 * The `beams` best (score, then lowest w * vocab + token) with score > -inf are the
 * row's next beams in that order; fewer: parent -1, token -1, score -inf, finished. */
#define TG_MAX_BEAMS 32

typedef struct tg_beam tg_beam;

/* A handle for up to max_batch rows of `beams` beams; owns the workspace (one
 * stream at a time).  status bits: 0: a state id outside [0, num_states) (its row
 * is unmasked), 1: a history length outside [0, history_stride] (clamped). */
int32_t tg_beam_create(int32_t device, int32_t vocab, int32_t beams, int32_t max_batch, tg_beam** out);
int32_t tg_beam_destroy(tg_beam* h);
int32_t tg_beam_device_status(tg_beam* h, uint32_t* out_bits);

/* Device pointers; asynchronous on `stream`, allocates nothing.
 *   logits     [batch * beams, row_stride] of dtype (TG_DTYPE_F32 or TG_DTYPE_BF16)
 *   scores     [batch, beams] float
 *   finished   [batch, beams] int32, non-zero = finished (NULL: none)
 *   mask_table, num_states, state_id [batch * beams]: as tg_sample (NULL: no masks)
 *   eos_id     a beam that takes it is finished (-1: none); pad_id in [0, vocab)
 *   history    [batch * beams, history_stride] int32, history_len [batch * beams]
 *              (NULL: no histories), as tg_sample reads them
 *   out_parent, out_token [batch, beams] int32; out_score float; out_finished int32
 *              (may be NULL)
 *   out_history [batch * beams, history_stride], out_history_len: the parent's
 *              history, then the token unless the parent was finished or its
 *              history is full; -1 past the length.  Not the input arrays. */
int32_t tg_beam_select(tg_beam* h, const void* logits, int32_t dtype, int64_t row_stride, int32_t batch,
                       const float* scores, const int32_t* finished, const uint32_t* mask_table,
                       int32_t num_states, const int32_t* state_id, int32_t eos_id, int32_t pad_id,
                       const int32_t* history, const int32_t* history_len, int32_t history_stride,
                       int32_t* out_parent, int32_t* out_token, float* out_score, int32_t* out_finished,
                       int32_t* out_history, int32_t* out_history_len, void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* TGSAMPLE_H */
