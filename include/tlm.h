/*
 * tlm.h -- C ABI of the MI355X-native per-token decoder path of three-llm.
 *
 * Every compute entry point runs hand-written HIP kernels for gfx950.  All
 * functions return 0 (TLM_OK) or a negative TLM_ERR_* code; the message of the
 * last failure on the calling thread is tlm_last_error(), formatted like the
 * reference's errors ("Component: message").
 *
 * Reference interfaces replaced (paths relative to packages/three-llm/src/):
 *   ops      tsl/TSLLinear.ts:13-82, tsl/TSLRMSNorm.ts:18-81, tsl/TSLSiLUMul.ts:10-36,
 *            tsl/TSLGatedMLP.ts:17-90, tsl/TSLAttention.ts:19-449,
 *            tsl/TSLLogits.ts:40-69 and :201-274 (chunked logits + greedy sampler)
 *   runner   decoder/DecoderTSLRunner.ts:62-594 (computeToken :487-502,
 *            prefillTokens :504-530, readLogits :532-535, sampleToken :537-539,
 *            resetCache :541-546), driven by runtime/generate.ts:31-49.
 *
 * Device pointers are plain `void*`/`float*` obtained from tlm_alloc (or any
 * HIP allocation on the context's device).  Work is enqueued on the context's
 * stream; tlm_download / tlm_read_* / tlm_sync wait for it.  A context or model
 * must not be used from two threads at once.
 */
#ifndef TLM_H
#define TLM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TLM_ABI_VERSION 3

enum {
  TLM_OK = 0,
  TLM_ERR_INVALID = -1, /* bad argument (shape, range, null) */
  TLM_ERR_HIP = -2,     /* HIP runtime error */
  TLM_ERR_OOM = -3,     /* device allocation failed */
  TLM_ERR_STATE = -4,   /* call not valid in the current state */
  TLM_ERR_RANGE = -5    /* token or position out of range */
};

/* Weight storage formats (canonical host layouts):
 *   TLM_FMT_F16: uint16 fp16 bits, [N][K] row-major (row = output feature).
 *   TLM_FMT_Q4 : packed nibbles uint8 [N][K/2] (even k in the low nibble,
 *                value q+8 for q in [-8,7]) plus fp16 scales uint16 [N][K/32];
 *                w = f32(scale[n][k/32]) * q.  K must be a multiple of 32.
 *   TLM_FMT_F32: float [N][K] (embedding tables only). */
enum { TLM_FMT_F16 = 1, TLM_FMT_Q4 = 2, TLM_FMT_F32 = 3 };
/*   TLM_FMT_F8: 8-bit floating point (e4m3: sign, 4 bits of exponent, 3 of
 *                mantissa; up to 448, no infinities) with an fp32 scale, a power of
 *                two, for each 32 tokens and kv head (paged caches only). */
enum { TLM_FMT_F8 = 4 };

typedef struct tlm_ctx tlm_ctx;
typedef struct tlm_linear tlm_linear;
typedef struct tlm_attn tlm_attn;
typedef struct tlm_model tlm_model;
typedef struct tlm_paged tlm_paged;

/* ---------------------------------------------------------------- context */
int tlm_abi_version(void);
const char* tlm_last_error(void);
/* Opens device `device` (HIP ordinal) with one stream of default priority. */
int tlm_open(int device, tlm_ctx** out);
void tlm_close(tlm_ctx* ctx);
int tlm_sync(tlm_ctx* ctx);
/* Device name and compute-unit count (for reports). */
int tlm_device_info(tlm_ctx* ctx, char* name, size_t name_len, int* cu_count);
/* Free and total device memory of the context's GPU (hipMemGetInfo; for
 * reports and for checking that an entry point allocates nothing).  No
 * counterpart in the reference (the browser exposes no device memory). */
int tlm_device_memory(tlm_ctx* ctx, size_t* free_bytes, size_t* total_bytes);

/* Device buffers (thin helpers so hosts need no HIP binding of their own). */
int tlm_alloc(tlm_ctx* ctx, size_t bytes, void** dptr);
int tlm_free(tlm_ctx* ctx, void* dptr);
int tlm_upload(tlm_ctx* ctx, void* dst, const void* src, size_t bytes);   /* blocking */
int tlm_download(tlm_ctx* ctx, void* dst, const void* src, size_t bytes); /* waits for the stream */
/* Device-to-device copy enqueued on the context stream (bytes % 16 == 0): a
 * plain streaming kernel of known size.  A utility with no reference
 * counterpart (the reference copies through WebGPU buffers); it also scales
 * hardware byte counters against a known transfer. */
int tlm_copy(tlm_ctx* ctx, void* dst, const void* src, size_t bytes);

/* ------------------------------------------------------------------ linear
 * TSLLinear (tsl/TSLLinear.ts:13-82): y[n] = b[n] + sum_k W[n][k] x[k].
 * The reference takes fp32 W [in][out]; here W is fp16 or q4 in the canonical
 * [out][in] layout above, repacked at creation into the device tile layout. */
int tlm_linear_create(tlm_ctx* ctx, int fmt, int n_out, int k_in, const void* weights, const uint16_t* scales,
                      tlm_linear** out);
void tlm_linear_destroy(tlm_linear* lin);
/* Dequantizes the device copy back to fp32 [N][K] on the host (bit-exact
 * parity check of the device layout: q4 -> f32(s)*q, fp16 -> f32). */
int tlm_linear_dequant(tlm_linear* lin, float* host_out);
/* y = bias + W x.  x: fp32[K] device, bias: fp32[N] device or NULL, y: fp32[N] device. */
int tlm_op_linear(tlm_linear* lin, const float* x, const float* bias, float* y);
/* The same linear over `rows` tokens at once, as one MFMA GEMM (the batched
 * prefill's linear; the reference applies TSLLinear once per replayed token,
 * DecoderTSLRunner.ts:472-480).  x: fp16 bits device [rows][K] (K % 32 == 0),
 * y: fp32 device [rows][N].  W is dequantised to fp16 ((code - 8) * s rounded
 * once), products accumulate in fp32.  x may start at any address; one that is no
 * multiple of 16 bytes costs a copy of the rows.  Enqueue only. */
int tlm_op_linear_rows(tlm_linear* lin, const uint16_t* x, int32_t rows, const float* bias, float* y);
/* How a batched linear of that size runs on `cus` compute units: plan[0] rows by
 * plan[1] columns of a block, plan[2] slices of K; us[0] the predicted time of
 * that choice, us[1] of the best one on another block size (inf: none weighed).
 * partial: the partial sums of the batched prefill (QKV, O and down GEMM),
 * else tlm_op_linear_rows.  Host only: needs no device; for tests and reports,
 * without a counterpart in the reference. */
int tlm_rows_plan(int fmt, int partial, int32_t rows, int32_t n_out, int32_t k_in, int32_t cus, int32_t* plan,
                  float* us);

/* ----------------------------------------------------------- element ops */
/* TSLRMSNorm (tsl/TSLRMSNorm.ts:18-81): y = x * rsqrt(mean(x^2) + eps) * (offset ? 1 + w : w). */
int tlm_op_rmsnorm(tlm_ctx* ctx, const float* x, const float* w, int n, double eps, int offset, float* y);
/* TSLSiLUMul (tsl/TSLSiLUMul.ts:10-36): out = silu(gate) * up. */
int tlm_op_silu_mul(tlm_ctx* ctx, const float* gate, const float* up, int n, float* out);
/* TSLGatedMLP (tsl/TSLGatedMLP.ts:17-90), SwiGLU: y = down(silu(gate x) * (up x)).
 * gate_up holds 2*I rows (gate rows then up rows), down is [H][I]. */
int tlm_op_gated_mlp(tlm_linear* gate_up, tlm_linear* down, const float* x, float* y);

/* --------------------------------------------------------------- attention
 * TSLAttention (tsl/TSLAttention.ts:19-449) for the Llama/Qwen2 recipe:
 * RoPE (rotate-half over rotary_dim, table from ropeParameters), KV append
 * at `position`, causal softmax attention over [max(0,pos-W+1), pos] with
 * grouped KV heads, split over the sequence with an online-softmax combine. */
typedef struct tlm_attn_desc {
  int32_t heads, kv_heads, head_dim, max_tokens;
  int32_t rotary_dim;       /* 0 disables RoPE */
  int32_t sliding_window;   /* 0 = full causal */
  int32_t kv_fmt;           /* TLM_FMT_F16 (default) or TLM_FMT_F32 */
  int32_t reserved;
  const float* inv_freq;    /* host, rotary_dim/2 entries (ropeParameters) */
  double attention_factor;  /* ropeParameters().attentionFactor */
  double attn_scale;        /* <= 0 selects 1/sqrt(head_dim) */
} tlm_attn_desc;

int tlm_attn_create(tlm_ctx* ctx, const tlm_attn_desc* desc, tlm_attn** out);
void tlm_attn_destroy(tlm_attn* attn);
/* qkv: fp32 device [(heads + 2 kv_heads) * head_dim] (packed Q|K|V, pre-RoPE);
 * out: fp32 device [heads * head_dim], anywhere, also over qkv.  q and the
 * probabilities are fp32, past 1024 positions over an fp16 cache (head_dim 64 or
 * 128) pairs of fp16 values: |q| * attn_scale * log2 e below 65520 there. */
int tlm_op_attention(tlm_attn* attn, const float* qkv, int position, float* out);
/* `rows` consecutive positions position0.. at once (the batched prefill's
 * attention; the reference runs TSLAttention once per replayed token): qkv fp32
 * device [rows][(heads + 2 kv_heads) * head_dim], bias included; RoPE, the K/V
 * rows appended to the cache, causal attention of each row over
 * [max(0, pos - W + 1), pos] on MFMA; out: fp16 bits device [rows][heads * head_dim].
 * Needs an fp16 cache and head_dim 64 or 128.  Waits for the stream. */
int tlm_op_attention_rows(tlm_attn* attn, const float* qkv, int32_t rows, int32_t position0, uint16_t* out);
/* Allocation-free tlm_op_attention_rows.  No counterpart in the reference: it
 * is for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops).  The same kernels and results; the rotated
 * fp16 queries are staged in a fixed 4 MiB device array of the library (one
 * per device, held until the process ends) instead of a buffer of the context
 * or one allocated per call, so rows * heads * head_dim * 2 may not exceed 4 MiB (TLM_ERR_RANGE
 * otherwise).  Enqueue only: no allocation, free or wait.  Every call on one
 * device shares that array, so calls that overlap on one device (other
 * streams or contexts) race. */
int tlm_op_attention_rows_noalloc(tlm_attn* attn, const float* qkv, int32_t rows, int32_t position0, uint16_t* out);
int tlm_attn_reset(tlm_attn* attn);
/* Cache rows [0, count) as fp32 [count][kv_heads*head_dim] (host). */
int tlm_attn_read_cache(tlm_attn* attn, int count, float* k_out, float* v_out);

/* ------------------------------------------------------- paged attention
 * TSLAttention's step (tsl/TSLAttention.ts:19-449: RoPE, KV append, causal
 * softmax attention with grouped KV heads and an optional sliding window) for
 * many sequences at once, whose keys and values lie in pages of a shared pool.
 * The reference keeps one sequence in one cache; the pages have no counterpart
 * there.  A handle holds a model's head shapes and RoPE table; the pools, the
 * page tables and the batch belong to the caller, so one handle serves every
 * layer. */
typedef struct tlm_paged_desc {
  int32_t heads, kv_heads, head_dim, max_tokens; /* head_dim 32, 64, 96 or 128; heads / kv_heads at most 16;
                                                    max_tokens: positions a sequence can have */
  int32_t rotary_dim;       /* 0 disables RoPE */
  int32_t sliding_window;   /* 0 = full causal */
  int32_t kv_fmt;           /* TLM_FMT_F16, TLM_FMT_F32 or TLM_FMT_F8 */
  int32_t page_tokens;      /* a power of two from 32 to 1024 */
  const float* inv_freq;    /* host, rotary_dim/2 entries (ropeParameters) */
  double attention_factor;  /* ropeParameters().attentionFactor */
  double attn_scale;        /* <= 0 selects 1/sqrt(head_dim) */
} tlm_paged_desc;

/* One step's rows.  Sequence s has `tokens` rows, of which the first counts[s]
 * are there (counts NULL: all), at the positions starts[s], starts[s] + 1, ...
 * A sequence with starts[s] < 0 or counts[s] < 1 is idle.  What rows
 * that are not there hold does not matter, and what the outputs hold for them stays.
 * Position p lies in page tables[s][p / page_tokens]; only the entries of
 * pages that hold a position in use are read (a window's earlier pages may be
 * given back, their entries anything).  Sequences may share pages that they
 * read; a position that two of them append to gets either's row.
 * All pointers are device memory; the struct itself is the host's and is read
 * during the call.  seqs * tokens * heads is at most 2^22. */
typedef struct tlm_paged_batch {
  void* k_pages;            /* pools of num_pages * kv_heads * page_tokens * head_dim kv_fmt elements (TLM_FMT_F8: */
  void* v_pages;            /* and scales; tlm_paged_page_bytes a page), 16-byte aligned and apart, in the order */
                            /* that tlm_paged_locate tells */
  const int32_t* tables;    /* [seqs][table_width] */
  const int32_t* starts;    /* [seqs] */
  const int32_t* counts;    /* [seqs] or NULL */
  int32_t num_pages, table_width, seqs, tokens;
} tlm_paged_batch;

int tlm_paged_create(tlm_ctx* ctx, const tlm_paged_desc* desc, tlm_paged** out);
void tlm_paged_destroy(tlm_paged* paged);
/* Bytes of a page in one pool.  Host only: needs no device. */
int tlm_paged_page_bytes(const tlm_paged_desc* desc, size_t* bytes);
/* Positions [0, sinks) stay visible behind a sliding window (attention sinks, a
 * system prompt): a row at position p attends to them and to (p - W, p].  For the
 * calls on the handle from here on; 0 at first.  Positions stay what they are. */
int tlm_paged_set_sinks(tlm_paged* paged, int32_t sinks);
/* One step's page tables from the lengths of its sequences.  Sequence s has
 * lengths[s] positions (< 0: it has ended) and wants min(counts[s], tokens) rows
 * more (counts NULL: tokens; < 1: none now).  It needs the pages of its new rows
 * and of what its next row sees: all before it, or its window and its sinks.
 * Pages that its table holds besides are given back: refs - 1.  Then the
 * sequences get the pages that they lack, in their order, the free ones (refs 0)
 * lowest first, refs 1, for as long as what they have lacked so far is no more than
 * what is free; one that it is not enough for keeps what it holds.  An entry
 * that is no page of the pool is none.  refs counts the tables that a page is in,
 * and holds of the caller's own (a prefix that is kept); pages may be shared, each
 * table counted, but for those that a sequence appends to.
 * starts: lengths[s] where the sequence's rows are served, else -1 (no rows
 * wanted, no pages left, or a page with positions that it needs below its length is
 * not held: tlm_paged_status reports that, and rows past max_tokens or
 * the table, which are left out).  slots (or NULL): page * page_tokens + token of
 * each row, -1 of those that are not there.  Entries that hold no page are -1.
 * tables, starts and counts are then a batch's.  All pointers are device memory;
 * the struct is the host's and read during the call. */
typedef struct tlm_paged_request {
  const int32_t* lengths;   /* [seqs] */
  const int32_t* counts;    /* [seqs] or NULL */
  const int32_t* tables;    /* [seqs][table_width], as they are */
  const int32_t* refs;      /* [num_pages] */
  int32_t* out_tables;      /* as they become: tables and refs themselves, or apart */
  int32_t* out_refs;        /* (what would be given, without giving it) */
  int32_t* starts;          /* [seqs] */
  int64_t* slots;           /* [seqs][tokens] or NULL */
  int32_t num_pages, table_width, seqs, tokens;
} tlm_paged_request;
/* seqs * tokens * heads is at most 2^22, seqs 2^20, num_pages 2^27, table_width
 * 2^26.  The results are apart from each other and from the inputs, but for tables
 * and refs in place.  Enqueue only. */
int tlm_op_paged_reserve(tlm_paged* paged, const tlm_paged_request* request);
/* qkv: fp32 [seqs][tokens][(heads + 2 kv_heads) * head_dim] (Q|K|V, bias
 * included, pre-RoPE).  The rotated K and the V rows go to their pages; q, when
 * not NULL: fp32 [seqs][tokens][heads * head_dim], the rotated queries.  qkv, q,
 * the pools and the batch's tables and lengths are apart.  Any number of tokens.
 * Enqueue only.
 * TLM_FMT_F8: a value is its code times the scale of its 32 aligned positions and kv
 * head, 2^e from 2^-32 to 2^31, the least that takes the largest magnitude to at
 * most 448.  Rows that start within 32 positions keep the scale that these have or, if
 * they need it, raise it; it never falls again, also where the rows that raised it are
 * dropped (drafts that fell).  The positions before them are then rounded again, exact
 * but for magnitudes below 2^-6 of the new scale: at most 2^-13.8 of the largest that it
 * was raised for.  Of rows that start within 32 positions
 * the earlier ones have been appended (or their page is all zeros).  Positions behind
 * the appended rows, to the end of their 32, keep their codes, not their values; 32
 * positions that two sequences append to in one call are lost.  Values that are not
 * finite become NaN, magnitudes past 448 * 2^31 become that. */
int tlm_op_paged_append(tlm_paged* paged, const tlm_paged_batch* batch, const float* qkv, float* q);
/* Attention of every row over positions [max(0, pos - W + 1), pos] of its
 * sequence, which the pages hold (append first).  q: fp32 [seqs][tokens]
 * [heads * head_dim], rotated; out: the same shape in out_fmt, TLM_FMT_F16 or
 * TLM_FMT_F32, apart from q and all that the batch names.  Scores and the weighted sum to 32 bits: an fp16
 * cache's products take q and the probabilities as pairs of fp16 values, each to
 * 2^-22 of itself or 2^-39 of its row's largest (an 8-bit cache's too, whose codes
 * are exact in fp16; there the probabilities times V's scales).  What masked
 * positions hold does not matter; attended K and V are finite.  Enqueue only. */
int tlm_op_paged_attention(tlm_paged* paged, const tlm_paged_batch* batch, const float* q, int out_fmt, void* out);
/* Waits for the stream and tells of what the calls since the last status met on
 * the device: TLM_ERR_RANGE where counts[s] was above `tokens`, a row's position
 * beyond max_tokens or its table (such rows were left out), or a table entry in
 * use was no page of the pool (its rows were not appended, its positions not
 * attended to; a row with no position left is zero). */
int tlm_paged_status(tlm_paged* paged);
/* Where element `dim` of `position` lies: its index in a K and in a V pool, from
 * a host copy of the sequence's table.  Host only: needs no device. */
int tlm_paged_locate(const tlm_paged_desc* desc, int32_t num_pages, const int32_t* table, int32_t table_width,
                     int32_t position, int32_t kv_head, int32_t dim, int64_t* k_index, int64_t* v_index);
/* TLM_FMT_F8: where the fp32 scale of `position` lies, in bytes from the start of a K
 * or a V pool.  Host only: needs no device. */
int tlm_paged_scale_at(const tlm_paged_desc* desc, int32_t num_pages, const int32_t* table, int32_t table_width,
                       int32_t position, int32_t kv_head, int64_t* byte);

/* ------------------------------------------------------------------ logits
 * TSLLogits chunk layers + greedy sampler (tsl/TSLLogits.ts:40-69, :201-274):
 * logits = head x; token = argmax, ties to the lower id.  logits may be NULL. */
int tlm_op_logits(tlm_linear* head, const float* x, float* logits, int32_t* token);
int tlm_op_argmax(tlm_ctx* ctx, const float* logits, int n, int32_t* token);
/* TSLLogitSampler candidate levels (tsl/TSLLogits.ts:276-330): the k best
 * (token, score) of logits[0, n) in the greedy order (higher score, ties to
 * the lower id), scores after the softcap cap * tanh(x / cap) when softcap > 0
 * (:185-191).  Entries at or below LOWEST_FLOAT (-inf, NaN included) never
 * take part; missing slots are (0, LOWEST_FLOAT).  1 <= k <= 16; device
 * tokens[k], scores[k].  Enqueue only. */
int tlm_op_topk(tlm_ctx* ctx, const float* logits, int n, int k, double softcap, int32_t* tokens, float* scores);
/* Penalties for repeated tokens, biases and masks on logits, for many sequences'
 * rows at once, before a token is picked (tlm_op_argmax, tlm_op_topk,
 * tlm_op_verify_drafts).  No counterpart in the reference, whose sampler takes the
 * logits as they are (TSLLogits.ts:185-191: but for a softcap).
 * Row j of sequence s follows its history and its drafts 0 .. j - 1; with c(v) the
 * times that token v is in these, in this order:
 *   c(v) > 0:  x = (x > 0 ? x / repetition : x * repetition) - presence - frequency * c(v)
 *   x = x + the biases of v (one listed twice: both, in the list's order)
 *   x = -inf where bit v % 32 of word v / 32 of the row's mask is 0.
 * -inf never takes part in picking; where a mask leaves nothing, no token does.
 * All three penalties count the same history.  Repetition over prompt and reply with
 * frequency and presence over the reply alone are two calls: the first with the whole
 * history and repetition only, the second with the reply's and all the rest.
 * Token ids outside the vocabulary are nobody's. */
typedef struct tlm_logit_rules {
  const float* logits;           /* [seqs][tokens][vocab] */
  float* out;                    /* the same shape: logits itself, or apart from all inputs */
  const int32_t* counts;         /* [seqs] rows that are there (NULL: tokens); the others' results stay */
  const int32_t* history;        /* [seqs][history_width] */
  const int32_t* history_counts; /* [seqs] tokens of it that are there (NULL: all) */
  const int32_t* drafts;         /* [seqs][tokens - 1], or NULL: none counts */
  const float* repetition;       /* [seqs], above 0 (NULL: 1) */
  const float* frequency;        /* [seqs] (NULL: 0) */
  const float* presence;         /* [seqs] (NULL: 0) */
  const int32_t* bias_ids;       /* [seqs][bias_width] */
  const float* biases;           /* [seqs][bias_width] */
  const uint32_t* masks;         /* [seqs][tokens][(vocab + 31) / 32] (NULL: nothing is masked) */
  int32_t seqs, tokens, vocab, history_width, bias_width;
} tlm_logit_rules;
/* tokens <= 64, vocab <= 524288, seqs * tokens <= 2^20, bias_width <= 4096,
 * history_width <= 2^30; seqs * tokens * vocab, vocab rounded up to a multiple of 4096, below 2^35.
 * Enqueue only. */
int tlm_op_adjust_logits(tlm_ctx* ctx, const tlm_logit_rules* rules);
/* Verification of drafted tokens, for many sequences at once: which of a
 * sequence's drafts the target's distribution lets stand, and the token after
 * them.  No counterpart in the reference (it samples one token at a time,
 * TSLLogits.ts:336-383); without drafts (tokens = 1) it is that sampling over
 * the whole vocabulary.
 * logits: fp32 [seqs][tokens][vocab]; of sequence s the first counts[s] rows
 * (NULL: tokens; < 1: idle, its results stay as they are) are there, row j
 * following the drafts 0 .. j - 1, so it has counts[s] - 1 drafts.
 * drafts: [seqs][tokens - 1]; draft_logits: fp32 [seqs][tokens - 1][vocab], what
 * they were drawn from, or NULL: drafted for certain (a lookup, a greedy model).
 * uniforms: fp32 [seqs][tokens] in [0, 1).  With p_j and q_j the softmax of
 * logits / temperature, draft x_j stands where uniforms[s][j] q_j(x_j) < p_j(x_j)
 * (q_j(x_j) = 1 without draft_logits); at the first that does not, the lowest
 * token whose running sum of max(p_j - q_j, 0) passes uniforms[s][tokens - 1] of
 * the whole is drawn (of p_j where nothing is left), after the last draft from
 * p_j; sums in 64 bits.  temperature 0: a draft stands where it is the row's
 * argmax (ties to the lower id), which the row gives otherwise; draft_logits and
 * uniforms are not read.  Temperatures up to 1e-6 count as 1e-6 (math.ts:527-547).
 * Entries at or below LOWEST_FLOAT (-inf, NaN included) never take part; a draft
 * outside the vocabulary never stands; a row without entries gives -1.
 * accepted: [seqs] drafts that stand; out_tokens: [seqs][tokens] those, the token
 * after them, then -1; both apart from the inputs and each other.  tokens <= 64, vocab <= 524288;
 * 12 bytes for every 2048 entries of 4096 sequences' rows fit the context's 32 MiB
 * (TLM_ERR_RANGE otherwise).  Enqueue only. */
int tlm_op_verify_drafts(tlm_ctx* ctx, const float* logits, const float* draft_logits, const int32_t* drafts,
                         const int32_t* counts, const float* uniforms, int32_t seqs, int32_t tokens, int32_t vocab,
                         double temperature, int32_t* accepted, int32_t* out_tokens);

/* ------------------------------------------------------------------- model */
typedef struct tlm_model_desc {
  int32_t hidden_size, intermediate_size, num_layers, num_heads, num_kv_heads, head_dim, vocab_size;
  int32_t max_tokens;
  int32_t rotary_dim;
  int32_t sliding_window;
  int32_t linear_fmt;  /* TLM_FMT_Q4 or TLM_FMT_F16 for the decoder linears */
  int32_t head_fmt;    /* TLM_FMT_F16 or TLM_FMT_Q4 for an untied LM head */
  int32_t embed_fmt;   /* TLM_FMT_F16 or TLM_FMT_F32 embedding table */
  int32_t kv_fmt;      /* TLM_FMT_F16 or TLM_FMT_F32 cache */
  int32_t qkv_bias;    /* 1: upload TLM_T_BQKV per layer */
  int32_t tied;        /* 1: LM head = embedding table (fp16 embedding only) */
  double rms_eps;
  double attention_factor;
  const float* inv_freq; /* host, rotary_dim/2 entries */
  /* ABI 2.  DecoderCPURunner.attention (decoder/DecoderCPURunner.ts:140-160)
   * passes recipe.attnScale and the block's slidingWindow per layer
   * (DecoderWeights.ts:307-311: sliding_attention layers get the recipe's
   * window, full_attention layers 0 when the config lists layer types). */
  double attn_scale;             /* <= 0 selects 1/sqrt(head_dim) (attnScale undefined) */
  const int32_t* layer_windows;  /* host, num_layers entries (0 = full causal), copied at
                                    create; NULL: every layer uses sliding_window */
} tlm_model_desc;

enum {
  TLM_T_EMBED = 0,      /* [V][H] embed_fmt */
  TLM_T_LM_HEAD = 1,    /* [V][H] head_fmt (untied only) */
  TLM_T_LM_HEAD_SCALES = 2,
  TLM_T_FINAL_NORM = 3, /* fp32 [H] */
  TLM_T_ATTN_NORM = 4,  /* fp32 [H] per layer */
  TLM_T_FFN_NORM = 5,   /* fp32 [H] per layer */
  TLM_T_WQKV = 6,       /* [(Hq+2Hkv)*D][H], rows Q|K|V */
  TLM_T_WQKV_SCALES = 7,
  TLM_T_BQKV = 8,       /* fp32 [(Hq+2Hkv)*D] */
  TLM_T_WO = 9,         /* [H][Hq*D] */
  TLM_T_WO_SCALES = 10,
  TLM_T_WGATE = 11,     /* [I][H] */
  TLM_T_WGATE_SCALES = 12,
  TLM_T_WUP = 13,       /* [I][H] */
  TLM_T_WUP_SCALES = 14,
  TLM_T_WDOWN = 15,     /* [H][I] */
  TLM_T_WDOWN_SCALES = 16
};

/* Flags of tlm_compute_token. */
enum { TLM_LOGITS = 1 };

int tlm_model_create(tlm_ctx* ctx, const tlm_model_desc* desc, tlm_model** out);
void tlm_model_destroy(tlm_model* model);
/* Copies a canonical host tensor to the device (the caller keeps ownership,
 * like uploadAndReleaseStaticWeights in tsl/releaseCPU.ts:79-110). */
int tlm_model_upload(tlm_model* model, int tensor, int layer, const void* host, size_t bytes);
/* Builds the per-token HIP graphs; implicit on the first compute. */
int tlm_model_finalize(tlm_model* model);
/* computeToken (DecoderTSLRunner.ts:487-502): enqueue one token at `position`.
 * With TLM_LOGITS the LM head and the greedy argmax run too. */
int tlm_compute_token(tlm_model* model, int32_t token, int32_t position, int flags);
/* prefillTokens (DecoderTSLRunner.ts:504-530): positions [start, end), no logits. */
int tlm_prefill(tlm_model* model, const int32_t* tokens, int32_t start, int32_t end);
/* Batched prefill control: tlm_prefill runs chunks of up to `chunk` positions
 * with at least `min_rows` positions (default 64, chunk 2048) as row batches
 * (MFMA GEMMs and flash attention per layer, tlm_op_linear_rows /
 * tlm_op_attention_rows) and replays the decode graph per position below
 * that, as the reference always does (DecoderTSLRunner.ts:472-480).
 * min_rows <= 0 turns the batched path off; TLM_ERR_INVALID names why a model
 * cannot use it (fp32 cache, head_dim other than 64/128, sizes not multiples
 * of 32, a q4 scale above 8188).  The row batches keep activations in fp16:
 * when one rounds to inf or is NaN, a device flag trips and tlm_prefill
 * replays that chunk on the fp32 decode graph (it waits for the stream after
 * each batched chunk to read the flag; tlm_model_describe counts such chunks). */
int tlm_model_set_prefill(tlm_model* model, int32_t min_rows, int32_t chunk);
/* readLogits (DecoderTSLRunner.ts:532-535): waits, copies n <= vocab floats. */
int tlm_read_logits(tlm_model* model, float* out, size_t n);
/* sampleToken greedy (TSLLogits.ts:359-361): waits, returns the argmax. */
int tlm_read_token(tlm_model* model, int32_t* token);
/* Greedy decode on the device: computes `token` at `position`, then feeds each
 * argmax back for n steps without host round trips; out[i] = argmax after
 * position+i.  Equals n rounds of computeToken + sampleToken. */
int tlm_decode_greedy(tlm_model* model, int32_t token, int32_t position, int n, int32_t* out);
/* resetCache (DecoderTSLRunner.ts:541-546): every cache row reads back zero
 * afterwards.  Only the rows some call could have written since the last
 * reset are cleared (positions below the highest one a compute, decode,
 * prefill, fill, write or timing call named), so a reset after a short
 * sequence costs little and leaves the weights in the last-level cache. */
int tlm_reset_cache(tlm_model* model);
/* Cache access in the canonical [count][kv_heads][head_dim] order, kv_fmt
 * element type (uint16 fp16 bits or float). */
int tlm_kv_write(tlm_model* model, int layer, int pos0, int count, const void* k, const void* v);
int tlm_kv_read(tlm_model* model, int layer, int pos0, int count, void* k, void* v);
/* Fills positions [0, count) of every layer with N(0,1) values from a
 * counter-based generator on the device (long-context benchmarks). */
int tlm_kv_fill_normal(tlm_model* model, uint64_t seed, int count);
/* readCandidates (TSLLogits.ts:336-349) over the model's last logits
 * (a token computed with TLM_LOGITS): k <= 16 (token, score) pairs to host
 * memory, best first; waits for the stream.  sampleTopKCandidates
 * (runtime/math.ts:527-547) then draws from them on the host. */
int tlm_read_candidates(tlm_model* model, int k, double softcap, int32_t* tokens, float* scores);
/* Final hidden state (after the final norm) of the last token with logits. */
int tlm_read_hidden(tlm_model* model, float* out, size_t n);

/* Timing with HIP events on the model stream.  tlm_time_decode: greedy
 * decode of n tokens after `warmup` untimed ones, from `position`; ms total.
 * tlm_time_kernel: average ms of one launch of kernel `which` (0 = LM head,
 * 1 = attention of layer 0, 2 = fused gate|up/SwiGLU/down MLP of layer 0,
 * 4 = QKV of layer 0, 5 = O of layer 0, 6 = top-8 candidates over the logits)
 * over iters back-to-back launches;
 * afterwards the residual accumulators are cleared (the next token starts
 * from the cache and ctrl state as left). */
int tlm_time_decode(tlm_model* model, int32_t token, int32_t position, int warmup, int n, double* ms);
int tlm_time_kernel(tlm_model* model, int which, int iters, double* avg_ms);
/* tlm_time_head / tlm_time_layers: n greedy decode steps from (token,
 * position), each the layer part (the persistent kernel, or the layer graph in
 * the long-window case) then the LM head, each part bracketed by its own pair
 * of events on the model stream; average ms of the LM head launch, or of the
 * layer part, inside a real step (weights cold in the caches, as in decode).
 * Leaves the cache and ctrl state advanced like tlm_decode_greedy.  No
 * reference counterpart (measurement). */
int tlm_time_head(tlm_model* model, int32_t token, int32_t position, int n, double* avg_ms);
int tlm_time_layers(tlm_model* model, int32_t token, int32_t position, int n, double* avg_ms);
/* tlm_trace_decode: n greedy decode steps from (token, position) through the
 * persistent schedule, launched directly with its timeline on; `out` receives
 * the last step's timeline: for every (block, wave), layer l < L and stage
 * (0 qkv, 1 attention, 2 O, 3 gate|up, 4 down), 4 wall-clock stamps (100 MHz:
 * weights issued, input ready, computed, published; 0 where the wave had no
 * such work); layer slot L, stage 0 holds the kernel's start and end.
 * n_out must be blocks * 16 * (L + 1) * 5 * 4 (see tlm_model_describe for the
 * block count).  TLM_ERR_STATE when the model has no
 * persistent schedule or a position needs the long-window kernels.  Tracing
 * has no counterpart in the reference (the browser has no device clock). */
int tlm_trace_decode(tlm_model* model, int32_t token, int32_t position, int n, uint64_t* out, size_t n_out);
/* Launch layout chosen for the model (for reports): per-stage grid sizes. */
int tlm_model_describe(tlm_model* model, char* out, size_t len);
/* Work the model has handed to its stream since it was created: the
 * counterpart of the reference's submission count
 * (src/test/submission.browser.test.ts:46-57: one submission per decode token,
 * one per prefill chunk).  A captured per-token graph is one graph launch;
 * kernels enqueued directly (the token/position write before a token, the
 * kernels of a batched prefill chunk, the eager schedule with graphs off)
 * count one each. */
typedef struct tlm_model_counts {
  uint64_t graph_launches;
  uint64_t kernel_launches;
  uint64_t prefill_chunks;      /* batched row chunks run (replayed ones excluded) */
  uint64_t replayed_positions;  /* prompt positions run through the decode graph */
  uint64_t recomputed_positions; /* positions recomputed on the per-stage graph after a failed
                                    token of the persistent schedule (a wait ran out, or an
                                    fp16 input overflow of its q4 linears) */
  uint64_t persistent_tokens;    /* token steps run on the persistent schedule (the rest ran
                                    the per-stage graph: long windows, shapes without it) */
} tlm_model_counts;
int tlm_model_counts_read(tlm_model* model, tlm_model_counts* out);

/* ------------------------------------------------------- host-side helpers
 * Synthetic inputs: N(0, std) from SplitMix64 -> Box-Muller, one counter
 * stream per (seed, stream id); identical output for any thread count. */
int tlm_synth_normal(uint64_t seed, uint64_t stream, size_t n, float stddev, float* out);
int tlm_synth_tokens(uint64_t seed, uint64_t stream, size_t n, int32_t vocab, int32_t* out);
/* q4 quantizer of the canonical format (fp16 scale = max|w|/7, ties-to-even codes). */
int tlm_quantize_q4(const float* w, int n_out, int k_in, uint8_t* packed, uint16_t* scales);
int tlm_f32_to_f16(const float* in, size_t n, uint16_t* out);

#ifdef __cplusplus
}
#endif
#endif /* TLM_H */
