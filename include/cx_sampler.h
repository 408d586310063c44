/*
 * cx_sampler.h -- C-ABI of the MI355X (gfx950) token-sampling library.
 *
 * The reference exposes these operations as Python methods only; each entry
 * point below names the reference code it replaces.  Plain pointers and
 * sizes, no framework types.  Device entry points take device pointers and
 * a hipStream_t (passed as void*), never synchronise and never allocate;
 * the "_host" variants take host memory, run on an internal stream and
 * return when the results are on the host.
 *
 * A workspace belongs to one stream.  A call queues several kernels that pass
 * results through it, so threads that share a stream and a workspace call one
 * at a time; on streams and workspaces of their own they need no order.
 *
 * Return value: 0 on success; CX_EINVAL (-1) for bad arguments, CX_EHIP (-2)
 * for a HIP runtime error, CX_ENOSPACE (-3) when the workspace is too small.
 * cx_last_error() gives a thread-local message for the last failure.
 *
 * Per-row outcomes are reported in row_status (CX_ROW_*), mirroring the
 * reference's control flow: which rows consumed their uniform, which fell
 * back to argmax, and which would have raised ValueError in numpy.
 */
#ifndef CX_SAMPLER_H
#define CX_SAMPLER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CX_OK        0
#define CX_EINVAL   (-1)
#define CX_EHIP     (-2)
#define CX_ENOSPACE (-3)

/* row_status low byte: outcome */
#define CX_ROW_OK          0  /* stochastic draw; consumed its uniform          (sampler.py:127) */
#define CX_ROW_GREEDY      1  /* T == 0: argmax of penalised logits              (sampler.py:114-115) */
#define CX_ROW_ARGMAX      2  /* filtered mass <= 0: argmax of penalised logits  (sampler.py:123-125) */
#define CX_ROW_ERROR       3  /* reference raises ValueError (NaN probabilities in choice) */
#define CX_ROW_UNSUPPORTED 4  /* input outside the library's limits (history window) */
/* row_status high bits: how the row was computed (informational) */
#define CX_ROW_FLAG_SLOW   0x100  /* resolved by the exact multi-pass row path */
#define CX_ROW_FLAG_DEEP   0x400  /* with CX_ROW_FLAG_SLOW: by its three-pass deep-nucleus variant */
#define CX_ROW_FLAG_EXACT  0x200  /* normaliser recomputed in fp64 for a near-threshold decision */

/* Per-row sampling parameters, 64 bytes.  Mirrors SamplingParams
 * (sampler.py:23-35) plus presence/frequency penalties, which the reference
 * lacks (0 = off; with both 0 the result is the reference's).  The doubles
 * are Python floats: they must not be rounded to fp32. */
typedef struct cx_row_params {
  double temperature;        /* 0 => greedy                                   */
  double top_p;              /* 1 => off                                      */
  double min_p;              /* 0 => off                                      */
  double typical_p;          /* 1 => off                                      */
  double repetition_penalty; /* 1 => off                                      */
  double presence_penalty;   /* 0 => off; subtracted once per id seen         */
  double frequency_penalty;  /* 0 => off; subtracted once per occurrence      */
  int32_t top_k;             /* 0 => off                                      */
  int32_t n_keep;            /* >0: penalty window = last max(64, n_keep) ids */
} cx_row_params;

/*
 * Sampler.sample for a batch of rows (sampler.py:108-127, with
 * apply_penalties :63-73 and _truncate :75-106).  Replaces a per-row loop of
 * `Sampler.sample(logits[b], params[b], generated_ids[b])` (engine.py:165,
 * speculative.py:126,171, scheduler.py:61).
 *
 *  logits    [B, ld] fp32 (cx_sample_f32) or bf16 bit patterns (cx_sample_bf16);
 *            row b holds V logits.  Never written.
 *  hist      [B, ldh] int32 token ids (generated_ids); hist_len[b] of them are
 *            used; ids outside [0, V) are ignored (sampler.py:68).  May be
 *            NULL when ldh == 0.
 *  prm       [B] cx_row_params
 *  u         [B] fp64 uniforms in [0, 1): the variate numpy's
 *            Generator.choice would draw (rows that do not draw ignore it).
 *  out_id    [B] int32 sampled ids
 *  row_status[B] int32 CX_ROW_* outcome | flags
 *  out_probs [B, V] fp32 post-filter normalised probabilities, or NULL.
 *            Costs one extra write of the batch; for verification.
 *  workspace device scratch of cx_sample_workspace_bytes(B, V, ldh) bytes;
 *            needs no initial contents (every call writes what it reads
 *            there before reading it).  One workspace per stream.
 */
int cx_sample_f32(const float* logits, int64_t ld, int32_t B, int32_t V,
                  const int32_t* hist, const int32_t* hist_len, int64_t ldh,
                  const cx_row_params* prm, const double* u,
                  int32_t* out_id, int32_t* row_status, float* out_probs,
                  void* workspace, size_t ws_bytes, void* stream);

int cx_sample_bf16(const uint16_t* logits, int64_t ld, int32_t B, int32_t V,
                   const int32_t* hist, const int32_t* hist_len, int64_t ldh,
                   const cx_row_params* prm, const double* u,
                   int32_t* out_id, int32_t* row_status, float* out_probs,
                   void* workspace, size_t ws_bytes, void* stream);

/* fp64 logits (the reference's Sampler.sample takes any float row; its model
 * produces fp32).  Same contract as cx_sample_f32; every row runs the exact
 * multi-pass fp64 path (slower than the fused fp32 / bf16 kernel). */
int cx_sample_f64(const double* logits, int64_t ld, int32_t B, int32_t V,
                  const int32_t* hist, const int32_t* hist_len, int64_t ldh,
                  const cx_row_params* prm, const double* u,
                  int32_t* out_id, int32_t* row_status, float* out_probs,
                  void* workspace, size_t ws_bytes, void* stream);

size_t cx_sample_workspace_bytes(int32_t B, int32_t V, int64_t ldh);

/*
 * cx_sample_f32 without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  No counterpart in the reference, which
 * has no device code.  It allocates nothing: its workspace is a static
 * device array of 64 MiB (CX_NOALLOC_SCRATCH_BYTES) that each GPU the
 * library runs on holds until the process ends.  Inputs, outputs, results
 * and errors are cx_sample_f32's; a batch whose workspace
 * (cx_sample_workspace_bytes) exceeds the scratch returns CX_EINVAL before
 * any device work.  Every call on one GPU shares that GPU's scratch: calls
 * that overlap on one GPU (on different streams or threads) race and must
 * be serialised by the caller.  No state carries from one call to the next.
 */
#define CX_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)
int cx_sample_f32_noalloc(const float* logits, int64_t ld, int32_t B, int32_t V,
                          const int32_t* hist, const int32_t* hist_len, int64_t ldh,
                          const cx_row_params* prm, const double* u,
                          int32_t* out_id, int32_t* row_status, float* out_probs,
                          void* stream);


/* Host-memory variants: same arguments on host memory; allocate, copy,
 * launch, copy back and synchronise.  dtype: 0 = fp32, 1 = bf16, 2 = fp64. */
int cx_sample_host(const void* logits, int32_t dtype, int64_t ld, int32_t B, int32_t V,
                   const int32_t* hist, const int32_t* hist_len, int64_t ldh,
                   const cx_row_params* prm, const double* u,
                   int32_t* out_id, int32_t* row_status, float* out_probs);

/*
 * Sampler.apply_penalties (sampler.py:63-73) for a batch of rows: out[b] is
 * float64(logits[b]) with the repetition penalty (x / rp if x > 0 else
 * x * rp, once per distinct in-range id of the window) and then the
 * presence / frequency penalties applied.  The window and id filtering are
 * those of cx_sample_f32.  Never writes the logits.
 *
 *  logits     [B, ld] of dtype 0 = fp32, 1 = bf16 bit patterns, 2 = fp64
 *  out        [B, ldo] fp64
 *  row_status [B] CX_ROW_OK, or CX_ROW_UNSUPPORTED when the row's window is
 *             longer than 4095 ids (out[b] is then not written)
 * No workspace; stream-ordered, never synchronises.
 */
int cx_apply_penalties(const void* logits, int32_t dtype, int64_t ld, int32_t B, int32_t V,
                       const int32_t* hist, const int32_t* hist_len, int64_t ldh,
                       const cx_row_params* prm, double* out, int64_t ldo,
                       int32_t* row_status, void* stream);

int cx_apply_penalties_host(const void* logits, int32_t dtype, int64_t ld, int32_t B, int32_t V,
                            const int32_t* hist, const int32_t* hist_len, int64_t ldh,
                            const cx_row_params* prm, double* out, int32_t* row_status);

/*
 * Sampler._truncate (sampler.py:75-106) for a batch of rows of fp64
 * probabilities: top-k (ties kept), top-p, min-p and typical-p on the
 * values as given (not renormalised, as the reference does), in that order.
 * out[b, i] = probs[b, i] where kept, else 0.  Equal values are ordered by
 * ascending id in the top-p and typical orders (numpy's argsort leaves that
 * order unspecified).  Uses temperature-independent fields of prm only.
 *
 *  row_status [B] CX_ROW_OK, or CX_ROW_ERROR for a row holding NaN or a
 *             negative value (out[b] is then not written)
 * No workspace; stream-ordered, never synchronises.
 */
int cx_truncate_f64(const double* probs, int64_t ld, int32_t B, int32_t V,
                    const cx_row_params* prm, double* out, int64_t ldo,
                    int32_t* row_status, void* stream);

int cx_truncate_host(const double* probs, int64_t ld, int32_t B, int32_t V,
                     const cx_row_params* prm, double* out, int32_t* row_status);

/*
 * Speculative-decoding verify step (speculative.py:145-171, with _softmax
 * :67-69) for B sequences at once.  Replaces the inline loop of
 * SpeculativeDecoder.generate.  All gamma positions are evaluated in parallel;
 * the result is what the reference's serial loop returns.
 *
 *  target     [B, gamma+1, V] fp32 target logits (row gamma = bonus row)
 *  draft      [B, gamma, V] fp32 draft logits (q rows); may be NULL if every
 *             temperature is 0
 *  draft_ids  [B, gamma] int32 proposed tokens
 *  u          [B, gamma+1] fp64: the verify generator's next gamma+1 variates
 *  temperature[B] fp32 (0 = greedy); the reference divides the fp32 row by
 *             fp32(T)
 *  accepted   [B] int32 accepted draft tokens
 *  next_tok   [B] int32 correction token, argmax of the bonus row (greedy),
 *             or -1 when every draft token was accepted in stochastic mode
 *             (the caller samples row gamma with the full sampler, :171)
 *  used       [B] int32 number of uniforms the reference would have consumed
 *  row_status [B] int32 CX_ROW_* flags
 *  workspace  device scratch of cx_spec_verify_workspace_bytes(B, gamma, V)
 *             bytes; any contents (every call writes what it reads).  One
 *             workspace per stream.
 */
int cx_spec_verify_f32(const float* target, const float* draft, const int32_t* draft_ids,
                       const double* u, const float* temperature,
                       int32_t B, int32_t gamma, int32_t V,
                       int32_t* accepted, int32_t* next_tok, int32_t* used,
                       int32_t* row_status, void* workspace, size_t ws_bytes, void* stream);

size_t cx_spec_verify_workspace_bytes(int32_t B, int32_t gamma, int32_t V);

int cx_spec_verify_host(const float* target, const float* draft, const int32_t* draft_ids,
                        const double* u, const float* temperature,
                        int32_t B, int32_t gamma, int32_t V,
                        int32_t* accepted, int32_t* next_tok, int32_t* used,
                        int32_t* row_status);

/*
 * LM-head projection with the greedy draw fused (transformer.py:102-104,
 * logits = h @ out_w.T, then sampler.py:114-115, argmax of the row, for a
 * greedy request with no penalty): the [B, V] logits never reach HBM.
 * bf16 operands, fp32 accumulation on MFMA.
 *
 *  hidden     [B, ldh] bf16 bits: the final-normed hidden states
 *  weight     [V, ldw] bf16 bits: the head weights (out_w, or the tied
 *             token embedding)
 *  D          hidden size, a multiple of 128; rows 16-byte aligned
 *  out_id     [B] int32: the first index of the row maximum, or of the
 *             first NaN (numpy's argmax)
 *  out_max    nullable [B] fp32: that logit
 *  out_logits nullable [B, V] fp32: every logit (verification only; this
 *             write is what the fusion saves)
 *  workspace  device scratch of cx_lmhead_workspace_bytes(B, V) bytes; any
 *             contents.  The size grows with B and with V: one workspace of
 *             the largest batch and vocabulary serves every smaller call.
 * Each logit is an fp32 sum over D.  Its order is the same for every batch of
 * up to 64 rows and for every larger one, but not for both where ldw is a
 * multiple of 2048 and D of 1024 (four quarter sums, or one sum, in k order):
 * there a near tie can go to another id from B = 64 to B = 65, or with the
 * weight rows padded.
 * Device pointers, stream-ordered, no synchronisation, no allocation.
 */
int cx_lmhead_argmax_bf16(const uint16_t* hidden, int64_t ldh, const uint16_t* weight,
                          int64_t ldw, int32_t B, int32_t D, int32_t V, int32_t* out_id,
                          float* out_max, float* out_logits, void* workspace, size_t ws_bytes,
                          void* stream);

size_t cx_lmhead_workspace_bytes(int32_t B, int32_t V);

/*
 * The paged KV cache between two sampling calls: the new tokens' keys and
 * values written to pages, their attention over the pages, pages copied.  The
 * reference keeps such a cache, attends over it and rotates positions in numpy
 * on the host (engine/radix_kv.py, core/attention.py:43-148,
 * core/tensor.py:36-180).
 *
 * A page of one layer holds page_tokens tokens of every kv head.  A head's
 * part is contiguous, all of it in 16-byte chunks of E elements (E = 8 for
 * bf16, 16 for e4m3), D = head_dim, P = page_tokens:
 *   K   chunk (d / E) * P + t holds dims d .. d + E - 1 of token t
 *   V   chunk (t / E) * D + d holds tokens t .. t + E - 1 of dim d
 *   e4m3 only: P fp32 scales of the tokens' keys, then P of their values
 * (2 P D elements, and 8 P bytes of scales).  An e4m3 code stands for its value
 * times its token's scale.
 *
 * One forward pass over a batch of sequences: sequence b's new tokens are rows
 * q_start[b] .. q_start[b + 1] - 1 of q, k, v and the outputs (q_start from 0 to
 * T; NULL: one new token each, T = B), and the last ones of its kv_len[b]
 * tokens; token t lies in page table[b][t / P].  A token whose position is
 * negative or past the table's pages, or whose page id is outside [0, n_pages),
 * is neither written nor attended.
 */
#define CX_KV_BF16 1
#define CX_KV_E4M3 3                     /* OCP e4m3: largest value 448 */
#define CX_KV_MAX_BATCH 4096
#define CX_TREE_MAX_WORDS 16             /* nodes of a tree that masks reach: 1024 */
typedef struct cx_kv_batch {
  void* pages;               /* one layer's pages, 16-byte aligned             */
  int64_t page_stride;       /* bytes from one page to the next                */
  const int32_t* table;      /* [B, ld_table] page ids                         */
  int64_t ld_table;
  const int32_t* kv_len;     /* [B] tokens, the new ones included              */
  const int32_t* q_start;    /* [B + 1], or NULL                               */
  int32_t n_pages, kv_heads;
  int32_t head_dim;          /* 64, 128 or 256                                 */
  int32_t page_tokens;       /* 16, 32, 64, 128 or 256                         */
  int32_t dtype;             /* CX_KV_BF16 or CX_KV_E4M3                       */
  int32_t B, max_pages, T;   /* max_pages: ids of a table row                  */
} cx_kv_batch;

/*
 * The new tokens of a forward pass made ready for attention: q and k normed
 * per head (optional), rotated to their positions (optional), q written to
 * q_out, k and v to the pages.  One pass over q, k and v.  fp32 arithmetic (the
 * norm's squares too: a row's largest value between 2^-60 and 2^60, or an eps
 * that covers smaller ones), each result rounded once.
 *
 *  q, k, v    bf16 bits, row (token, head) at token * _token + head * _head
 *             elements, rows 16-byte aligned
 *  q_norm, k_norm  nullable [D] bf16 bits: x * rsqrt(mean(x^2) + eps) * weight
 *  rope       nullable [rope_rows, rotary_dim] fp32: the cosines of position p
 *             (rotary_dim / 2), then the sines; rope_rows at least max_pages *
 *             page_tokens.  The first rotary_dim dims of a head are rotated (a
 *             multiple of 16), pairs (j, j + rotary_dim / 2), or (2 j, 2 j + 1)
 *             if interleaved
 *  q_out      [T, q_heads, D] bf16 bits; of a token whose position is outside the
 *             table's pages, rotated as at position 0
 * e4m3: a (token, head)'s scale is the fp32 quotient max|x| / 448, 1 where that
 * is 0, and a code the nearest of the fp32 quotient x / scale; a row holding inf
 * or NaN gets a NaN scale and zero codes.
 * Device pointers, stream-ordered, no synchronisation, no allocation.
 */
int cx_kv_append_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token, int64_t q_head,
                      const uint16_t* k, int64_t k_token, int64_t k_head, const uint16_t* v,
                      int64_t v_token, int64_t v_head, int32_t q_heads, const float* rope,
                      int32_t rope_rows, int32_t rotary_dim, int32_t interleaved,
                      const uint16_t* q_norm, const uint16_t* k_norm, double eps,
                      uint16_t* q_out, void* stream);

/*
 * The same for a tree of drafted tokens: the new token of row t is written to its
 * place as above, but rotated as at position kv_len[b] - n + depth[t], n the new
 * tokens of its sequence (siblings stand at one position); clamped to the rows of
 * the table's pages.
 *
 *  depth      [T] int32, or NULL: as above
 */
int cx_kv_append_tree_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token,
                           int64_t q_head, const uint16_t* k, int64_t k_token, int64_t k_head,
                           const uint16_t* v, int64_t v_token, int64_t v_head, int32_t q_heads,
                           const float* rope, int32_t rope_rows, int32_t rotary_dim,
                           int32_t interleaved, const uint16_t* q_norm, const uint16_t* k_norm,
                           double eps, const int32_t* depth, uint16_t* q_out, void* stream);

/*
 * Attention of the new tokens over the pages: a decode step's single tokens, a
 * verify round's gamma + 1, several together.  q head h reads kv head
 * h / (q_heads / kv_heads).  The token at position p attends to the
 * positions t <= p, t > p - window (window 0: all), with scores scale * q.k,
 * capped to softcap * tanh(score / softcap) if softcap > 0 (infinity: not
 * capped; the cap adds an error of about 2^-22 of a softcap up to 256, 2^-19 of
 * the score above).  A token that attends to nothing gets zeros.  fp32
 * scores, softmax and sums, the weights with 16 bits in their products; out is
 * rounded once.  Short tables take one launch, others two; results do not
 * depend on timing.
 * T is at most 2^28; calls whose row blocks times table units (16 rows, 32
 * tokens) reach 2^38 are refused.
 *
 *  q          bf16 bits, row (token, head) at token * q_token + head * q_head
 *             elements, rows 16-byte aligned
 *  max_new    the most new tokens of a sequence: picks the kernel's tile, and
 *             any value >= 1 gives right results
 *  out        [T, q_heads, D] bf16 bits
 *  workspace  device scratch of cx_paged_attention_workspace_bytes(...) bytes;
 *             16-byte aligned, any contents.  One workspace per stream.  The
 *             size grows with max_new and with the q heads of a kv head: one
 *             of the largest call serves every smaller one, of either cache
 *             type.
 * Device pointers, stream-ordered, no synchronisation, no allocation.
 */
int cx_paged_attention_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token,
                            int64_t q_head, int32_t q_heads, int32_t max_new, double scale,
                            int32_t window, double softcap, uint16_t* out, void* workspace,
                            size_t ws_bytes, void* stream);

size_t cx_paged_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                          int32_t max_new);

/*
 * Attention of a tree of drafted tokens: as cx_paged_attention_bf16, but which of
 * the new tokens a new token attends to is given.  The n new tokens of sequence b
 * are its nodes 0 .. n - 1, in the slots kv_len[b] - n ..  A node attends to every
 * slot before them and to the nodes whose bits its mask has, in any order (its own
 * bit too, if it attends to itself).  A window w leaves of the slots before them
 * those whose position is above kv_len[b] - n + depth - w; nodes go by the mask
 * alone (cx_tree_masks_window leaves out those that the window has passed).
 *
 *  mask       [T, mask_words], at most CX_TREE_MAX_WORDS: bit i % 64 of word i / 64 of a token's row is node i;
 *             nodes past the words are not attended to
 *  depth      [T] int32 >= 0, a node's distance from the first new position; NULL
 *             where window is 0
 *  max_new, workspace and the rest: as there, of this call's own workspace size
 *             (cx_tree_attention_workspace_bytes)
 * Device pointers, stream-ordered, no synchronisation, no allocation.
 */
int cx_tree_attention_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token,
                           int64_t q_head, int32_t q_heads, const uint64_t* mask,
                           int32_t mask_words, const int32_t* depth, int32_t max_new,
                           double scale, int32_t window, double softcap, uint16_t* out,
                           void* workspace, size_t ws_bytes, void* stream);

size_t cx_tree_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                         int32_t max_new);

/*
 * Masks and depths of trees from their parents: a node's mask has the bits of the
 * node and of its ancestors.  Sequence b's nodes are q_start[b] .. q_start[b + 1] - 1
 * of T (q_start NULL: one each, T = B).
 *
 *  parents    [T] int32: the parent's place among its sequence's nodes, below the
 *             node's own; anything else is a root
 *  mask       [T, words] (words >= 1; nodes past 64 words have no bit)
 *  depth      nullable [T] int32: the number of ancestors
 * Rows outside every sequence are not written.  Device pointers, stream-ordered, no
 * synchronisation, no allocation.
 */
int cx_tree_masks(const int32_t* parents, const int32_t* q_start, int32_t B, int32_t T,
                  uint64_t* mask, int32_t words, int32_t* depth, void* stream);

/*
 * The same for attention with a window: a mask has the bits of the node and of its
 * window - 1 nearest ancestors, those whose positions are above its own less window
 * (0: of all).  Depths count all ancestors.
 */
int cx_tree_masks_window(const int32_t* parents, const int32_t* q_start, int32_t B, int32_t T,
                         uint64_t* mask, int32_t words, int32_t* depth, int32_t window,
                         void* stream);

/*
 * The path of a tree that the sampled ids follow.  Node 0 is the last confirmed
 * token and always accepted; after node c comes its first child (the lowest index)
 * whose token is sampled[c], if it has one and the path is shorter than width.
 * sampled[c], a draw from the model's distribution after node c, may come from any
 * sampler: the tokens are then distributed as without drafts.
 *
 *  parents    [T] int32, as for cx_tree_masks (children have higher indices)
 *  tokens, sampled  [T] int32
 *  path       [B, width] int32: the accepted nodes, then -1
 *  count      [B] int32 accepted nodes, 0 for a sequence without nodes
 *  next       [B] int32: sampled of the last accepted node, -1 if there is none
 * Device pointers, stream-ordered, no synchronisation, no allocation.
 */
int cx_tree_accept(const int32_t* parents, const int32_t* tokens, const int32_t* sampled,
                   const int32_t* q_start, int32_t B, int32_t T, int32_t width, int32_t* path,
                   int32_t* count, int32_t* next, void* stream);

/*
 * Accepted tokens moved to their places in every layer: of sequence b, whose n new
 * tokens begin in slot s = kv_len[b] - n, slot s + j becomes a copy of slot
 * s + path[b][j] for j < count[b], as if every slot were read before any is written.
 * A row of path ends before an entry that is not above the one before it, or not
 * below n; where that is before j reaches count[b], the entry becomes -1.  A move from
 * or to a slot without a page in the pool is left out.  No page that is written to may
 * be another sequence's too.
 *
 *  kv         pages: layer 0's; layer l's are layer_stride bytes further each, not 0
 *  path       [B, width] int32
 *  count      [B] int32 (at most width are taken), or NULL: width each
 * Device pointers, stream-ordered, no synchronisation, no allocation.
 */
int cx_kv_commit(const cx_kv_batch* kv, int64_t layer_stride, int32_t n_layers,
                 int32_t* path, int32_t width, const int32_t* count, void* stream);

/*
 * Pages copied in every layer: page dst[i] becomes a copy of page src[i] (a
 * fork's last page before either sequence appends to it, a compaction's
 * moves).  A pair with an id outside [0, n_pages) is skipped.  No page may be
 * the destination of two pairs, or of one pair and the source of another.
 *
 *  pages      layer l's page i at l * layer_stride + i * page_stride bytes;
 *             page_bytes of it are copied (all multiples of 16)
 *  src, dst   [n] int32
 * Device pointers, stream-ordered, no synchronisation, no allocation.
 */
int cx_kv_copy_pages(void* pages, int64_t layer_stride, int64_t page_stride, int64_t page_bytes,
                     int32_t n_layers, int32_t n_pages, const int32_t* src, const int32_t* dst,
                     int32_t n, void* stream);

/*
 * Products of few rows with 4-bit weights: out = x W^T, W [N, K] with
 * W[n, k] = scale * code + shift of row n and group k / group, or, without shifts,
 * scale * (code - 8).  fp32 sums (of code / 16 + 1, less what that adds: the error
 * is about 5 times that of the same sum of W), out rounded once.  A row of x that
 * holds an infinity or NaN, or values above 2^100, gives NaN.
 *
 *  x          [M, ldx] bf16 bits, rows 16-byte aligned
 *  tiles      codes, 16-byte aligned: [N / 16, K / 128, 64, 4] words of 8 codes, both
 *             rounded up.  Word s of lane 16 j + r holds row r's codes of k = 128 t +
 *             32 s + 8 j + e, e = 0 .. 7, at bit 4 (e / 2) + 16 (e % 2)
 *  scales     fp16 bits, 16-byte aligned: [N / 16 rounded up, K / group, 16], or with
 *             shifts [.., 16, 2]: scale, shift
 *  group      32, 64 or 128; K a multiple of it; N, K < 2^28, M < 2^21
 *  out        [M, ldo] fp32, or bf16 bits if out_bf16
 * Rows of the last tile past N are read and not used.  The weights are read once for
 * up to 32 rows of x; 33 to 64 rows read them once where N is above 2048, else twice,
 * and more rows as often as they are 64 or, where N is small, 32.  Device pointers,
 * stream-ordered, no synchronisation, no allocation.
 */
int cx_w4_linear_bf16(const uint16_t* x, int64_t ldx, const uint32_t* tiles,
                      const uint16_t* scales, int32_t shifts, int32_t group, int32_t M, int32_t N,
                      int32_t K, void* out, int64_t ldo, int32_t out_bf16, void* stream);

/* Kernel timing (measurement only).  While enabled, every library kernel is
 * dispatched with a start / stop event pair recorded by the dispatch itself
 * (hipExtLaunchKernel): the kernel's execution interval on its stream.
 * cx_timing_read waits for the recorded events, returns the summed
 * milliseconds and launch count of one kernel kind and forgets its records.
 * No counterpart in the reference (which has no device code); callers are
 * benchmarks and profilers. */
#define CX_KERNEL_SAMPLE        0  /* fused sampler kernel            */
#define CX_KERNEL_SAMPLE_SLOW   1  /* region finisher / exact row kernel */
#define CX_KERNEL_VERIFY_STATS  2  /* verify: stats over all rows     */
#define CX_KERNEL_VERIFY_REST   3  /* verify: decide + residual draw  */
#define CX_KERNEL_SAMPLE_FINISH 4  /* reserved: no longer launched (the region
                                      finisher runs in CX_KERNEL_SAMPLE_SLOW) */
#define CX_KERNEL_PENALTIES     5  /* apply_penalties                 */
#define CX_KERNEL_TRUNCATE      6  /* _truncate                       */
#define CX_KERNEL_LMHEAD        7  /* LM head: projection tiles + argmax keys */
#define CX_KERNEL_LMHEAD_MERGE  8  /* LM head: per-row merge of the keys */
#define CX_KERNEL_KV_APPEND     9  /* q, k, v normed, rotated, k and v to the pages */
#define CX_KERNEL_ATTEND        10 /* paged attention                  */
#define CX_KERNEL_ATTEND_JOIN   11 /* paged attention: split rows joined */
#define CX_KERNEL_KV_COPY       12 /* page copies                      */
#define CX_KERNEL_TREE          13 /* tree attention                   */
#define CX_KERNEL_TREE_JOIN     14 /* tree attention: split rows joined */
#define CX_KERNEL_TREE_WALK     15 /* tree masks, accepted paths       */
#define CX_KERNEL_KV_COMMIT     16 /* accepted tokens moved            */
#define CX_KERNEL_W4            17 /* products with 4-bit weights      */
#define CX_KERNEL_KINDS         18
int cx_timing_enable(int on);
int cx_timing_read(int32_t kernel, double* total_ms, int64_t* launches);

/* Thread-local description of the last failure ("" if none). */
const char* cx_last_error(void);

/* Library version string. */
const char* cx_version(void);

#ifdef __cplusplus
}
#endif
#endif /* CX_SAMPLER_H */
