/*
 * pm_sample.h -- C ABI of the B200 token-selection path (libpm_sample.so).
 *
 * Replaces the per-step token selection of PagedMoE's decode loop: the
 * logits processors, the log-softmax, the sampler and the draft acceptance
 * of a verify pass.  All pointers are device pointers unless stated; every
 * function takes a cudaStream_t (as void*) and returns a status code, never
 * aborts and allocates nothing.  The only process-wide state is per device:
 * each kernel's shared-memory attribute and occupancy, set up on the first
 * launch on that device, and the scratch array of pm_sample_rows_static.
 * Calls with separate workspaces may come from several host threads on
 * different streams.
 *
 * Reference interfaces replaced (paths within noahclark556/paged-moe):
 *   pm_sample_rows      sampler(logprobs) -> tokens, built by mlx-lm's
 *                       make_sampler (call sites pagedmoe/verify_decode.py:839,
 *                       :903, pagedmoe/lookup_decode.py:359, run.py:53) plus
 *                       the processor loop before it (verify_decode.py:828-835,
 *                       :889-899) fused into one pass over the logits.
 *   pm_apply_processors proc(tokens, logits) -> logits, built by mlx-lm's
 *                       make_logits_processors (verify_decode.py:830-831,
 *                       :895-896; lookup_decode.py:344-356), and the
 *                       where(mask, x, -inf) processors of
 *                       pagedmoe/think_budget.py:107-109 and rescue.py:240-245.
 *   pm_logprobs         logits - logsumexp(logits) (verify_decode.py:835, :899;
 *                       lookup_decode.py:358).
 *   pm_verify           the accept loop of a verify pass
 *                       (lookup_decode.py:363-369, verify_decode.py:903-921),
 *                       plus residual rejection sampling (no reference code).
 *   pm_shard_summarize / pm_shard_merge
 *                       vocab-sharded sampling (no reference code: the
 *                       reference runs on one device).
 */
#ifndef PM_SAMPLE_H
#define PM_SAMPLE_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define PM_API __attribute__((visibility("default")))
#else
#define PM_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define PM_OK 0
#define PM_ERR_ARG (-1)          /* bad argument (null pointer, bad size, ...) */
#define PM_ERR_CUDA (-2)         /* a CUDA call failed; see pm_last_cuda_error */
#define PM_ERR_UNSUPPORTED (-3)  /* valid but outside this build's limits */
#define PM_ERR_WORKSPACE (-4)    /* workspace smaller than pm_*_workspace_bytes */

/* logits element types */
#define PM_DTYPE_F32 0
#define PM_DTYPE_BF16 1

/* noise sources */
#define PM_NOISE_PHILOX 0   /* Philox4x32-10 keyed by (seed, offset, row) */
#define PM_NOISE_INJECTED 1 /* caller-provided Gumbel values and uniforms */

/* pm_row_params.flags */
#define PM_F_GREEDY 0x1u    /* temperature == 0: argmax */
#define PM_F_TOP_P 0x2u     /* 0 < top_p < 1 */
#define PM_F_MIN_P 0x4u     /* min_p != 0 */
#define PM_F_REP 0x10u      /* repetition penalty on */
#define PM_F_PRES 0x20u     /* presence penalty on */
#define PM_F_FREQ 0x40u     /* frequency penalty on */
#define PM_F_UNBOUNDED 0x100u /* top_p or min_p on while top_k is off */
#define PM_F_FULL 0x200u    /* temperature > 0 and no filter: whole-vocabulary draw */

/* Per-row sampling and processor settings.  Scalars are the fp32 values the
 * reference's arithmetic sees: inv_temperature = fl32(1/temp),
 * top_p_comp = fl32(1 - top_p), log_min_p = fl32(log(min_p)), evaluated in
 * double first as Python does (mlx-lm make_sampler / make_logits_processors
 * keyword arguments; defaults resolved by pagedmoe/sampling.py:121-135). */
typedef struct pm_row_params {
    uint32_t flags;
    float inv_temperature;
    int32_t top_k;               /* <= 0: off */
    float top_p_comp;
    float log_min_p;
    int32_t min_tokens_to_keep;
    float repetition_penalty;
    int32_t repetition_context_size;
    float presence_penalty;
    int32_t presence_context_size;
    float frequency_penalty;
    int32_t frequency_context_size;
} pm_row_params;

/* Rows of logits plus the processors that act on them. */
typedef struct pm_rows {
    const void *logits;          /* [rows, row_stride] of dtype */
    int32_t dtype;               /* PM_DTYPE_* */
    int64_t rows;
    int64_t vocab;
    int64_t row_stride;          /* elements between rows (>= vocab) */
    const pm_row_params *params; /* [rows], or [1] when params_per_row == 0 */
    int32_t params_per_row;
    /* history the penalties read.  Without feed, row r uses
     * hist[r, 0:hist_len[r]].  With feed (a verify pass), row r belongs to
     * request b = r / feed_group at position i = r % feed_group and uses
     * hist[b, 0:hist_len[b]] followed by feed[b, 0:i+1], i.e. its history plus
     * [y] + drafts[:i] (reference verify_decode.py:889-898). */
    const int32_t *hist;         /* [hist_rows, hist_stride] or NULL */
    const int32_t *hist_len;     /* [hist_rows] or NULL (all hist_stride) */
    int64_t hist_stride;
    const int32_t *feed;         /* [rows / feed_group, feed_group] or NULL */
    int32_t feed_group;          /* rows per request when feed != NULL */
    /* logit bias shared by all rows (mlx-lm logit_bias) */
    const int32_t *bias_tokens;  /* [n_bias] distinct ids, ascending (an id out of order is not applied) */
    const float *bias_values;    /* [n_bias] */
    int32_t n_bias;
    /* allowed-token bitmask: bit v of word v/32 of row r; NULL = all allowed */
    const uint32_t *mask;        /* [rows, mask_stride] */
    int64_t mask_stride;         /* words, >= ceil(vocab / 32) */
    /* host-side bounds of the device params (they size the launch): the OR of
     * every row's flags, and the largest top_k of any row (0 if none). */
    uint32_t flags_any;
    int32_t top_k_max;
    /* forced token per row, -1 for none, or NULL: the row's logits become
     * where(arange == forced, logits, -inf) after the other processors (the
     * ThinkBudget processor, reference think_budget.py:107-109) */
    const int32_t *forced;
} pm_rows;

/* Noise of the draw. */
typedef struct pm_noise {
    int32_t mode;                /* PM_NOISE_* */
    uint64_t seed;
    uint64_t offset;             /* advances per step */
    uint32_t row_base;           /* Philox row id of row 0 */
    const float *gumbel;         /* injected: [rows, gumbel_stride] Gumbel values */
    int64_t gumbel_stride;
    const double *uniform;       /* injected: [rows, 2] uniforms in [0,1) */
} pm_noise;

/* Outputs of pm_sample_rows (only tokens is required). */
typedef struct pm_sample_out {
    int32_t *tokens;             /* [rows] */
    float *lse;                  /* [rows] row log-sum-exp of the processed logits, or NULL */
    float *token_logprob;        /* [rows] logprob of the chosen token, or NULL */
    int32_t *surv_ids;           /* [rows, surv_cap] survivors in rank order, or NULL */
    float *surv_probs;           /* [rows, surv_cap] their probabilities at temperature */
    int32_t *n_surv;             /* [rows] */
    int32_t surv_cap;
} pm_sample_out;

/* Workspace bytes pm_sample_rows needs for these rows.  Nothing in the
 * workspace needs to start at zero. */
PM_API size_t pm_sample_workspace_bytes(const pm_rows *rows);

/* One fused pass: processors, row log-sum-exp, top-k / top-p / min-p,
 * temperature and the draw, for every row.  Replaces mlx-lm's
 * make_sampler(...)(logprobs) after make_logits_processors(...) processors
 * (reference verify_decode.py:828-839). */
PM_API int pm_sample_rows(const pm_rows *rows, const pm_noise *noise, const pm_sample_out *out,
                   void *workspace, size_t workspace_bytes, void *stream);

/* Processed logits [rows, vocab] fp32 (logit bias, penalties, mask), the
 * callables of make_logits_processors (verify_decode.py:830-831). */
PM_API size_t pm_processors_workspace_bytes(const pm_rows *rows);
PM_API int pm_apply_processors(const pm_rows *rows, float *out, int64_t out_stride, void *workspace,
                        size_t workspace_bytes, void *stream);

/* Processed logits minus their row log-sum-exp (verify_decode.py:835). */
PM_API int pm_logprobs(const pm_rows *rows, float *out, int64_t out_stride, float *lse_out, void *workspace,
                size_t workspace_bytes, void *stream);

/* Draft acceptance of a verify pass.  rows->rows = requests * (k + 1): row
 * i of request b holds the target logits that judge drafts[b, i] (i < k) or
 * give the bonus token (i = k); rows->feed must be [y] + drafts per request
 * (feed_group = k + 1) so each row's processors see history + [y] + drafts[:i]
 * (reference verify_decode.py:889-898). */
#define PM_VERIFY_MATCH 0     /* reference rule: sample every row, keep drafts while equal
                                 (lookup_decode.py:363-369, verify_decode.py:915-921) */
#define PM_VERIFY_RESIDUAL 1  /* speculative rejection sampling: accept draft i when
                                 u_i * q_i(d) < p_i(d), else draw from max(p_i - q_i, 0) */

typedef struct pm_verify_args {
    int32_t mode;                /* PM_VERIFY_* */
    const int32_t *drafts;       /* [requests, n_draft] */
    int32_t n_draft;             /* k >= 0 */
    const void *draft_logits;    /* residual: [requests * k, draft_row_stride] logits of q */
    int32_t draft_dtype;         /* PM_DTYPE_* */
    int64_t draft_row_stride;
    const double *u_accept;      /* injected: [requests, k] uniforms, else Philox */
    const double *u_residual;    /* injected: [requests] uniforms, else Philox */
    int32_t *tokens;             /* out [requests, k + 1]: accepted drafts, then the
                                    request's own token; -1 after it */
    int32_t *n_accepted;         /* out [requests] */
    int32_t *row_tokens;         /* optional out [requests * (k + 1)]: each row's sample */
} pm_verify_args;

PM_API size_t pm_verify_workspace_bytes(const pm_rows *rows, const pm_verify_args *v);
PM_API int pm_verify(const pm_rows *rows, const pm_noise *noise, const pm_verify_args *v, void *workspace,
                     size_t workspace_bytes, void *stream);

/* Vocabulary-sharded sampling (no reference code: the reference runs on one
 * device).  A tensor-parallel LM head leaves shard i with the contiguous ids
 * [i * shard_width, min((i + 1) * shard_width, vocab_total)) of every row;
 * every shard but the last must be a whole number of 1024-token tiles.  Each
 * shard calls pm_shard_summarize on its slice (rows->vocab = its width, the
 * mask its slice of words, bias ids shifted to the slice; history ids stay
 * global), the caller all-gathers the summaries in shard order (one NCCL
 * all-gather of pm_shard_summary_bytes per shard), and pm_shard_merge gives
 * every rank the row's tokens -- the same tokens, log-sum-exp and survivor
 * lists pm_sample_rows gives on the unsharded rows.  Rows whose unbounded
 * top-p / min-p keeps more than 256 tokens are flagged (status 1, token -1):
 * the caller finishes them with pm_sample_rows on their whole rows (the
 * Python layer all-gathers the flagged rows' slices for that). */
typedef struct pm_shard {
    int32_t shard_index;
    int32_t n_shards;
    int64_t vocab_total;
    int64_t shard_width;         /* ids per shard (the last may hold fewer) */
} pm_shard;

PM_API size_t pm_shard_summary_bytes(const pm_rows *rows, const pm_shard *shard);
PM_API int pm_shard_summarize(const pm_rows *rows, const pm_shard *shard, const pm_noise *noise, void *summary,
                              void *workspace, size_t workspace_bytes, void *stream);
/* rows: the sampler settings (params, flags_any, top_k_max, rows) with
 * vocab = vocab_total; logits are not read.  summaries: [n_shards] summaries
 * back to back.  workspace: at least 4 * rows bytes (row status). */
PM_API int pm_shard_merge(const pm_rows *rows, const pm_shard *shard, const pm_noise *noise, const void *summaries,
                          const pm_sample_out *out, void *workspace, size_t workspace_bytes, void *stream);

/* Batched n-gram drafts: replaces lookup_decode.draft_ngram
 * (pagedmoe/lookup_decode.py:184-221), which scans one request's context per
 * call in Python.  For every request, up to k tokens that followed the
 * latest earlier occurrence of the longest suffix (n_max down to n_min
 * tokens; reference defaults 8 and 3, config.py:1288-1289) -- the latest
 * occurrence with k tokens after it, else the one with the most.  hist:
 * [requests, hist_stride] device ids with optional lengths; drafts:
 * [requests, k] (-1 after draft_len); match_n: the n that matched (0: none),
 * may be NULL.  n_max <= 32. */
PM_API int pm_draft_ngram(const int32_t *hist, const int32_t *hist_len, int64_t hist_stride, int64_t requests,
                          int32_t k, int32_t n_min, int32_t n_max, int32_t *drafts, int32_t *draft_len,
                          int32_t *match_n, void *stream);

/* Device ThinkBudget (reference pagedmoe/think_budget.py:75-109): for every
 * row, the token the close text forces next, or -1.  gen: [rows, gen_stride]
 * ids generated after the prompt (gen_len per row); piece_len / piece_end:
 * [table_size] decoded length and sentence-end flag per id; chars: per-row
 * budget; close: [n_close] ids ending with end_id; start_id < 0 when the
 * template opens reasoning in the prompt (open_in_prompt) -- else reasoning
 * counts only after the model's own start_id; slack: tokens to wait for a
 * sentence end (reference SLACK_TOKENS = 48).  forced: [rows] out, usable as
 * pm_rows.forced. */
PM_API int pm_think_budget(const int32_t *gen, const int32_t *gen_len, int64_t gen_stride, int64_t rows,
                           const int32_t *piece_len, const uint8_t *piece_end, int64_t table_size,
                           const int32_t *chars, const int32_t *close, int32_t n_close, int32_t end_id,
                           int32_t start_id, int32_t slack, int32_t *forced, void *stream);

/* The LM head: logits = hidden @ weight^T on the tensor cores (bf16 in, fp32
 * accumulate), the producer of the logits that the reference's decode step
 * computes before its processors and sampler (pagedmoe/verify_decode.py:821,
 * :824 for a plain step, :887 for a verify pass).  hidden: [n_tokens,
 * hidden_stride] bf16 (the final-norm output); weight: [vocab,
 * weight_stride] bf16 (row v: token v's output embedding).  Both 16-byte
 * aligned with strides a multiple of 8 elements. */
typedef struct pm_lmhead {
    const void *hidden;
    int64_t n_tokens;
    int64_t hidden_size;
    int64_t hidden_stride;       /* elements between rows */
    const void *weight;
    int64_t weight_stride;       /* elements between rows */
} pm_lmhead;

/* The logits themselves: [n_tokens, logits_stride] fp32 (stride a multiple
 * of 4, 16-byte aligned). */
PM_API int pm_lmhead_logits(const pm_lmhead *h, int64_t vocab, float *logits, int64_t logits_stride,
                            void *stream);

/* LM head fused with pm_sample_rows: the GEMM's epilogue writes the tile
 * statistics and candidates of each row, so the logits never reach device
 * memory; the results are those of pm_sample_rows on the logits that
 * pm_lmhead_logits computes (tokens, log-sum-exp, survivors, bit for bit).
 * rows: rows == h->n_tokens and rows->logits unused; greedy rows and rows
 * with 0 < top_k <= 256 (temperature, top_p and min_p on top), with the
 * processors (logit bias, repetition / presence / frequency penalties over
 * rows->hist) and the allowed-token mask.  Verify feeds, forced tokens,
 * unbounded top-p / min-p and whole-vocabulary draws return
 * PM_ERR_UNSUPPORTED (use pm_lmhead_logits + pm_sample_rows).  Row status
 * bit 128: a logit was NaN or +inf.  The workspace needs no zeroing. */
PM_API size_t pm_lmhead_sample_workspace_bytes(const pm_lmhead *h, const pm_rows *rows);
PM_API int pm_lmhead_sample(const pm_lmhead *h, const pm_rows *rows, const pm_noise *noise,
                            const pm_sample_out *out, void *workspace, size_t workspace_bytes, void *stream);

/* Top log-probabilities (no counterpart in the reference, whose sampler
 * returns the whole log-softmax row, pagedmoe/verify_decode.py:835): the k
 * largest logits of every row in descending order (ties: the lowest id) and
 * their log-probabilities under softmax(logits * inv_temperature) over the
 * allowed tokens -- what an API answers with beside a token, a beam's list of
 * continuations, a teacher's targets for pm_distill.  Tokens that are
 * disallowed or -inf are no candidates: places left over hold id -1 and
 * log-probability -inf.  A row with a NaN or +inf among its allowed logits
 * gives ids -1 and NaN.  1 <= k <= 256. */
typedef struct pm_top_rows {
    const void *logits;          /* [rows, row_stride] of dtype */
    int32_t dtype;               /* PM_DTYPE_* */
    int64_t rows;
    int64_t vocab;
    int64_t row_stride;          /* elements between rows (>= vocab) */
    const uint32_t *mask;        /* [rows, mask_stride] allowed-token bits, or NULL */
    int64_t mask_stride;         /* words, >= ceil(vocab / 32); 0: one mask for every row */
    int32_t k;
    double inv_temperature;      /* > 0; log2(e) times it fits fp32 (4.3e-39 <= T <= 2e45) */
} pm_top_rows;

/* ids, logprobs: [rows, k]; lse: [rows] log-sum-exp of logits *
 * inv_temperature, or NULL. */
PM_API int pm_top_logprobs(const pm_top_rows *t, int32_t *ids, float *logprobs, float *lse, void *stream);

/* One step of beam search (no counterpart in the reference, which decodes one
 * sequence a request): row w of item i holds the logits after beam w, with
 * score scores[i, w].  The n best continuations of every item over its beams
 * and the vocabulary, by
 *     total = score + (logit - log-sum-exp of the beam's allowed logits)
 * in 64 bits, divided by length ^ length_penalty (length: lengths[i, w] + 1),
 * best first; ties go to the lower beam, then the larger logit, then the
 * lower token.  A finished beam (done != 0) offers one candidate, token eos
 * at its own score and length, and its logits are not read.  A beam of score
 * -inf, and one whose allowed logits hold a NaN, a +inf or nothing finite,
 * offers none.  Places left over hold score -inf, parent -1, token -1,
 * length 0.  keep_slots (n == beams): the best child of every beam that lives
 * on takes that beam's place, the others fill the free places in ascending
 * order, so that moving states in place touches only the beams that ended.
 * 1 <= beams <= 64, 1 <= n <= 256, |length_penalty| <= 16. */
typedef struct pm_beam {
    const void *logits;          /* [items * beams, row_stride] of dtype */
    int32_t dtype;               /* PM_DTYPE_* */
    int64_t items;
    int32_t beams;
    int64_t vocab;
    int64_t row_stride;
    const uint32_t *mask;        /* [items * beams, mask_stride], or NULL */
    int64_t mask_stride;         /* words; 0: one mask for every row */
    const float *scores;         /* [items, beams] */
    const uint8_t *done;         /* [items, beams], or NULL */
    const int32_t *lengths;      /* [items, beams] tokens so far, or NULL (length_penalty must be 0) */
    int32_t eos;                 /* the token that ends a beam, -1: none (done must be NULL) */
    double length_penalty;
    int32_t n;
    int32_t keep_slots;
} pm_beam;

typedef struct pm_beam_out {
    float *scores;               /* [items, n] totals, not divided by the length */
    int32_t *parents;            /* [items, n] beam of the item, -1: none */
    int32_t *tokens;             /* [items, n], -1: none */
    int32_t *lengths;            /* [items, n], or NULL */
    uint8_t *done;               /* [items, n] (token == eos, or the parent was done), or NULL */
} pm_beam_out;

/* The workspace is 16-byte aligned. */
PM_API size_t pm_beam_select_workspace_bytes(const pm_beam *b);
PM_API int pm_beam_select(const pm_beam *b, const pm_beam_out *out, void *workspace, size_t workspace_bytes,
                          void *stream);

/* Moves per-beam states to the beams that continue them (no counterpart in
 * the reference): row i * beams + j of every state becomes row i * beams +
 * parents[i, j] as it was before the call; a parent outside [0, beams) leaves
 * the row its own.  One launch moves up to PM_MAX_STATES states, in place
 * (dst == src, the same strides; only rows whose parent is another are
 * touched) or into a second buffer (every row is written).  A row is `outer`
 * runs of run_bytes bytes each.  With lengths [items, beams] and pos_bytes >
 * 0 only the first lengths[parent's row] positions of a run move, pos_bytes
 * bytes each; what lies behind them in the destination stays as it was.
 * States must not overlap one another, nor a state's rows and runs each other. */
#define PM_MAX_STATES 128

typedef struct pm_state {
    const void *src;
    void *dst;
    int64_t src_row_stride;      /* bytes between rows */
    int64_t dst_row_stride;
    int64_t outer;               /* runs of a row, >= 1 */
    int64_t src_outer_stride;    /* bytes between a row's runs */
    int64_t dst_outer_stride;
    int64_t run_bytes;           /* bytes of a run */
    int64_t pos_bytes;           /* bytes of one position of a run, 0: the state has no positions */
} pm_state;

PM_API int pm_beam_reorder(const pm_state *states, int32_t n_states, const int32_t *parents, int64_t parents_stride,
                           const int32_t *lengths, int64_t items, int32_t beams, void *stream);

/* Distillation loss of a draft model from a teacher's top log-probabilities
 * (no counterpart in the reference, which loads its drafters ready trained,
 * pagedmoe/mtp.py): the KL divergence that lowers the rejections of
 * pm_verify's residual mode.  Row r has the student's logits x and up to k
 * teacher entries (ids, logprobs), those of pm_top_logprobs at the same
 * temperature T; ids outside [0, vocab) are no entries.  With q = softmax(x / T):
 *   PM_TAIL_DROP    p = the entries' probabilities divided by their sum:
 *       loss = sum over the entries e of token v of p_e (log p_e - log q_v)
 *       dloss/dx_v = (q_v - p_v) / T
 *   PM_TAIL_BUCKET  p as given; the rest p_t = max(0, 1 - sum p) and q_t = the
 *       student's mass outside the entries are one more outcome:
 *       loss = sum p_e (log p_e - log q_v) + p_t (log p_t - log q_t)
 *       dloss/dx_v = (q_v - p_v) / T on the entries, q_v (1 - p_t / q_t) / T elsewhere
 *       (q_t below 2^-100 counts as 2^-100; without a token outside the
 *       entries the bucket is left out)
 * p_v is the sum of the token's entries.  Entries that list an id twice stay two
 * outcomes of the teacher: the loss is the divergence of the summed
 * probabilities plus sum p_e log(p_e / p_v), a constant that may take it below
 * 0.  A row whose entries hold no mass has loss 0 and gradient 0 under
 * PM_TAIL_DROP.  weights [rows] multiply the rows; a row of weight 0 is not
 * read, its loss and gradient are 0.  PM_REDUCE_MEAN divides by the sum of the
 * weights (by rows without weights; a sum of 0 gives 0).  1 <= k <= 256. */
#define PM_TAIL_DROP 0
#define PM_TAIL_BUCKET 1
#define PM_REDUCE_NONE 0
#define PM_REDUCE_SUM 1
#define PM_REDUCE_MEAN 2

typedef struct pm_distill {
    const void *logits;          /* [rows, row_stride] of dtype */
    int32_t dtype;               /* PM_DTYPE_* */
    int64_t rows;
    int64_t vocab;
    int64_t row_stride;
    const int32_t *ids;          /* [rows, k] */
    const float *logprobs;       /* [rows, k] */
    int32_t k;
    double inv_temperature;      /* as in pm_top_rows */
    int32_t tail;                /* PM_TAIL_* */
    int32_t reduction;           /* PM_REDUCE_* */
    const float *weights;        /* [rows], or NULL */
} pm_distill;

/* loss: [rows] under PM_REDUCE_NONE, else one value; NULL: only the gradient.
 * grad: [rows, grad_stride] of the logits' type, or NULL: only the loss; it
 * must not overlap the logits.  grad_loss: the gradient of whatever follows
 * with respect to the loss, [rows] under PM_REDUCE_NONE, else one value; NULL
 * means 1. */
/* The workspace is 16-byte aligned. */
PM_API size_t pm_distill_workspace_bytes(const pm_distill *d);
PM_API int pm_distill_loss(const pm_distill *d, float *loss, void *grad, int64_t grad_stride,
                           const float *grad_loss, void *workspace, size_t workspace_bytes, void *stream);

/* grad *= *factor (device memory) over [rows, vocab], nothing where it is 1:
 * a gradient computed with its loss, once the loss's own gradient is known. */
PM_API int pm_distill_scale(void *grad, int32_t dtype, int64_t rows, int64_t vocab, int64_t grad_stride,
                            const float *factor, void *stream);

/* pm_sample_rows on scratch owned by the library (no counterpart in the
 * reference, which runs on MLX's allocator): for callers that cannot hand
 * over a device workspace or must not allocate between decode steps.
 * The scratch is a fixed device array of PM_STATIC_SCRATCH_BYTES per device;
 * a call whose rows need more (pm_sample_workspace_bytes(rows) larger than
 * that) returns PM_ERR_WORKSPACE and does nothing: use pm_sample_rows with a
 * workspace of that size instead.  The first call on a device looks the
 * scratch address up, so make it before any stream capture.  Nothing in the
 * scratch needs to start at zero.  One scratch per device: calls on the same
 * device must not overlap (they race on it); keep them on one stream or
 * serialise them. */
#define PM_STATIC_SCRATCH_BYTES (32u << 20)
PM_API int pm_sample_rows_static(const pm_rows *rows, const pm_noise *noise, const pm_sample_out *out,
                                 void *stream);

/* Self-check of the hardware 2^a that the bracketed statistics rely on (no
 * counterpart in the reference): evaluates it on the current device for
 * every fp32 a in [-126, 1] and writes the largest relative error against
 * the fp64 2^a to *max_rel_err (host memory).  Synchronous; allocates and
 * frees a few bytes of device memory.  The library's error budget assumes
 * at most 2^-20. */
PM_API int pm_selfcheck_ex2(double *max_rel_err);

/* Last CUDA error seen by this thread (cudaError_t value), 0 if none. */
PM_API int pm_last_cuda_error(void);

/* Library version string. */
PM_API const char *pm_version(void);

#ifdef __cplusplus
}
#endif

#endif /* PM_SAMPLE_H */
