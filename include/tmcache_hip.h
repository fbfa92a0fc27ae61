/*
 * tmcache_hip.h -- C ABI of the paged key/value cache operators (gfx950), in
 * the same library as tmsample_hip.h and by the same rules: device pointers,
 * sizes, a hipStream_t, an int status; the calls allocate nothing, are
 * stream-ordered, never synchronise and can be captured into a HIP graph, and
 * run on the current device (the stream's device must be current).
 * There is no context: scratch memory is the caller's (`workspace`).
 * TensorMark keeps one sequence's keys and values in one flat host buffer
 * (tensormark/llama.h, the kv_* members of Llama); nothing of it is paged or
 * bounded, so these calls have no counterpart to cite line by line.
 *
 * Layout.  A pool holds `pages` pages of `page_size` slots for each of
 * `kv_heads` heads; a slot is head_dim values, contiguous; the page, head and
 * slot strides are the caller's.  Sequence b's position j is slot
 * j % page_size of page tables[b][j / page_size].  An entry outside
 * [0, pages) is an unmapped page: nothing is read from or written to it, and
 * its positions are seen by no row.  Positions at or past
 * table_stride * page_size, and at or past kv_len[b], do not exist.
 *
 * New tokens.  Sequence b's are q_start[b] <= t < q_start[b + 1] of the
 * call's `tokens`, and stand at the last positions of its kv_len[b] (which
 * counts them): token t is position kv_len[b] - (q_start[b + 1] - t).
 * `max_q` and `max_kv` are host bounds on any sequence's new tokens and
 * kv_len: new tokens past max_q are left out, and so are positions past max_kv
 * in tms_kv_add_scores and tms_kv_evict (attention reads them, more slowly).
 * Lengths are taken as at most 2^29.
 *
 * Past the limits below a call answers TMS_ERR_CAPACITY.
 *
 * Visible positions.  A row at position p sees j <= p on mapped pages; with
 * window > 0 only j > p - window or j < sinks.
 */
#ifndef TMCACHE_HIP_H
#define TMCACHE_HIP_H

#include "tmsample_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TMS_CACHE_MAX_HEAD_DIM 256
#define TMS_CACHE_MIN_PAGE 8
#define TMS_CACHE_MAX_PAGE 65536
#define TMS_CACHE_MAX_PAIRS 1048576              /* batch times kv_heads */
#define TMS_CACHE_MAX_TOKENS 268435456
#define TMS_APPEND_MAX_BATCH 65535
#define TMS_SCORES_MAX_KV 4194304                /* max_kv */
#define TMS_ATTENTION_MAX_SLOT_STRIDE 67108864   /* elements; tms_paged_attention */
#define TMS_ATTENTION_MAX_ROWS 2097152           /* max_q times query heads a key head; where a page's stride or
                                                    slots span 2^32 bytes, batch times kv_heads times
                                                    tiles of 32 such rows is below 2^31 too */
#define TMS_SCORES_MAX_Q_STRIDE 8388608          /* elements between tokens, and that a key head's
                                                    query heads span; tms_kv_add_scores */

/* The pools, page tables and lengths of one call. */
typedef struct tms_cache {
    void* k;                  /* device, keys; 16-byte aligned */
    void* v;                  /* device, values; 16-byte aligned; unused (may be null)
                                 by tms_kv_add_scores */
    float* scores;            /* device, [pages][kv_heads][page_size], 16-byte aligned,
                                 nullable (not in tms_kv_add_scores, tms_kv_evict): the
                                 attention weight each key has drawn so far */
    int64_t k_stride[3];      /* elements between pages, heads, slots: multiples of 8 */
    int64_t v_stride[3];
    int32_t dtype;            /* TMS_DTYPE_F16 or TMS_DTYPE_BF16 */
    int32_t pages;
    int32_t kv_heads;
    int32_t page_size;        /* a power of two, TMS_CACHE_MIN_PAGE..TMS_CACHE_MAX_PAGE */
    int32_t head_dim;         /* a multiple of 8 up to TMS_CACHE_MAX_HEAD_DIM */
    int32_t batch;
    const int32_t* tables;    /* device, [batch][table_stride] page ids */
    int64_t table_stride;
    const int32_t* kv_len;    /* device, [batch] */
    const int32_t* q_start;   /* device, [batch + 1]; unused (may be null) by tms_kv_evict */
    int32_t tokens;           /* rows of the new tokens' tensors */
    int32_t max_q;
    int32_t max_kv;
    int32_t reserved;         /* must be 0 */
} tms_cache;

/*
 * Write the new tokens' keys and values to their slots and zero those slots'
 * scores.  k_new, v_new: device, [tokens][kv_heads][head_dim] of the cache's
 * dtype, with strides (elements, multiples of 8) between tokens and heads,
 * 16-byte aligned.  Tokens whose position is negative, past the table or on
 * an unmapped page are dropped.  A page that two sequences share is written
 * by both, in no order.
 */
typedef struct tms_append_args {
    const void* k_new;
    const void* v_new;
    int64_t k_new_stride[2];  /* token, head */
    int64_t v_new_stride[2];
} tms_append_args;
int tms_kv_append(const tms_cache* cache, const tms_append_args* args, hipStream_t stream);

/*
 * Attention of the new tokens' queries over the cache: for each token and
 * query head (head h reads key head h / (q_heads / kv_heads)), over its
 * visible positions j,
 *   s_j = scale * q . k_j,  lse = log(sum_j exp(s_j)),
 *   out = sum_j exp(s_j - lse) v_j.
 * A row that sees nothing (or every s_j = -inf) gives out = 0, lse = -inf.
 * scale is any finite number.  Sums and products are held in fp32; the weights are rounded once to the
 * cache's dtype for the product with v, the output once at the end.  The
 * same inputs give the same bits on every call.
 */
typedef struct tms_attention_args {
    const void* q;            /* device, [tokens][q_heads][head_dim]; 16-byte aligned */
    void* out;                /* device, like q, of the same dtype; may be q itself with q's
                                 strides, and shares no other memory with the inputs */
    float* lse;               /* device, [tokens][q_heads] contiguous, nullable */
    int64_t q_stride[2];      /* token, head: multiples of 8 */
    int64_t out_stride[2];
    int32_t q_heads;          /* a multiple of kv_heads */
    int32_t window;           /* <= 0: none */
    int32_t sinks;            /* with a window: first positions that stay visible */
    float scale;
    void* workspace;          /* device, 16-byte aligned, tms_paged_attention_workspace bytes;
                                 contents need not be kept or cleared */
    size_t workspace_bytes;
} tms_attention_args;
/* Bytes of workspace that the call needs (0 is possible); a TMS_ERR_* code,
 * negative, for arguments that the call would refuse. */
int64_t tms_paged_attention_workspace(const tms_cache* cache, const tms_attention_args* args);
int tms_paged_attention(const tms_cache* cache, const tms_attention_args* args, hipStream_t stream);

/*
 * Add to each key's score the weight that the new tokens' queries give it:
 *   out[j] = scores[j] + sum over rows that see j of exp(scale * q . k_j - lse).
 * `lse` is tms_paged_attention's, for the same q, window, sinks and scale;
 * rows with lse = -inf add nothing.  `out` has the layout of cache->scores
 * and may be the same array, but not overlap it otherwise; every mapped position below kv_len is written,
 * nothing else.  Sums are in a fixed order.  A page that two sequences share
 * may get either one's sum.
 */
typedef struct tms_score_args {
    const void* q;            /* as in tms_attention_args */
    const float* lse;         /* device, [tokens][q_heads] contiguous */
    float* out;               /* device; null: cache->scores */
    int64_t q_stride[2];
    int32_t q_heads;
    int32_t window;
    int32_t sinks;
    float scale;
} tms_score_args;
int tms_kv_add_scores(const tms_cache* cache, const tms_score_args* args, hipStream_t stream);

/*
 * Cut each sequence to at most `budget` positions, per head.  Positions on
 * unmapped pages go first of all and are never kept.  Of the others, those
 * below `sinks` and among the last `recent` of the kv_len[b] positions are kept,
 * then those of the largest scores (ties: the lowest position; a NaN score ranks below
 * every number).  Kept entries keep their order and go, with their scores,
 * to positions 0, 1, ... of dst_tables (pages of the same pools that are none
 * of the sequence's own, or of another's of this call).  new_len[b] is the
 * number kept, min(budget, positions on mapped pages); kept[b][h][i] is the old
 * position of new position i, -1 past new_len.  Entries to an unmapped page
 * are not copied.
 * max_kv may be up to TMS_EVICT_MAX_KV.
 */
#define TMS_EVICT_MAX_KV 1048576
typedef struct tms_evict_args {
    const int32_t* dst_tables;   /* device, [batch][dst_table_stride] */
    int64_t dst_table_stride;    /* >= ceil(min(budget, max_kv) / page_size) */
    int32_t budget;              /* >= 1, >= sinks + recent */
    int32_t sinks;
    int32_t recent;
    int32_t reserved;            /* must be 0 */
    int32_t* new_len;            /* device, [batch]; may be the array kv_len */
    int32_t* kept;               /* device, [batch][kv_heads][budget] */
} tms_evict_args;
int tms_kv_evict(const tms_cache* cache, const tms_evict_args* args, hipStream_t stream);

/*
 * The logits rules on rows of logits, for callers that sample elsewhere or
 * verify drafts (tms_spec_verify takes rows as they are).  Row r belongs to
 * sequence r / steps and is its step r % steps; its history is the sequence's
 * first n_recent ids of `recent` and then its first (r % steps) ids of
 * `drafts`.  In order, in fp32, rounded once to out_dtype:
 *   1. ids whose mask bit is clear become -inf, whatever follows;
 *   2. repetition penalty over the last repeat_last_n ids of the history, then
 *      frequency and presence, as tms_sample_batch has them (steps 2 and 3 of
 *      tmsample_hip.h, apply_repeat_penalty, tensormark/tmsample.h:52-63);
 *   3. the sum of the sequence's biases for an id, taken in list order, is added.
 * Ids outside [0, vocab) are left out.  `out` may be `logits` (same dtype and
 * stride), but not overlap it otherwise.  Of params only repeat_penalty, repeat_last_n, frequency_penalty
 * and presence_penalty are read.
 */
typedef struct tms_adjust_args {
    const void* logits;       /* device, [seqs * steps][row_stride] of dtype */
    void* out;                /* device, [seqs * steps][out_stride] of out_dtype */
    int32_t dtype;            /* TMS_DTYPE_* */
    int32_t out_dtype;        /* dtype or TMS_DTYPE_F32 */
    int32_t seqs;
    int32_t steps;            /* rows a sequence, >= 1 */
    int32_t vocab;            /* <= 1048576 */
    int32_t n_bias;           /* biases a sequence, 0..65535 */
    int64_t row_stride;       /* >= vocab */
    int64_t out_stride;
    const tms_row_params* params;   /* device, [seqs]; nullable: no penalties */
    const int32_t* recent;    /* device, [seqs][recent_stride], nullable */
    const int32_t* n_recent;  /* device, [seqs], nullable: all n_history */
    int64_t recent_stride;    /* >= n_history */
    int32_t n_history;        /* ids that a sequence's row of `recent` holds */
    int32_t reserved;         /* must be 0 */
    const int32_t* drafts;    /* device, [seqs][steps - 1], nullable: none counted */
    const int32_t* bias_ids;  /* device, [seqs][n_bias], nullable with n_bias = 0 */
    const float* bias_values; /* device, [seqs][n_bias] */
    const uint32_t* mask;     /* device, [seqs * steps][mask_stride], nullable */
    int64_t mask_stride;      /* >= ceil(vocab / 32) */
} tms_adjust_args;
int tms_adjust_logits(const tms_adjust_args* args, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TMCACHE_HIP_H */
