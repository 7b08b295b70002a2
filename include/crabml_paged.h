/*
 * crabml_paged.h -- several sequences in one call: a key/value cache in pages, appended to and attended over, in 16 or in 8 bits.
 *
 * The ring caches of crabml_seqops.h hold one sequence each, as 32-bit numbers, and a call works on one of them.  Here the sequences of a step share a pool of
 * pages; a call carries the new tokens of all of them, as many each as it has (a prompt's portion, drafted tokens, one decoded token, none).
 *
 * Conventions are those of crabml_cuda.h and crabml_seqops.h: status codes, all work on the device's stream, nothing blocks, eager devices only.  Which pages a
 * sequence has, and how long it is, the host knows: it says so once a step, in a plan, which is checked as a whole and then used by every layer.
 */
#ifndef CRABML_PAGED_H
#define CRABML_PAGED_H

#include "crabml_seqops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the plan of a step ------------------------------------------------------------------------------------------------------- */
typedef struct cc_page_plan cc_page_plan;
typedef struct cc_page_plan_desc {
    int32_t n_seqs;
    int32_t page_size;           /* tokens of a page: 16, 32, 64 or 128 */
    int32_t table_cols;          /* pages a row of the table has room for */
    int64_t n_pages, n_slots;    /* what page and slot numbers stay below: the caches' pages, and half of their open blocks (0: caches without) */
    const int64_t* pos0;         /* [n_seqs] tokens that the sequence has in the cache: the position of its first new one */
    const int32_t* counts;       /* [n_seqs] its new tokens; 0: none */
    const int32_t* table;        /* [n_seqs, table_cols] its pages in order, of which ceil((pos0 + count) / page_size) are read */
    const int32_t* slots;        /* [n_seqs] its slot, or NULL: sequence i has slot i */
} cc_page_plan_desc;
/* The tokens of a call are rows of matrices, sequence after sequence.  Refused (CC_ERR_TENSOR): numbers out of range; a page that takes new tokens of one
 * sequence and belongs to another one too, or to the same one twice; a slot of two sequences.  Pages that no new token goes to may be shared (a common prefix).
 * The arrays are read during the call, which waits for the device only where the copies of 64 plans are still queued.  The plan stays usable until it is released;
 * work queued before that finishes with it. */
CC_API int cc_page_plan_create(cc_device* dev, const cc_page_plan_desc* desc, cc_page_plan** out);
CC_API void cc_page_plan_release(cc_page_plan* plan);
CC_API int64_t cc_page_plan_tokens(const cc_page_plan* plan);

/* ---- a layer's cache -------------------------------------------------------------------------------------------------------------- */
/* k: [n_pages, n_kv, page_size, dk], v: [n_pages, n_kv, page_size, dv]; dk and dv multiples of 16, up to 256; n_kv up to 1024, and n_heads, a multiple of it, up to 8192.
 * F16: every row rounded to 16 bits; the other four are not used (buf NULL).
 * I8: a page holds a block of page_size tokens once all of them are there.  Per head, with a the largest magnitude of the block's 16-bit numbers x: the factor
 *   a / 127 in k_scale, v_scale [n_pages, n_kv] (F32) and the codes round(127 x / a), ties to even; every number is rounded to 8 bits once, whatever portions a
 *   sequence came in.  Tokens of a block that is not complete lie in k_open, v_open [2 * n_slots, n_kv, page_size, dk / dv] (F16): block b of the sequence with
 *   slot s in row 2 s + b mod 2.  So do those of the block before it; of blocks that a call completes further back it leaves no 16-bit rows.  A sequence may go
 *   back (rejected drafts: a plan with pos0 below its length) to the start of any block, and to any token from page_size * (e / page_size - 1) on, though not
 *   below the start that it last went back to, where e is the furthest it has reached since then.  Of a sequence at the end of a block that is page_size tokens.
 *   Nothing notices one that goes back elsewhere: its block takes rows that are not its own.
 * Finite numbers beyond the range of 16 bits become its largest.  A block that holds an infinity or a NaN has the factor NaN. */
typedef struct cc_paged_cache {
    cc_view k, v, k_scale, v_scale, k_open, v_open;
} cc_paged_cache;

/* ---- from projections to pages --------------------------------------------------------------------------------------------------------- */
/* For the plan's T tokens: queries in the columns q_col0 .. q_col0 + n_heads * dk of q_src's rows, keys (n_kv * dk) and values (n_kv * dv) likewise; the three may
 * be one matrix.  freq ([P] F32 or NULL): P column pairs of every query and key head, from column `offset` on, turn by position * freq[i] (a 64-bit product), as
 *   (x, y) <- (mag (x cos - y sin), mag (y cos + x sin)); pairing as in cc_qk_prepare_append.  The turn is computed in 64 bits and rounded to F32 once.
 * The keys and values go to their pages, which are tensors of their own (one tensor for both, or for their factors or open blocks, is refused); out: F32
 * [T, n_heads * dk], the queries.  q_src NULL: keys and values alone (n_heads is ignored, *out is NULL). */
CC_API int cc_paged_append(cc_device* dev, const cc_page_plan* plan, const cc_paged_cache* cache, const cc_view* q_src, int32_t q_col0, const cc_view* k_src,
                           int32_t k_col0, const cc_view* v_src, int32_t v_col0, int32_t n_heads, const cc_view* freq, int32_t pairing, int32_t offset, float mag,
                           cc_buf** out);

/* ---- attention ------------------------------------------------------------------------------------------------------------------------ */
/* q: F32 [T, n_heads * dk].  The token at position i of its sequence sees the positions j <= i of that sequence with i - j < window (window <= 0: all), as the
 * cache holds them after the append:
 *   score = scale * (q . k), or softcap * tanh(that / softcap) with softcap > 0; softmax with a denominator that also holds exp(sink[h]) (sink: [n_heads] or
 *   NULL); the weighted sum of the values.
 * Head h reads key head h / (n_heads / n_kv).  out: F32 [T, n_heads * dv], sums of 32 bits of weights of 22: a weight is off by 2^-22 of
 * itself or by 2^-33 of the row's largest, whichever is more (8-bit pages: that holds for weights times their blocks' factors, down to 2^-64 of the largest
 * weight), and 16-bit numbers below 2^-14 are summed with the rounding errors of 2^-14.  Equal calls give equal bits on a device.  A key or value that is not finite reaches the results of
 * the queries that see it (not all of them, where its weight is zero) and no others; a query that holds a NaN or an infinity has the result NaN; rows behind a
 * sequence's end are not looked at.
 * Workspace, which the device's pool keeps: sequences with more than 32 rows (new tokens x n_heads / n_kv) have their visible keys and values of heads up to 128
 * laid out as 16-bit numbers, 64 columns and 128 tokens at a time, within 256 MB or one sequence and key head at a time, and up to 256 MB for sums of slices of
 * their keys; the others 10 MB. */
CC_API int cc_paged_attention(cc_device* dev, const cc_page_plan* plan, const cc_paged_cache* cache, const cc_view* q, int32_t n_heads, float scale, int32_t window,
                              float softcap, const cc_view* sink, cc_buf** out);

#ifdef __cplusplus
}
#endif
#endif /* CRABML_PAGED_H */
