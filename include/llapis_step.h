/*
 * llapis_step.h -- the operators of a decode step around the MoE layer
 * (llapis_moe.h): a paged key-value cache with its append, attention and page
 * operations, pages and slots for a step's new tokens, the norms and rotary
 * positions of queries and keys, the norms before and after a block, sampling
 * and the verification of drafted tokens.
 *
 * The conventions are llapis_moe.h's: device pointers and a hipStream_t of the
 * current device passed as void*, nothing allocated, launches on that stream
 * only, no kernel that waits on another workgroup; 0 on success, -1 on a
 * refused call with the reason in llapis_last_error().  A refused call has
 * launched nothing.  Every call can be captured in a HIP graph, writes each
 * workspace word before it reads it and may share a workspace with calls that
 * it does not overlap.  Results do not depend on how workgroups are scheduled.
 */
#ifndef LLAPIS_STEP_H
#define LLAPIS_STEP_H

#include <stdint.h>

#include "llapis_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ggml's tags of the 16-bit types (with LLAPIS_T_F32 and LLAPIS_T_Q8_0) */
enum { LLAPIS_T_F16 = 1, LLAPIS_T_BF16 = 30 };

/* ------------------------------------------------------- paged cache
 *
 * One layer's keys and values in pages of page_size tokens (16, 32, 64, 128
 * or 256), head_dim 64, 96, 128, 192, 256 or 512:
 *   a K page [n_kv][page_size][head_dim], a V page [n_kv][head_dim][page_size]
 * in F16 or BF16.  V is held transposed: the matrix cores take eight keys of
 * one column at a time.  In Q8_0 each head's part of a page is its int8 values
 * in that order and after them their fp16 scales [head_dim / 32][page_size]
 * (K's and V's alike), one for 32 consecutive values of a token's vector:
 * ggml's q8_0 blocks with the planes apart (d = amax / 127 rounded to fp16,
 * q = x times the fp32 reciprocal of the unrounded d, rounded to nearest even; a
 * block with a NaN has a NaN scale, one with an infinity an infinite one: either is
 * NaN throughout).  Attention takes a value q d from fp16 parts: one that rounds
 * past fp16's largest, 65504, which takes a scale of 515 and more, is read as NaN.
 * Page p is at base + p * stride bytes; strides are multiples of 16 and at
 * least llapis_kv_page_bytes (pages of several layers may interleave). */
typedef struct llapis_kv_cache {
    int32_t  type;                 /* LLAPIS_T_F16, LLAPIS_T_BF16 or LLAPIS_T_Q8_0 */
    int32_t  n_kv, head_dim, page_size, n_pages;
    void *   k;                    /* 16-byte aligned */
    void *   v;
    uint64_t k_stride, v_stride;
} llapis_kv_cache;
/* Bytes of a K page (a V page is as long); 0 if unsupported. */
uint64_t llapis_kv_page_bytes(int32_t type, int32_t n_kv, int32_t head_dim, int32_t page_size);

/* The sequences of a step.  Sequence s has lens[s] tokens, its new ones among
 * them, on the pages page_table[s * table_stride + i] (token t: entry
 * t / page_size).  Its new tokens are rows new_start[s] .. new_start[s + 1] - 1
 * of the step's activations, the last of its tokens in order (new_start NULL:
 * row s alone).  All three arrays are read on the device when the call runs, and
 * stay as they are until it has; a sequence may have no token or no new one.  The host gives the bounds:
 * n_tokens rows, max_new new tokens of a sequence, max_pages table entries a
 * row.  What lies beyond them is not touched: rows past n_tokens, new tokens
 * past max_new of a sequence, keys past max_pages * page_size.  A table entry
 * outside 0 .. n_pages - 1 has no page: its keys are masked and what would be
 * appended there is dropped.  An append takes fewer than 2^24 sequences. */
typedef struct llapis_kv_batch {
    int32_t n_seq, n_tokens, max_new, max_pages;
    int64_t table_stride;          /* entries from a sequence's row to the next */
    const int32_t * page_table;    /* [n_seq][table_stride] */
    const int32_t * lens;          /* [n_seq] */
    const int32_t * new_start;     /* [n_seq + 1] or NULL */
} llapis_kv_batch;

/* Write the new tokens' keys and values into their pages: k, v [n_tokens]
 * [n_kv][head_dim] of x_type (F32, F16 or BF16), rows k_stride / v_stride
 * values apart, rounded to nearest even into F16 / BF16 or quantised.  Any
 * number of new tokens (prompt chunks too).  Two tokens must not share a slot. */
int32_t llapis_kv_append(const llapis_kv_cache * c, const llapis_kv_batch * b, int32_t x_type, const void * k,
                         int64_t k_stride, const void * v, int64_t v_stride, void * stream);

/* Attention of the new tokens (llapis_kv_batch.max_new <= 16) over the cache,
 * into which they have been appended.  Token at position t of its sequence,
 * query head a, on kv head a / (n_head / n_kv): over the keys i <= t, with
 * window > 0 those with i > t - window,
 *   out = sum_i e^(s_i) v_i / sum_i e^(s_i),   s_i = scale q . k_i
 *   lse = ln sum_i e^(s_i)
 * A row that sees no key gets out 0 and lse -infinity, whatever the masked
 * places hold.  q, out: [n_tokens][n_head][head_dim] of `type`, rows q_stride /
 * out_stride values apart, 16-byte aligned, out apart from q; lse [n_tokens]
 * [n_head] or NULL.
 * Scores, sums and the running maximum are fp32, and cached values enter with all
 * their bits.  Queries and probabilities are multiplied as sums of 16-bit parts, equal
 * to them to 2^-22 and better (a part in 2^37 of the row's largest is the least); 16-bit
 * queries exactly; the probabilities of 16-bit results over BF16 pages to 2^-17, a
 * 64th of an F16 result's own rounding, a 512th of a BF16 one's.
 * Refused: batches of 2^29 and more units of work (64 or 128 keys of a kv head), and
 * with several units a head of 2^24 and more (sequence, kv head, 32 query rows). */
typedef struct llapis_kv_query {
    int32_t type, n_head, window;
    float   scale;
    const void * q;
    int64_t q_stride;
    void *  out;
    int64_t out_stride;
    float * lse;
} llapis_kv_query;
/* Device scratch (bytes) of an attention call; 0 if it would be refused.  It serves
 * every call of fewer sequences, new tokens and pages too.
 * Reads c's geometry, b's n_seq, max_new and max_pages, and n_head. */
uint64_t llapis_kv_attention_workspace_size(const llapis_kv_cache * c, const llapis_kv_batch * b, int32_t n_head);
int32_t  llapis_kv_attention(const llapis_kv_cache * c, const llapis_kv_batch * b, const llapis_kv_query * a,
                             void * workspace, uint64_t ws_bytes, void * stream);

/* The same attention (without a window) of a batch whose sequences begin with the
 * same tokens on the same pages, as llapis_kv_fork leaves them: group g is the
 * sequences groups[g] .. groups[g + 1] - 1, in whose rows of the page table the first
 * prefix[g] tokens' entries are the same; they are read from the first of them with new
 * tokens, once for the whole group (in tiles of 64 to 256 query rows of a kv head),
 * and each sequence's other keys are attended as above.  Both arrays are read on the
 * device; groups are in order (as the rows of new_start are), sequences before the first
 * and behind the last share nothing.  A prefix is cut to what every sequence of its group
 * with new tokens had before them, and to a multiple of 64 tokens and of a page; what is
 * cut off counts as each one's own.  Results are llapis_kv_attention's but for the order
 * of sums, with its precision of every part.  n_group is 256 at most; with none the call
 * is attention's.  Refused: what attention refuses, and with groups more than 2^24 rows
 * (n_tokens), 2^31 query rows of a kv head and more, 2^24 and more (sequence, kv head,
 * 32 query rows) however short the table, and prefixes of 2^30 and more units of work (32
 * or 64 keys of a kv head for a tile of rows).  The workspace serves every call of fewer
 * sequences, rows, new tokens, pages and groups too; its size reads b's n_tokens beside
 * what attention's does. */
typedef struct llapis_kv_prefix {
    int32_t n_group;
    const int32_t * groups;        /* [n_group + 1] */
    const int32_t * prefix;        /* [n_group] */
} llapis_kv_prefix;
uint64_t llapis_kv_prefix_attention_workspace_size(const llapis_kv_cache * c, const llapis_kv_batch * b, int32_t n_head,
                                                   int32_t n_group);
int32_t  llapis_kv_prefix_attention(const llapis_kv_cache * c, const llapis_kv_batch * b, const llapis_kv_query * a,
                                    const llapis_kv_prefix * x, void * workspace, uint64_t ws_bytes, void * stream);

/* ------------------------------------------------------------- pages
 *
 * Operations on whole pages, the same in every plane: a plane is one layer's
 * K or V pool, pages of `bytes` bytes (a multiple of 16) `stride` apart.  More
 * planes than LLAPIS_KV_MAX_PLANES take several calls.  n_pages and max_pages are
 * 2^30 at most, n_seq below 2^24 in page_refs and compact, n_forks 65535 at most. */
#define LLAPIS_KV_MAX_PLANES 128
typedef struct llapis_kv_planes {
    int32_t n_planes, n_pages, page_size;
    int32_t reserved;
    void *   base[LLAPIS_KV_MAX_PLANES];       /* 16-byte aligned */
    uint64_t stride[LLAPIS_KV_MAX_PLANES];
    uint64_t bytes[LLAPIS_KV_MAX_PLANES];
} llapis_kv_planes;

/* Copy page pairs[2 i] to page pairs[2 i + 1] in every plane, i < n_pairs
 * (device array).  A pair with an id outside the pool is skipped.  No page may
 * be the target of two pairs, nor the target of one and the source of another. */
int32_t llapis_kv_copy_pages(const llapis_kv_planes * p, const int32_t * pairs, int32_t n_pairs, void * stream);

/* Fork sequences: forks [n_forks][3] (device array) of {source row, target
 * row, fresh page}.  The target gets the source's length and shares its full
 * pages; a partly filled last page is copied to the fresh page, which takes its
 * place in the target's row (a source that ends on a page's border leaves the
 * fresh page unused).  The rest of the target's row becomes -1.  A fork is
 * skipped whose rows are outside the table or the same, whose length is
 * outside 0 .. max_pages * page_size, or which needs a fresh page and has none
 * in the pool; so is one whose source has no valid last page to copy.  No row
 * may be the target of two forks or of one and the source of another, and the
 * fresh pages must be free and different. */
int32_t llapis_kv_fork(const llapis_kv_planes * p, int32_t * page_table, int64_t table_stride, int32_t max_pages,
                       int32_t * lens, int32_t n_seq, const int32_t * forks, int32_t n_forks, void * stream);

/* Which pages are in use: refs [n_pages] = how many of the n_seq rows' entries
 * within their lengths name a page (a sequence is freed by setting its length
 * to 0), free_pages [n_pages] = the pages of no reference, ascending, then -1;
 * n_free [1].  free_pages and n_free may be NULL.  With refs in hand a page
 * that several sequences share is told from one that may be written. */
int32_t llapis_kv_page_refs(int32_t n_pages, int32_t page_size, const int32_t * page_table, int64_t table_stride,
                            int32_t max_pages, const int32_t * lens, int32_t n_seq, int32_t * refs,
                            int32_t * free_pages, int32_t * n_free, void * stream);

/* Move the pages in use to the front of the pool: with n_live pages referenced,
 * the i-th referenced page (ascending) at or past n_live moves to the i-th free
 * page before n_live, in every plane, and table_out (the layout of page_table)
 * names the new places: entries beyond a row's length, or that name no page,
 * become -1.  page_table is left as it is unless table_out is page_table.
 * refs [n_pages] (NULL: not wanted) gets the counts at the new places, n_live
 * [1] the number of pages in use: pages n_live .. n_pages - 1 are free.  All
 * planes of a pool have to move by one call or by calls with the same
 * page_table.  The workspace holds llapis_kv_compact_workspace_size bytes. */
uint64_t llapis_kv_compact_workspace_size(int32_t n_pages);
int32_t  llapis_kv_compact(const llapis_kv_planes * p, const int32_t * page_table, int64_t table_stride,
                           int32_t max_pages, const int32_t * lens, int32_t n_seq, int32_t * table_out, int32_t * refs,
                           int32_t * n_live, void * workspace, uint64_t ws_bytes, void * stream);

/* ------------------------------------------- pages and slots of a step
 *
 * Make room for the new tokens of a step: sequence s of lens[s] tokens asks for
 * n_new[s] more (negative numbers count as 0).  A sequence gets all that it asks
 * for or nothing.  It gets nothing where
 *   - lens[s] + n_new[s] tokens are more than its row's max_pages hold, else where
 *   - the asked of sequences 0 .. s that passed are more than n_tokens, else where
 *   - it needs a page, and the pages that sequences 0 .. s need that passed are
 *     more than n_free.
 * Pages come from the end of free_pages (an array of n_pages entries, of which the
 * first n_free[0] are free), sequence by sequence: entry ceil(lens / page_size) of
 * a row and those behind it.  Then, each array as long as the new state needs:
 *   lens_out [n_seq]       lengths with the new tokens (may be lens)
 *   n_free_out [1]         the free pages left, the first of free_pages (may be n_free)
 *   new_start [n_seq + 1]  first row of each sequence's new tokens: llapis_kv_batch's
 *   pos, seq [n_tokens]    a row's position in its sequence, and which that is
 *   slots [n_tokens]       page * page_size + place in the page; -1 without a page
 * with -1 in rows past the last token; pos, seq and slots may be NULL.  n_seq is
 * below 2^24, n_tokens, n_pages and max_pages * page_size 2^30 at most. */
typedef struct llapis_kv_extend_args {
    int32_t page_size, n_pages, n_seq, n_tokens, max_pages;
    int32_t reserved;
    int64_t table_stride;
    int32_t * page_table;
    const int32_t * lens;
    const int32_t * n_new;
    const int32_t * free_pages;
    const int32_t * n_free;
    int32_t * lens_out;
    int32_t * n_free_out;
    int32_t * new_start;
    int32_t * pos;
    int32_t * seq;
    int64_t * slots;
} llapis_kv_extend_args;
uint64_t llapis_kv_extend_workspace_size(int32_t n_seq);
int32_t  llapis_kv_extend(const llapis_kv_extend_args * a, void * workspace, uint64_t ws_bytes, void * stream);

/* ------------------------------------- norms and positions of q and k
 *
 * Frequencies of a rotation, computed on the host: freq[i], i < rot_dim / 2, is
 * base^(-2 i / rot_dim), divided by divisors[i] (NULL: none), and with `kind`
 *   LINEAR  divided by factor;
 *   NTK     from the base  base * factor^(rot_dim / (rot_dim - 2));
 *   YARN    f (1 - r) + f / factor r, r = (i - lo) / (hi - lo) within 0 .. 1,
 *           lo = floor(d(high)) >= 0, hi = ceil(d(low)) <= rot_dim - 1 (0.001 apart at
 *           least), d(t) = rot_dim ln(trained / (2 pi t)) / (2 ln base);
 *   BANDS   f s + f / factor (1 - s), s = (trained f / (2 pi) - low) / (high - low)
 *           within 0 .. 1.
 * low and high are turns over the trained length (YARN: 1 and 32, BANDS: 1 and 4
 * are usual).  *magnitude, what cosine and sine are multiplied by: 0.1 ln factor + 1
 * for YARN with a factor above 1, else 1. */
enum { LLAPIS_ROPE_PLAIN = 0, LLAPIS_ROPE_LINEAR = 1, LLAPIS_ROPE_NTK = 2, LLAPIS_ROPE_YARN = 3, LLAPIS_ROPE_BANDS = 4 };
typedef struct llapis_rope_rule {
    int32_t kind, rot_dim;
    double  base, factor, trained, low, high;
    const double * divisors;
} llapis_rope_rule;
int32_t llapis_rope_frequencies(const llapis_rope_rule * rule, double * freq, float * magnitude);

/* The norms of queries and keys for each head, and their rotary positions, in
 * one pass: for every head x of head_dim values (up to 512) of a token at pos[t]
 *   y = norm ? x / sqrt(mean x^2 + eps) * weight : x
 *   (y_a, y_b) -> magnitude (y_a cos z - y_b sin z, y_b cos z + y_a sin z),  z = pos[t] freq[i]
 * for i < rot_dim / 2 with, by `layout`, (a, b) = (i, i + rot_dim / 2) or (2 i, 2 i + 1);
 * values from rot_dim on are not rotated (rot_dim 0: none are).  Angles are formed in
 * 64 bits, the rest in fp32, and rounded once.  q [n_tokens][n_head][head_dim] and k
 * [n_tokens][n_kv][head_dim] (n_kv 0: no k) are of `type`, rows q_stride values apart
 * and so on, in any alignment to a value; outputs may lie on inputs row for row, and
 * overlap them in no other way.  Weights fp32 [head_dim] or NULL (ones).  A row with
 * pos[t] < 0 is neither read nor written. */
enum { LLAPIS_ROPE_HALF = 0, LLAPIS_ROPE_PAIRS = 1 };
typedef struct llapis_qk_rope_args {
    int32_t type;                  /* LLAPIS_T_F32, LLAPIS_T_F16 or LLAPIS_T_BF16 */
    int32_t n_tokens, n_head, n_kv, head_dim, rot_dim, layout, norm;
    float   eps, magnitude;
    const int32_t * pos;           /* [n_tokens]; NULL with rot_dim 0: every row */
    const double *  freq;          /* [rot_dim / 2] */
    const void *  q;      int64_t q_stride;
    void *        q_out;  int64_t q_out_stride;
    const float * q_weight;
    const void *  k;      int64_t k_stride;
    void *        k_out;  int64_t k_out_stride;
    const float * k_weight;
} llapis_qk_rope_args;
int32_t llapis_qk_rope(const llapis_qk_rope_args * a, void * stream);

/* -------------------------------------------------------- block norms
 *
 * What lies between one block and the next of a residual stream, in one
 * kernel (llapis_residual_rmsnorm with the parts that sandwich-normed models
 * have: gemma4's layer norms the block's output before it is added, scales the
 * layer's output, and feeds its dense FFN, its router and its experts from
 * three norms of the same stream, gemma4.cpp:384-430):
 *   u  = post_norm ? y / rms(y) * post_weight : y
 *   h' = alpha h + beta gate u
 *   x_j = h' / rms(h') * weight_j      j < n_out
 * with rms(z) = sqrt(mean z^2 + eps) over a token's d values, sums in fp32;
 * each output is rounded once (x_j is computed from the unrounded h').
 * Activations are of `type`, weights fp32; y NULL leaves the second term out.
 * h_out and the x_j may lie on h or y row for row; other overlaps are not allowed. */
#define LLAPIS_NORM_MAX_OUT 4
typedef struct llapis_block_norm_args {
    int32_t type;                  /* LLAPIS_T_F32, LLAPIS_T_F16 or LLAPIS_T_BF16 */
    int32_t n_tokens, d, n_out;    /* d <= 16384, n_out <= LLAPIS_NORM_MAX_OUT */
    int32_t post_norm;
    float   eps, alpha, beta;
    const void *  h;      int64_t h_stride;          /* [n_tokens][d], rows h_stride values apart */
    const void *  y;      int64_t y_stride;          /* [n_tokens][d] or NULL */
    const float * post_weight;                       /* [d] or NULL (ones) */
    const void *  gate;                              /* or NULL (ones): value (t, i) at */
    int64_t gate_token_stride, gate_value_stride;    /* t gate_token_stride + i gate_value_stride (0 or 1) */
    void *  h_out;        int64_t h_out_stride;      /* or NULL; may be h */
    const float * weight[LLAPIS_NORM_MAX_OUT];       /* [d] or NULL (ones) */
    void *  x[LLAPIS_NORM_MAX_OUT];
    int64_t x_stride[LLAPIS_NORM_MAX_OUT];
} llapis_block_norm_args;
int32_t llapis_block_norm(const llapis_block_norm_args * a, void * stream);

/* ----------------------------------------------------------- sampling
 *
 * The next token of each sequence from its logits [n_seq][vocab] of `type`, rows
 * logits_stride values apart, with numbers u [n_seq] in [0, 1) that the caller
 * draws.  With M a row's largest logit, values in the order (value descending,
 * index ascending) and w_i = e^((x_i - M) / temperature):
 *   top_k   keeps the first top_k values (0 and less: all);
 *   top_p   keeps of those the fewest first ones whose weights' sum is at least
 *           top_p of theirs (1 and more: all), the first always;
 *   min_p   keeps of those the ones with w_i >= min_p (M's weight is 1);
 *   the token is the smallest v for which the kept w_0 + .. + w_v > u sum w.
 * A temperature that is not positive, and a min_p above 1, take the first value.
 * The settings are read on the device, one for each sequence; NULL: temperature 1,
 * the others off.  Weights are fp64, their sums fp64 or, next to where a filter
 * ends, whole numbers of 2^-49 or less of the largest weight there: as little as lets
 * top_p end within a 32nd of a value's weight of its place in rows of up to 2^20 values.
 * NaN and -infinity are no values (the token of a row without any is -1); where
 * +infinity is the largest, the others have no weight.  With top_k or top_p a value
 * whose weight is below 2^-63 may not be kept.
 * probs [n_seq][vocab] of `type`, rows probs_stride apart, or NULL: the probabilities
 * that the token was drawn with, rounded once (what llapis_verify_drafts takes as a
 * draft's); not on logits.  n_seq is 65535 at most, vocab 2^30 (else the workspace size is 0). */
typedef struct llapis_sample_args {
    int32_t type;                  /* LLAPIS_T_F32, LLAPIS_T_F16 or LLAPIS_T_BF16 */
    int32_t n_seq, vocab;
    const void *    logits;  int64_t logits_stride;
    const float *   u;
    const float *   temperature;
    const int32_t * top_k;
    const float *   top_p;
    const float *   min_p;
    int32_t *       tokens;
    void *          probs;   int64_t probs_stride;
} llapis_sample_args;
uint64_t llapis_sample_workspace_size(int32_t n_seq, int32_t vocab);
int32_t  llapis_sample(const llapis_sample_args * a, void * workspace, uint64_t ws_bytes, void * stream);

/* ------------------------------------------------ draft verification
 *
 * The end of a speculative step: of n drafted tokens x_0 .. x_(n-1) of a
 * sequence, the first a that the target model takes, and one token more.
 * target [n_seq][max_draft + 1][vocab] are the target's probabilities at each
 * draft's place and behind the last, draft [n_seq][max_draft][vocab] those the
 * drafts were drawn from (NULL: the drafts were certain), of `type`, rows
 * target_stride / draft_stride values apart (a sequence's rows follow each
 * other); drafts [n_seq][max_draft]; n_draft [n_seq] (NULL: max_draft each);
 * u [n_seq][max_draft] and u_next [n_seq] given numbers in [0, 1).
 *   draft i is taken iff every earlier one was and u_i q_i(x_i) < p_i(x_i);
 *   r = max(p_a - q_a, 0) if a < n (p_a itself where that is 0 everywhere),
 *       p_n if all were taken;
 *   the next token is the smallest v with r_0 + .. + r_v > u_next sum r.
 * Products, differences and sums are fp64.  Values that are not positive and
 * finite count as 0, a draft outside the vocabulary is not taken; n_draft is
 * clamped to 0 .. max_draft.  tokens [n_seq][max_draft + 1] receives the taken
 * drafts, the next token and -1 behind it, accepted [n_seq] the number a.  The
 * next token is -1 where the target row has no positive value.  n_seq is 65535
 * at most, max_draft 63, vocab 2^30 (the workspace size of more is 0). */
typedef struct llapis_verify_args {
    int32_t type;                  /* LLAPIS_T_F32, LLAPIS_T_F16 or LLAPIS_T_BF16 */
    int32_t n_seq, max_draft, vocab;
    const void * target;  int64_t target_stride;
    const void * draft;   int64_t draft_stride;
    const int32_t * drafts;
    const int32_t * n_draft;
    const float * u;
    const float * u_next;
    int32_t * tokens;
    int32_t * accepted;
} llapis_verify_args;
uint64_t llapis_verify_drafts_workspace_size(int32_t n_seq, int32_t vocab);
int32_t  llapis_verify_drafts(const llapis_verify_args * a, void * workspace, uint64_t ws_bytes, void * stream);

#ifdef __cplusplus
}
#endif
#endif
