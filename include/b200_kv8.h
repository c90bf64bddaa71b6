/* b200_kv8.h -- a paged cache of keys and values in 8 bits: what writes it, what attends over it, and what manages its pages.
 *
 * The caches of b200_ggml_ops.h hold f32 rows by cell, those of b200_ggml.h one run of rows per sequence.  Here a layer's cache is a pool of
 * pages; a page holds page_size consecutive tokens of one sequence, int8, with one f32 scale for each head of its keys and of its values:
 * a quarter of the bytes of the f32 caches, and sequences that begin alike share pages.  No counterpart in the reference.
 *
 * A page's record (b200_kv8_page_bytes, a multiple of 128):
 *   int8 k[n_head_kv][page_size][dim], int8 v[n_head_kv][page_size][vdim], float k_scale[n_head_kv], v_scale[n_head_kv]; a value is int * scale.
 * A table names the pages of every row (a sequence): table[row * table_stride + i] is the page of the tokens i * page_size .. of that row, or
 * -1.  Entries outside [0, n_pages) are pages that are not there: nothing is stored in them, nobody sees their tokens, they read as zeros.
 * A step is described as elsewhere by seq_info, int32 [4][n_seq]: the sequence's first token in the batch, its count of new tokens, its
 * row, and how many tokens the row held before.  Token i of a sequence thus stands at position held + i.  The first tokens of the
 * sequences ascend (sequences lie one behind the other); a count of 0 is a sequence that has nothing in this step.  Rows outside
 * [0, n_rows) are left out, and so is whatever lies outside the n_tokens rows of the batch.  A row appears once in a step; sequences whose
 * tables share pages may be read together, and what is stored must not lie in a shared page (b200_op_kv8_grow sees to that).
 *
 * Types of rows of activations: B200_TYPE_F32, B200_TYPE_F16, B200_TYPE_BF16, at any alignment of their own type; strides in values.
 * All functions return a b200_status, check their arguments on the host, launch on `stream` and the current device, allocate nothing, do
 * not synchronise and can be captured into CUDA graphs.  Workspaces start zeroed and serve one call after the other on one stream (graphs that
 * may run at the same time have one each).
 */
#ifndef B200_KV8_H
#define B200_KV8_H

#include "b200_ggml.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_KV8_MAX_SEQ 1024     /* sequences of a step, rows of a call of the page operators */
#define B200_KV8_MAX_CACHES 128   /* layers whose pages one call copies */

typedef struct {
    void   *pages;      /* n_pages records, 16-byte aligned */
    int32_t n_pages;
    int32_t page_size;  /* 16, 32, 64 or 128 */
    int32_t n_head_kv;
    int32_t dim, vdim;  /* multiples of 16, at most 256 */
    int32_t _pad;
} b200_kv8_cache;

/* 0 for sizes that no cache has */
B200_API size_t b200_kv8_page_bytes(int32_t page_size, int32_t n_head_kv, int32_t dim, int32_t vdim);

/* New rows k [n_tokens][n_head_kv * dim], v [n_tokens][n_head_kv * vdim] go to the pages of their sequences.  For every page and head that
 * gets new values, with a their largest magnitude and c = a / 127 (f32; below 2^-126: 0):
 *   the page begins with this call (its first token is new): scale = c;
 *   else c <= scale: the scale stays;  else: scale = max(c, 1.25 scale), and what the page held follows, q' = round(q scale_before / scale);
 *   q = round(x / scale) within -127 .. 127, 0 where the scale is 0.
 * All roundings are to the nearest, ties to even, of the exact quotient.  A page that fills up in one call is thus off by half a step of
 * its largest value at most; the steps by a quarter keep the error of one that fills token by token below 2.5 steps (half a step for each time the
 * scale grew, each a step of a scale that is 0.8 of the next).  Where one of the new values is not finite, or the scale was not, the scale
 * becomes NaN and the new q 0: whoever sees a token of that page and head gets NaN, until the page is begun anew. */
typedef struct {
    b200_kv8_cache cache;
    const void *k; int64_t k_stride;
    const void *v; int64_t v_stride;
    const int32_t *seq_info;
    const int32_t *table; int64_t table_stride;
    int32_t n_rows, n_seq, n_tokens;
    int32_t type;                          /* of k and v */
} b200_kv8_store_args;
B200_API int b200_op_kv8_store(const b200_kv8_store_args *a, b200_stream_t stream);

/* The values that the cache holds: tokens held .. held + count - 1 of each row go to rows first .. of k and v (seq_info as above, its "tokens
 * held before" being where reading begins).  k and v may be NULL each. */
typedef struct {
    b200_kv8_cache cache;
    void *k; int64_t k_stride;
    void *v; int64_t v_stride;
    const int32_t *seq_info;
    const int32_t *table; int64_t table_stride;
    int32_t n_rows, n_seq, n_tokens;
    int32_t type;                          /* of k and v */
} b200_kv8_load_args;
B200_API int b200_op_kv8_load(const b200_kv8_load_args *a, b200_stream_t stream);

/* Attention of n_head query heads (query head h reads kv head h / (n_head / n_head_kv)) over the cached tokens of the token's own row,
 * the new ones (stored before) among them: position pos sees position j where j <= pos, its page is there, and window == 0 or pos - j <
 * window or j < keep_first.  score = scale * q . k, softcap * tanh(score / softcap) where softcap > 0; softmax in f32, whose denominator
 * also holds exp(sink[h]) when sink != NULL.  A token that sees nothing gets zeros.  Rows of dst that belong to no sequence stay as they are.
 * q [n_tokens][n_head * dim], dst [n_tokens][n_head * vdim], of one type.  Sums, maxima and exponentials are f32.  int8 is exact in f16, which
 * the tensor cores take: with rows of bf16, and with f16_products != 0, queries and weights are rounded to f16 (relative to the row's largest); with rows
 * of f16 weights enter as two f16, 22 bits, and queries as they are; with rows of f32 both as two.  What a result is off by, as a share of its mass (the sum of
 * weight times |value|), besides its own rounding: with rows of f32 1e-6 or so (root mean square; in prompts 3e-6 where values are of one sign, 2^-17 at most: the tensor cores
 * cut sums off, f32 additions take over after 128 of theirs), with rows of f16 in prompts 2^-15 at most (512 of theirs), else 2^-12 of each weight, whatever the length.  Weights count in steps
 * of 2^-30 of the row's largest, times the largest scale that the values of any page in its sight have: a page 2^20 times as loud as the others leaves them 10 bits,
 * even where its own tokens have no weight.  A query that is not finite gives NaN.
 * max_new: no sequence of the step has more new tokens than that (0: not known).  It only chooses how the work is laid out.
 * n_tokens * n_head below 2^31.  The workspace is zero before its first call and may then go from call to call of one stream, whatever their sizes; the bytes
 * asked for do not depend on lengths.  */
typedef struct {
    b200_kv8_cache cache;
    const void *q; int64_t q_stride;
    void *dst; int64_t dst_stride;
    const int32_t *seq_info;
    const int32_t *table; int64_t table_stride;
    int32_t n_rows, n_seq, n_tokens, max_new;
    int32_t n_head, type;                  /* type: of q and dst */
    const float *sink;                     /* [n_head] or NULL */
    int32_t window, keep_first;
    float   scale, softcap;
    int32_t f16_products;
} b200_kv8_attn_args;
B200_API size_t b200_kv8_attn_workspace_bytes(const b200_kv8_attn_args *a);
B200_API int b200_op_kv8_attn(const b200_kv8_attn_args *a, void *workspace, size_t workspace_bytes, b200_stream_t stream);
/* The same with the limit of each of the kernel's own waits in clock cycles (b200_op_kv8_attn: about two seconds' worth; 0: it gives up at
 * once), where many new tokens run on tcgen05 (heads of up to 128).  When one runs out the call ends early: rows of dst are right, NaN or as they were, and b200_gemm_status() becomes 1. */
B200_API int b200_op_kv8_attn_wait(const b200_kv8_attn_args *a, void *workspace, size_t workspace_bytes, int64_t wait_cycles, b200_stream_t stream);

/* ---- pages: who holds what, on the device (all layers' pools go by one table) -----------------------------------------------------------------
 * refs[p]: how many table entries name page p; len[row]: tokens that the row holds; entries from ceil(len / page_size) on are -1.  A caller
 * begins with refs = 0, len = 0, table = -1 and then leaves all three to these calls (it may take entries out of a table for pages that no window
 * reaches any more: refs goes down by one, the entry becomes -1).  `rows`, `src`, `dst` name n rows, n <= B200_KV8_MAX_SEQ; rows outside [0,
 * n_rows) and a row named a second time in one call count as refused.  *refused (optional) is raised by the number of refused rows. */
typedef struct {
    int32_t *table; int64_t table_stride;
    int32_t *len, *refs;
    int32_t n_rows, n_pages, page_size, _pad;
} b200_kv8_map;

/* Rows keep their first keep[i] tokens (keep NULL: none), at most what they hold; pages behind are given back, refs 0 is free. */
B200_API int b200_op_kv8_cut(const b200_kv8_map *m, const int32_t *rows, const int32_t *keep, int32_t n, b200_stream_t stream);

/* Row dst[i], which holds nothing, becomes row src[i]: it names the same pages.  Nothing is copied until one of them grows.  Refused: a dst that
 * holds something or is named twice, and a src that is a dst of the same call. */
B200_API int b200_op_kv8_fork(const b200_kv8_map *m, const int32_t *src, const int32_t *dst, int32_t n, int32_t *refused, b200_stream_t stream);

/* Rows get room for n_new[i] >= 0 more tokens: new pages are those with refs 0, the lowest numbers first, in the order of the list; a last
 * page that is shared and not full is first replaced by a copy of its own (in all the caches) if n_new[i] > 0.  len grows by n_new[i].  A
 * row that does not fit its table, or for which the pages no longer reach (with those before it in the list, refused ones too), is
 * refused: it stays as it is.  seq_info (optional) [4][n] becomes the step over these rows: tokens in the order of the list, n_new[i] each (negative ones
 * count as 0 and are refused), rows that were refused with a count of 0 in their place; a row whose tokens would reach beyond the step's 2^31 - 1st is refused too. */
B200_API size_t b200_kv8_grow_workspace_bytes(int32_t n);
B200_API int b200_op_kv8_grow(const b200_kv8_map *m, const b200_kv8_cache *caches, int32_t n_caches, const int32_t *rows, const int32_t *n_new, int32_t n, int32_t *seq_info,
                              int32_t *refused, void *workspace, size_t workspace_bytes, b200_stream_t stream);

/* Pages with refs > 0 move to the front of the pool: with L of them, those numbered L and above go, in ascending order, to the free numbers below
 * L, in ascending order; tables, refs and the records of all caches follow.  *n_live (optional) = L. */
B200_API size_t b200_kv8_compact_workspace_bytes(int32_t n_pages);
B200_API int b200_op_kv8_compact(const b200_kv8_map *m, const b200_kv8_cache *caches, int32_t n_caches, int32_t *n_live, void *workspace, size_t workspace_bytes, b200_stream_t stream);

/* Record src[i] is copied to dst[i] in all caches, i < n (pairs outside the pool are left out; no dst is a src or a dst of another pair). */
B200_API int b200_op_kv8_copy_pages(const b200_kv8_cache *caches, int32_t n_caches, const int32_t *src, const int32_t *dst, int32_t n, b200_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* B200_KV8_H */
