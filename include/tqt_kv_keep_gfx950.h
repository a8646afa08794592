/*
 * The rows of accepted tokens in a paged cache: after a tree of drafted tokens has been verified, the keys and
 * values of the path that was accepted move together behind the context, in one layer's cache or in all layers'
 * at once. No counterpart in the reference library.
 *
 * Sequence b has kv_len[b] tokens in the cache, the last q_len = q_start[b + 1] - q_start[b] of them drafted, and
 * its context before them, base = kv_len - q_len. keep[b][0 .. keep_len[b]) are the numbers of the accepted ones
 * among the drafted, ascending: token base + keep[b][j] becomes token base + j, and kv_len_out[b] = base + the
 * number of them. The list ends before the first entry that is not above the one before it or not below
 * q_len (a negative one is neither), and after max_keep entries. Rows past the kept ones are left as they were, to be
 * overwritten by the next step's. Rows whose page (of either place) is outside [0, num_pages) are not moved. Rows are
 * copied bit for bit, int8 rows with their scales.
 *
 * Layer l's cache is kv with its k and v at l * layer_stride elements, its scales at l * scale_layer_stride; layers
 * share the block table. kv_len_out may be NULL, and may not overlap kv_len: the layers of a model may be called
 * one by one, and then the last call writes it. A kv_len above ld_table * page_size counts as that; a sequence with
 * fewer tokens in the cache than drafted ones keeps none, and its kv_len_out is 0. Two sequences may not share a page
 * that holds drafted tokens.
 *
 * A step that may refuse sequences (tqt_run_paged_plan_* had no pages for one) gives positions, the plan's for rows 0 to
 * tokens: a sequence whose first drafted row's position is not below its kv_len, or whose rows begin at tokens or
 * later, was refused, its kv_len does not count its drafted tokens, and so nothing moves and kv_len_out is kv_len. slots, which
 * the rows were appended with, may stand for them (they are not read with positions): a sequence was refused whose
 * drafted rows have negative ones although their tokens' pages are kept. They cannot tell so where none of the last
 * q_len tokens' pages is one of the cache, and such a sequence counts as served.
 * The function's name gives the cache's type. Conventions as in tqt_rope_gfx950.h, of the cache as in
 * tqt_kv_append_rope_gfx950.h.
 */
#ifndef TQT_KV_KEEP_GFX950_H
#define TQT_KV_KEEP_GFX950_H

#include "tqt_kv_append_rope_gfx950.h"

#ifdef __cplusplus
extern "C" {
#endif

struct tqt_kv_keep_params
{
    size_t batch;
    size_t max_keep;
    const int32_t *q_start; /* [batch + 1] */
    const int32_t *kv_len;  /* [batch] */
    int32_t *kv_len_out;    /* [batch], or NULL */
    const int32_t *keep;    /* [batch][ld_keep], max_keep of them read at most */
    size_t ld_keep;
    const int32_t *keep_len;    /* [batch] */
    const int32_t *block_table; /* [batch][ld_table] */
    size_t ld_table;
    size_t layers;
    size_t layer_stride;       /* of k and v, in elements */
    size_t scale_layer_stride; /* int8 caches: of scale_k and scale_v */
    struct tqt_paged_kv kv;
    const int64_t *slots; /* [tokens], or NULL */
    size_t tokens;        /* rows that q_start counts in; not read without slots and positions */
    const int32_t *positions; /* [tokens], or NULL; without slots too every sequence was served */
};

const char *tqt_get_error_kv_keep_f16_gfx950(const struct tqt_kv_keep_params *params);
const char *tqt_get_error_kv_keep_bf16_gfx950(const struct tqt_kv_keep_params *params);
const char *tqt_get_error_kv_keep_qsi8dx_gfx950(const struct tqt_kv_keep_params *params);

void tqt_run_kv_keep_f16_gfx950(const struct tqt_kv_keep_params *params);
void tqt_run_kv_keep_bf16_gfx950(const struct tqt_kv_keep_params *params);
void tqt_run_kv_keep_qsi8dx_gfx950(const struct tqt_kv_keep_params *params);
void tqt_run_kv_keep_f16_gfx950_async(const struct tqt_kv_keep_params *params, void *stream);
void tqt_run_kv_keep_bf16_gfx950_async(const struct tqt_kv_keep_params *params, void *stream);
void tqt_run_kv_keep_qsi8dx_gfx950_async(const struct tqt_kv_keep_params *params, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
