/*
 * Attention of new tokens over a paged cache (tqt_kv_append_rope_gfx950.h): one decoded token of each
 * sequence, chunks of prompts, whole prompts, or all of them in one batch. No counterpart in the
 * reference library.
 *
 * Sequence b has the queries q_start[b] .. q_start[b + 1] - 1 of Q (rows of D and lse alike) and kv_len[b]
 * keys, its new tokens' own among them (they are appended first); its query i stands at position
 * kv_len[b] - q_len + i. Key j is on page block_table[b][j / page_size]. Query head h reads key head
 * h / (q_heads / kv_heads). A query sees key j when
 *   0 <= j < kv_len[b], and, causal: j <= position, and, window > 0: j > position - window,
 * and its page is one of the cache's: entries outside [0, num_pages) mark pages that are not kept, whose
 * keys nobody sees. With s_j = scale * (q . k_j) over the keys seen,
 *   D = sum_j exp(s_j) v_j / sum_j exp(s_j),   lse = log(sum_j exp(s_j))
 * and a row that sees no key (or only keys with s_j = -infinity) gets D = 0 and lse = -infinity. What lies
 * in the cache at keys past kv_len, or in pages not named, is not used, whatever bits it holds, and an
 * infinity or NaN at a key reaches only the rows that see this key.
 * Scores, sums and the softmax are held in f32; the probabilities are rounded once, to Q's type, for the matrix
 * product with the values. Int8 caches: the probability times the value's scale is rounded, to f16, relative to
 * the largest such term of the keys that the row sees (rows of zeros aside). Terms down to 2^-13 of it keep all
 * bits, those below 2^-24 may be lost; value scales below 2^-60 lose bits in the same way. Scales may have either
 * sign; one that is not finite makes the rows that see its key NaN.
 *
 * The function's name gives the type of Q and D, then the cache's: f16_f16, bf16_bf16, f16_qsi8dx,
 * bf16_qsi8dx (int8 with a scale for each token and head).
 *
 * Preconditions: q_heads a multiple of kv_heads; head_dim a multiple of 16 up to 256; rows of Q, D, k and
 * v on the 16-byte grid; scale times log2(e) finite; max_kv_len <= ld_table * page_size and below 2^30.
 * max_q_len and max_kv_len bound q_len and kv_len of every sequence: the launch and its workspace are sized by
 * them, so that lengths may change on the device between replays of a captured call. (A kv_len past max_kv_len
 * is taken as max_kv_len, queries past max_q_len of a sequence are left out. Bounds near the lengths make a call
 * faster.) q_start does not decrease, from 0 to at most q_tokens. workspace holds at least
 * tqt_get_workspace_size_attn_paged_gfx950 bytes on the 16-byte grid (it may be NULL for size 0), needs no
 * initial value, and is free again when the call has run. A row's sums do not depend on the order in which
 * workgroups run.
 * Conventions as in tqt_rope_gfx950.h.
 */
#ifndef TQT_ATTN_PAGED_GFX950_H
#define TQT_ATTN_PAGED_GFX950_H

#include "tqt_kv_append_rope_gfx950.h"

#ifdef __cplusplus
extern "C" {
#endif

struct tqt_attn_paged_params
{
    size_t batch;
    size_t q_tokens; /* rows of Q: q_start[batch] at most */
    size_t q_heads;
    size_t max_q_len;
    size_t max_kv_len;
    const void *Q;
    size_t q_token_stride;
    size_t q_head_stride;
    void *D;
    size_t d_token_stride;
    size_t d_head_stride;
    float *lse;                 /* [q_tokens][q_heads], or NULL */
    const int32_t *q_start;     /* [batch + 1] */
    const int32_t *kv_len;      /* [batch] */
    const int32_t *block_table; /* [batch][ld_table] */
    size_t ld_table;
    float scale;
    int32_t causal;
    size_t window; /* 0: none; needs causal */
    struct tqt_paged_kv kv;
    void *workspace;
    size_t workspace_size;
};

/* Depends on the sizes only (batch, q_tokens, q_heads, max_q_len, max_kv_len, window, kv's). */
size_t tqt_get_workspace_size_attn_paged_gfx950(const struct tqt_attn_paged_params *params);

const char *tqt_get_error_attn_paged_f16_f16_gfx950(const struct tqt_attn_paged_params *params);
const char *tqt_get_error_attn_paged_bf16_bf16_gfx950(const struct tqt_attn_paged_params *params);
const char *tqt_get_error_attn_paged_f16_qsi8dx_gfx950(const struct tqt_attn_paged_params *params);
const char *tqt_get_error_attn_paged_bf16_qsi8dx_gfx950(const struct tqt_attn_paged_params *params);

void tqt_run_attn_paged_f16_f16_gfx950(const struct tqt_attn_paged_params *params);
void tqt_run_attn_paged_bf16_bf16_gfx950(const struct tqt_attn_paged_params *params);
void tqt_run_attn_paged_f16_qsi8dx_gfx950(const struct tqt_attn_paged_params *params);
void tqt_run_attn_paged_bf16_qsi8dx_gfx950(const struct tqt_attn_paged_params *params);

void tqt_run_attn_paged_f16_f16_gfx950_async(const struct tqt_attn_paged_params *params, void *stream);
void tqt_run_attn_paged_bf16_bf16_gfx950_async(const struct tqt_attn_paged_params *params, void *stream);
void tqt_run_attn_paged_f16_qsi8dx_gfx950_async(const struct tqt_attn_paged_params *params,
                                                void *stream);
void tqt_run_attn_paged_bf16_qsi8dx_gfx950_async(const struct tqt_attn_paged_params *params,
                                                 void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
