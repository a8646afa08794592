/*
 * Attention of trees of drafted tokens over a paged cache: tqt_run_attn_paged_* with a mask among the new
 * tokens in the place of their order. No counterpart in the reference library.
 *
 * Sequence b's new tokens are the last q_len = q_start[b + 1] - q_start[b] of its kv_len[b] keys (they are appended
 * first), its context the base = kv_len[b] - q_len keys before them. Its query i, row q_start[b] + i of Q, sees
 * key base + t of the new tokens when bit t % 32 of word t / 32 of that row of mask is set (its own key among
 * them only if its own bit is), for t < q_len, and key j < base of the context always, or, with window > 0, when
 * j > base + n - 1 - window, n the number of its mask's bits below q_len: its position's window, where the mask names
 * a token's ancestors and itself. The window does not hide new tokens. Bits from 32 * ld_mask on count as 0.
 * Everything else, an empty row's result, pages that are not kept, values that are no numbers, types, rounding,
 * bounds and preconditions, is as in tqt_attn_paged_gfx950.h; attn.causal has to be 1 (the mask stands for the
 * order), and ld_mask words hold max_q_len bits. tqt_run_paged_plan_* makes such masks from parents.
 */
#ifndef TQT_ATTN_TREE_GFX950_H
#define TQT_ATTN_TREE_GFX950_H

#include "tqt_attn_paged_gfx950.h"

#ifdef __cplusplus
extern "C" {
#endif

struct tqt_attn_tree_params
{
    struct tqt_attn_paged_params attn;
    const uint32_t *mask; /* [q_tokens][ld_mask] */
    size_t ld_mask;
};

/* Depends on the sizes only, as that of tqt_run_attn_paged_*. */
size_t tqt_get_workspace_size_attn_tree_gfx950(const struct tqt_attn_tree_params *params);

const char *tqt_get_error_attn_tree_f16_f16_gfx950(const struct tqt_attn_tree_params *params);
const char *tqt_get_error_attn_tree_bf16_bf16_gfx950(const struct tqt_attn_tree_params *params);
const char *tqt_get_error_attn_tree_f16_qsi8dx_gfx950(const struct tqt_attn_tree_params *params);
const char *tqt_get_error_attn_tree_bf16_qsi8dx_gfx950(const struct tqt_attn_tree_params *params);

void tqt_run_attn_tree_f16_f16_gfx950(const struct tqt_attn_tree_params *params);
void tqt_run_attn_tree_bf16_bf16_gfx950(const struct tqt_attn_tree_params *params);
void tqt_run_attn_tree_f16_qsi8dx_gfx950(const struct tqt_attn_tree_params *params);
void tqt_run_attn_tree_bf16_qsi8dx_gfx950(const struct tqt_attn_tree_params *params);

void tqt_run_attn_tree_f16_f16_gfx950_async(const struct tqt_attn_tree_params *params, void *stream);
void tqt_run_attn_tree_bf16_bf16_gfx950_async(const struct tqt_attn_tree_params *params, void *stream);
void tqt_run_attn_tree_f16_qsi8dx_gfx950_async(const struct tqt_attn_tree_params *params, void *stream);
void tqt_run_attn_tree_bf16_qsi8dx_gfx950_async(const struct tqt_attn_tree_params *params, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
