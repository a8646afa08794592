/*
 * Appending keys and values to a paged cache, with the rotary positions of the keys (and, if given, of
 * the queries of the same tokens) applied on the way: one launch between a QKV product of this library
 * and tqt_run_attn_paged_*. No counterpart in the reference library.
 *
 * The cache is two tensors k and v of num_pages pages with page_size tokens each: element e of head h
 * of token o of page p is at p * page_stride + o * token_stride + h * head_stride + e (elements), the
 * same for both, so pages may hold [token][head][element] or [head][token][element]. Token t goes to
 * slots[t] = p * page_size + o. A slot outside the cache (a negative one marks padding) is not written;
 * two tokens of one call may not share a slot. The rotation is that of tqt_rope_gfx950.h; values are
 * copied.
 *
 * The function's name gives the cache's type, then the type of K, V and Q:
 *   f16_f16, bf16_bf16      the same types; Q_out has them too
 *   f16_f32, bf16_f32       results of the f32 GEMMs, rounded once; Q_out has the cache's type
 *   qsi8dx_f16, qsi8dx_bf16 an int8 cache, symmetric with one f32 scale for each token and head in
 *                           scale_k, scale_v [num_pages][kv_heads][page_size]: amax = max |x| of the
 *                           (rotated, f32) row, scale = amax * f32(1 / 127) (1 for a row of zeros),
 *                           q = clamp(nearbyint(x / scale), -127, 127). A row with a NaN or an infinity
 *                           gets a NaN for its scale, so it reads back as NaN. Q_out has Q's type.
 *
 * head_dim is a multiple of 16 up to 256; k, v and their strides keep rows on the 16-byte grid; K, V
 * and Q take any strides and alignment (rows on the 16-byte grid with rotary_dim a multiple of 16 are
 * the fast ones). Q and Q_out may be the same tensor (of one type, with the same strides). Pointers are
 * device pointers; conventions as in tqt_rope_gfx950.h.
 */
#ifndef TQT_KV_APPEND_ROPE_GFX950_H
#define TQT_KV_APPEND_ROPE_GFX950_H

#include "tqt_rope_gfx950.h"

#ifdef __cplusplus
extern "C" {
#endif

struct tqt_paged_kv
{
    void *k;
    void *v;
    float *scale_k; /* int8 caches, else NULL: [num_pages][kv_heads][page_size] */
    float *scale_v;
    size_t num_pages;
    size_t page_size;
    size_t kv_heads;
    size_t head_dim;
    size_t page_stride;
    size_t token_stride;
    size_t head_stride;
};

struct tqt_kv_append_rope_params
{
    size_t tokens;
    const void *K;
    size_t k_token_stride;
    size_t k_head_stride;
    const void *V;
    size_t v_token_stride;
    size_t v_head_stride;
    size_t q_heads; /* 0: no queries */
    const void *Q;
    size_t q_token_stride;
    size_t q_head_stride;
    void *Q_out;
    size_t qo_token_stride;
    size_t qo_head_stride;
    const int32_t *positions; /* [tokens], may be NULL when map.rotary_dim is 0 */
    const int64_t *slots;     /* [tokens] */
    struct tqt_rope_map map;
    struct tqt_paged_kv kv;
};

const char *tqt_get_error_kv_append_rope_f16_f16_gfx950(const struct tqt_kv_append_rope_params *params);
const char *tqt_get_error_kv_append_rope_bf16_bf16_gfx950(const struct tqt_kv_append_rope_params *params);
const char *tqt_get_error_kv_append_rope_f16_f32_gfx950(const struct tqt_kv_append_rope_params *params);
const char *tqt_get_error_kv_append_rope_bf16_f32_gfx950(const struct tqt_kv_append_rope_params *params);
const char *tqt_get_error_kv_append_rope_qsi8dx_f16_gfx950(const struct tqt_kv_append_rope_params *params);
const char *tqt_get_error_kv_append_rope_qsi8dx_bf16_gfx950(const struct tqt_kv_append_rope_params *params);

void tqt_run_kv_append_rope_f16_f16_gfx950(const struct tqt_kv_append_rope_params *params);
void tqt_run_kv_append_rope_bf16_bf16_gfx950(const struct tqt_kv_append_rope_params *params);
void tqt_run_kv_append_rope_f16_f32_gfx950(const struct tqt_kv_append_rope_params *params);
void tqt_run_kv_append_rope_bf16_f32_gfx950(const struct tqt_kv_append_rope_params *params);
void tqt_run_kv_append_rope_qsi8dx_f16_gfx950(const struct tqt_kv_append_rope_params *params);
void tqt_run_kv_append_rope_qsi8dx_bf16_gfx950(const struct tqt_kv_append_rope_params *params);

void tqt_run_kv_append_rope_f16_f16_gfx950_async(
    const struct tqt_kv_append_rope_params *params, void *stream);
void tqt_run_kv_append_rope_bf16_bf16_gfx950_async(
    const struct tqt_kv_append_rope_params *params, void *stream);
void tqt_run_kv_append_rope_f16_f32_gfx950_async(
    const struct tqt_kv_append_rope_params *params, void *stream);
void tqt_run_kv_append_rope_bf16_f32_gfx950_async(
    const struct tqt_kv_append_rope_params *params, void *stream);
void tqt_run_kv_append_rope_qsi8dx_f16_gfx950_async(
    const struct tqt_kv_append_rope_params *params, void *stream);
void tqt_run_kv_append_rope_qsi8dx_bf16_gfx950_async(
    const struct tqt_kv_append_rope_params *params, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
