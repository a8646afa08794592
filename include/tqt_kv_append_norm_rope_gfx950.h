/*
 * The append of keys and values to a paged cache (tqt_kv_append_rope_gfx950.h) with the heads of K and Q
 * normalised before they are turned (tqt_norm_rope_gfx950.h): one launch between a QKV product of this library
 * and attention in models that normalise their query and key heads. No counterpart in the reference library.
 *
 * append says what tqt_run_kv_append_rope_* would do; here every head of Q goes through q_norm and every head
 * of K through k_norm first, in f32 from the source's values, rounded only on the way into Q_out and the
 * cache (an int8 cache's scale is that of the normalised and turned row). Values are copied. Types, layouts and
 * conventions as there; weights are [head_dim] f32 on the device, on the 16-byte grid for the fast calls.
 */
#ifndef TQT_KV_APPEND_NORM_ROPE_GFX950_H
#define TQT_KV_APPEND_NORM_ROPE_GFX950_H

#include "tqt_kv_append_rope_gfx950.h"
#include "tqt_norm_rope_gfx950.h"

#ifdef __cplusplus
extern "C" {
#endif

struct tqt_kv_append_norm_rope_params
{
    struct tqt_kv_append_rope_params append;
    struct tqt_head_norm q_norm; /* not read where append.q_heads is 0 */
    struct tqt_head_norm k_norm;
};

const char *tqt_get_error_kv_append_norm_rope_f16_f16_gfx950(
    const struct tqt_kv_append_norm_rope_params *params);
const char *tqt_get_error_kv_append_norm_rope_bf16_bf16_gfx950(
    const struct tqt_kv_append_norm_rope_params *params);
const char *tqt_get_error_kv_append_norm_rope_f16_f32_gfx950(
    const struct tqt_kv_append_norm_rope_params *params);
const char *tqt_get_error_kv_append_norm_rope_bf16_f32_gfx950(
    const struct tqt_kv_append_norm_rope_params *params);
const char *tqt_get_error_kv_append_norm_rope_qsi8dx_f16_gfx950(
    const struct tqt_kv_append_norm_rope_params *params);
const char *tqt_get_error_kv_append_norm_rope_qsi8dx_bf16_gfx950(
    const struct tqt_kv_append_norm_rope_params *params);

void tqt_run_kv_append_norm_rope_f16_f16_gfx950(const struct tqt_kv_append_norm_rope_params *params);
void tqt_run_kv_append_norm_rope_bf16_bf16_gfx950(const struct tqt_kv_append_norm_rope_params *params);
void tqt_run_kv_append_norm_rope_f16_f32_gfx950(const struct tqt_kv_append_norm_rope_params *params);
void tqt_run_kv_append_norm_rope_bf16_f32_gfx950(const struct tqt_kv_append_norm_rope_params *params);
void tqt_run_kv_append_norm_rope_qsi8dx_f16_gfx950(const struct tqt_kv_append_norm_rope_params *params);
void tqt_run_kv_append_norm_rope_qsi8dx_bf16_gfx950(const struct tqt_kv_append_norm_rope_params *params);

void tqt_run_kv_append_norm_rope_f16_f16_gfx950_async(
    const struct tqt_kv_append_norm_rope_params *params, void *stream);
void tqt_run_kv_append_norm_rope_bf16_bf16_gfx950_async(
    const struct tqt_kv_append_norm_rope_params *params, void *stream);
void tqt_run_kv_append_norm_rope_f16_f32_gfx950_async(
    const struct tqt_kv_append_norm_rope_params *params, void *stream);
void tqt_run_kv_append_norm_rope_bf16_f32_gfx950_async(
    const struct tqt_kv_append_norm_rope_params *params, void *stream);
void tqt_run_kv_append_norm_rope_qsi8dx_f16_gfx950_async(
    const struct tqt_kv_append_norm_rope_params *params, void *stream);
void tqt_run_kv_append_norm_rope_qsi8dx_bf16_gfx950_async(
    const struct tqt_kv_append_norm_rope_params *params, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
