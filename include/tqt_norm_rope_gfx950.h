/*
 * Norm of every head with its rotary positions in one pass: the step between a QKV product of this library
 * and attention in models that normalise their query and key heads, and its gradient. No counterpart in
 * the reference library.
 *
 * For a head x of d = head_dim elements
 *   r = 1 / sqrt(mean(x^2) + eps),   n_e = x_e r (weight_e + shift),   y = n turned as in tqt_rope_gfx950.h
 * (weight NULL: n = x r, whatever shift is). The mean runs over the whole head, elements past rotary_dim among
 * them. It and r are computed in 64 bits, so that no finite x overflows them; the products are in f32, each
 * rounded on its own; y is rounded once to Y's type, not between the norm and the rotation. A head with a NaN
 * is NaN; one with infinities is NaN there and in the elements that the rotation pairs with them, else 0.
 *
 * The gradient takes dY and gives, with u = dY turned back, f = weight + shift and m = x r,
 *   dX = r (f u - m mean(f u m)),   dweight = sum over tokens and heads of u m
 * (written, not added to; dweight NULL: not wanted). Its sums over a head are held in 64 bits, those over rows in
 * f32 within a workgroup's share of them and in 64 bits over the workgroups, always in the same order: a call
 * repeated gives the same bits. forward.rope.Y and the Y strides are not used. dX may be dY or X, with the
 * same strides; they may not overlap otherwise. A position outside [0, max_pos) makes NaN of the rotated
 * elements of Y and of dweight, and of all of the token's dX.
 *
 * weight is [head_dim] f32 on the device (with the heads' rows on the 16-byte grid, head_dim and rotary_dim
 * multiples of 16, and head_dim up to 1024 the fast calls, if it lies there too). Y may be X, as in
 * tqt_rope_gfx950.h, whose conventions hold here. The gradient needs tokens * heads below 2^31 and a workspace of
 * tqt_get_workspace_size_norm_rope_grad_gfx950 bytes on the 16-byte grid (it may be NULL for size 0), which
 * needs no initial value and is free again when the call has run.
 */
#ifndef TQT_NORM_ROPE_GFX950_H
#define TQT_NORM_ROPE_GFX950_H

#include "tqt_rope_gfx950.h"

#ifdef __cplusplus
extern "C" {
#endif

struct tqt_head_norm
{
    const float *weight; /* [head_dim], or NULL */
    float shift;         /* added to the weight: 1 for weights stored around 0 */
    float eps;           /* > 0 */
};

struct tqt_norm_rope_params
{
    struct tqt_rope_params rope;
    struct tqt_head_norm norm;
};

struct tqt_norm_rope_grad_params
{
    struct tqt_norm_rope_params forward;
    const void *dY;
    size_t dy_token_stride;
    size_t dy_head_stride;
    void *dX;
    size_t dx_token_stride;
    size_t dx_head_stride;
    float *dweight; /* [head_dim], or NULL */
    void *workspace;
    size_t workspace_size;
};

/* Depends on tokens, heads, head_dim and on whether dweight is NULL only. */
size_t tqt_get_workspace_size_norm_rope_grad_gfx950(const struct tqt_norm_rope_grad_params *params);

const char *tqt_get_error_norm_rope_f32_gfx950(const struct tqt_norm_rope_params *params);
const char *tqt_get_error_norm_rope_f16_gfx950(const struct tqt_norm_rope_params *params);
const char *tqt_get_error_norm_rope_bf16_gfx950(const struct tqt_norm_rope_params *params);
const char *tqt_get_error_norm_rope_grad_f32_gfx950(const struct tqt_norm_rope_grad_params *params);
const char *tqt_get_error_norm_rope_grad_f16_gfx950(const struct tqt_norm_rope_grad_params *params);
const char *tqt_get_error_norm_rope_grad_bf16_gfx950(const struct tqt_norm_rope_grad_params *params);

void tqt_run_norm_rope_f32_gfx950(const struct tqt_norm_rope_params *params);
void tqt_run_norm_rope_f16_gfx950(const struct tqt_norm_rope_params *params);
void tqt_run_norm_rope_bf16_gfx950(const struct tqt_norm_rope_params *params);
void tqt_run_norm_rope_f32_gfx950_async(const struct tqt_norm_rope_params *params, void *stream);
void tqt_run_norm_rope_f16_gfx950_async(const struct tqt_norm_rope_params *params, void *stream);
void tqt_run_norm_rope_bf16_gfx950_async(const struct tqt_norm_rope_params *params, void *stream);

void tqt_run_norm_rope_grad_f32_gfx950(const struct tqt_norm_rope_grad_params *params);
void tqt_run_norm_rope_grad_f16_gfx950(const struct tqt_norm_rope_grad_params *params);
void tqt_run_norm_rope_grad_bf16_gfx950(const struct tqt_norm_rope_grad_params *params);
void tqt_run_norm_rope_grad_f32_gfx950_async(const struct tqt_norm_rope_grad_params *params, void *stream);
void tqt_run_norm_rope_grad_f16_gfx950_async(const struct tqt_norm_rope_grad_params *params, void *stream);
void tqt_run_norm_rope_grad_bf16_gfx950_async(const struct tqt_norm_rope_grad_params *params, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
