/*
 * Rotary positions: pairs of elements of every attention head turned by an angle that grows with the
 * token's position, the step between a QKV product of this library and attention. No counterpart in
 * the reference library.
 *
 * With r = rotary_dim and i < r / 2, the pair (x1, x2) of a head at position p becomes
 *   y1 = x1 * c - x2 * s,   y2 = x2 * c + x1 * s,   c = table[p][i],  s = table[p][r / 2 + i]
 * where the pair is (i, i + r / 2) (interleaved = 0) or (2 i, 2 i + 1) (interleaved = 1); elements from
 * r on are copied. inverse = 1 turns back (-s in the place of s), which is also the gradient of x for
 * the gradient of y. The arithmetic is in f32 with every product and sum rounded on its own, and the
 * result is rounded once to Y's type.
 *
 * X, Y, positions and the table are device pointers; strides count elements. X and Y may be the same
 * tensor (with the same strides); they may not overlap otherwise. Any head_dim, strides and alignment are
 * taken; rows on the 16-byte grid with head_dim and rotary_dim multiples of 16 are the fast ones. A
 * position outside [0, max_pos) makes the rotated elements of its token NaN.
 *
 * The run functions follow the library's conventions: NULL params return at once, a violated
 * precondition or a HIP error prints a message and aborts, the plain form returns with the output
 * written and the _async form enqueues on `stream` (a hipStream_t, NULL = the default stream).
 * tqt_get_error_* checks the params without running: NULL if a run would take them, else the reason.
 */
#ifndef TQT_ROPE_GFX950_H
#define TQT_ROPE_GFX950_H

#include "tqt_gfx950_common.h"

#ifdef __cplusplus
extern "C" {
#endif

/* How a head's elements pair up and by what they turn. rotary_dim = 0: nothing turns (the table may
 * then be NULL). */
struct tqt_rope_map
{
    const float *table; /* [max_pos][rotary_dim]: rotary_dim / 2 cosines, then as many sines */
    size_t max_pos;
    size_t rotary_dim; /* even, <= head_dim */
    int32_t interleaved;
    int32_t inverse;
};

struct tqt_rope_params
{
    size_t tokens;
    size_t heads;
    size_t head_dim;
    const void *X;
    size_t x_token_stride;
    size_t x_head_stride;
    void *Y;
    size_t y_token_stride;
    size_t y_head_stride;
    const int32_t *positions; /* [tokens] */
    struct tqt_rope_map map;
};

/* Frequencies of the table, f_i = base^(-2 i / rotary_dim), for contexts longer than the model's own:
 *   TQT_ROPE_PLAIN   f_i
 *   TQT_ROPE_LINEAR  f_i / factor (interpolated positions)
 *   TQT_ROPE_BASE    the base times factor^(r / (r - 2)): the slowest pair ends at f / factor, the
 *                    fastest stays
 *   TQT_ROPE_RAMP    f_i where the pair makes more than high_turns turns over original_max_pos tokens,
 *                    f_i / factor where fewer than low_turns, and in between a blend linear in i (from
 *                    the floor of the one index to the ceiling of the other); the table's values are
 *                    times 0.1 ln(factor) + 1 (times 1 for a factor up to 1) unless amplitude says
 *                    otherwise
 *   TQT_ROPE_TURNS   the same two ends, with a blend linear in the number of turns
 * amplitude multiplies cosines and sines; 0 stands for the default (1, or TQT_ROPE_RAMP's). */
#define TQT_ROPE_PLAIN 0
#define TQT_ROPE_LINEAR 1
#define TQT_ROPE_BASE 2
#define TQT_ROPE_RAMP 3
#define TQT_ROPE_TURNS 4

struct tqt_rope_table_params
{
    float *table; /* [max_pos][rotary_dim], written */
    size_t max_pos;
    size_t rotary_dim;
    int32_t scaling;
    double base;
    double factor;
    double original_max_pos;
    double low_turns;
    double high_turns;
    double amplitude;
};

const char *tqt_get_error_rope_f32_gfx950(const struct tqt_rope_params *params);
const char *tqt_get_error_rope_f16_gfx950(const struct tqt_rope_params *params);
const char *tqt_get_error_rope_bf16_gfx950(const struct tqt_rope_params *params);
const char *tqt_get_error_rope_table_f32_gfx950(const struct tqt_rope_table_params *params);

void tqt_run_rope_f32_gfx950(const struct tqt_rope_params *params);
void tqt_run_rope_f16_gfx950(const struct tqt_rope_params *params);
void tqt_run_rope_bf16_gfx950(const struct tqt_rope_params *params);
void tqt_run_rope_f32_gfx950_async(const struct tqt_rope_params *params, void *stream);
void tqt_run_rope_f16_gfx950_async(const struct tqt_rope_params *params, void *stream);
void tqt_run_rope_bf16_gfx950_async(const struct tqt_rope_params *params, void *stream);

/* The table of a model's positions, computed in f64 and rounded once. */
void tqt_run_rope_table_f32_gfx950(const struct tqt_rope_table_params *params);
void tqt_run_rope_table_f32_gfx950_async(const struct tqt_rope_table_params *params, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
