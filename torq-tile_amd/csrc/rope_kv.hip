// Rotary positions, their tables, and the append of keys and values to a paged cache on gfx950: the entry points.
#include "rope_rows.hpp"

namespace tqt {
namespace {

// cos and sin of position * frequency in f64: one thread per pair of a position.
__global__ __launch_bounds__(kRopeThreads) void rope_table_kernel(float *table, long long pairs, int half,
                                                                  double base, double factor, int scaling,
                                                                  double orig, double low_turns,
                                                                  double high_turns, double amplitude)
{
    const long long at = static_cast<long long>(blockIdx.x) * kRopeThreads + threadIdx.x;
    if (at >= pairs) {
        return;
    }
    const long long pos = at / half;
    const int i = static_cast<int>(at - pos * half);
    const double r = 2.0 * half, two_pi = 6.283185307179586;
    double f = pow(base, -2.0 * i / r);
    if (scaling == TQT_ROPE_LINEAR) {
        f /= factor;
    } else if (scaling == TQT_ROPE_BASE) {
        f = r > 2.0 ? pow(base * pow(factor, r / (r - 2.0)), -2.0 * i / r) : f;
    } else if (scaling == TQT_ROPE_RAMP) {
        // the pair that makes n turns over the original length: n 2 pi = orig base^(-2 i / r)
        const double lo = fmax(floor(r * log(orig / (high_turns * two_pi)) / (2.0 * log(base))), 0.0);
        const double hi = fmin(ceil(r * log(orig / (low_turns * two_pi)) / (2.0 * log(base))), r - 1.0);
        const double ramp = fmin(fmax((i - lo) / fmax(hi - lo, 0.001), 0.0), 1.0);
        f = f / factor * ramp + f * (1.0 - ramp);
    } else if (scaling == TQT_ROPE_TURNS) {
        const double smooth =
            fmin(fmax((orig * f / two_pi - low_turns) / (high_turns - low_turns), 0.0), 1.0);
        f = f / factor * (1.0 - smooth) + f * smooth;
    }
    double s, c;
    sincos(static_cast<double>(pos) * f, &s, &c);
    table[pos * 2 * half + i] = static_cast<float>(c * amplitude);
    table[pos * 2 * half + half + i] = static_cast<float>(s * amplitude);
}

template <typename T>
bool check_run_rope(const tqt_rope_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = rope_error(p);
    TQT_REQUIRE(error == nullptr, error);
    return run_rope<T, false>(p, nullptr, stream, where);
}

template <typename SRC, typename DST, typename CACHE>
bool check_run_append(const tqt_kv_append_rope_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = append_error(p, sizeof(CACHE), std::is_same<CACHE, int8_t>::value);
    TQT_REQUIRE(error == nullptr, error);
    return run_append<SRC, DST, CACHE, false>(p, nullptr, nullptr, stream, where);
}

// One thread per pair of a position.
long long table_blocks(const tqt_rope_table_params *p)
{
    const long long pairs = static_cast<long long>(p->max_pos) * static_cast<long long>(p->rotary_dim / 2);
    return (pairs + kRopeThreads - 1) / kRopeThreads;
}

const char *table_error(const tqt_rope_table_params *p)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    if (p->max_pos >= (1u << 31) || p->rotary_dim % 2 != 0 || p->rotary_dim >= (1u << 20)) {
        return "max_pos too large, or rotary_dim odd or too large";
    }
    if (p->max_pos == 0 || p->rotary_dim == 0) {
        return nullptr;
    }
    if (p->table == nullptr) {
        return "table == NULL";
    }
    if (!(p->base > 1.0) || !std::isfinite(p->base)) {
        return "base is not a finite number > 1";
    }
    if (p->scaling < TQT_ROPE_PLAIN || p->scaling > TQT_ROPE_TURNS) {
        return "unknown scaling";
    }
    if (p->scaling != TQT_ROPE_PLAIN && (!(p->factor > 0.0) || !std::isfinite(p->factor))) {
        return "factor is not a finite number > 0";
    }
    if ((p->scaling == TQT_ROPE_RAMP || p->scaling == TQT_ROPE_TURNS) &&
        (!(p->original_max_pos > 0.0) || !(p->low_turns > 0.0) || !(p->high_turns > p->low_turns))) {
        return "original_max_pos, low_turns and high_turns: 0 < low_turns < high_turns are needed";
    }
    if (table_blocks(p) * kRopeThreads >= 0x100000000ll) {
        return "max_pos * rotary_dim / 2 is too large for one launch";
    }
    return nullptr;
}

bool run_table(const tqt_rope_table_params *p, hipStream_t stream)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = table_error(p);
    TQT_REQUIRE(error == nullptr, error);
    if (p->max_pos == 0 || p->rotary_dim == 0) {
        return false;
    }
    double amplitude = p->amplitude;
    if (amplitude == 0.0) {
        amplitude = p->scaling == TQT_ROPE_RAMP && p->factor > 1.0 ? 0.1 * std::log(p->factor) + 1.0 : 1.0;
    }
    const int half = static_cast<int>(p->rotary_dim / 2);
    hipLaunchKernelGGL(rope_table_kernel, dim3(static_cast<unsigned>(table_blocks(p))), dim3(kRopeThreads), 0,
                       stream, p->table, static_cast<long long>(p->max_pos) * half, half, p->base, p->factor,
                       p->scaling, p->original_max_pos, p->low_turns, p->high_turns, amplitude);
    check_launch("tqt_run_rope_table_f32_gfx950");
    return true;
}

}  // namespace
}  // namespace tqt

using namespace tqt;

extern "C" {

#define TQT_ROPE_ENTRIES(NAME, T)                                                                     \
    const char *tqt_get_error_rope_##NAME##_gfx950(const struct tqt_rope_params *params)              \
    {                                                                                                 \
        return rope_error(params);                                                                    \
    }                                                                                                 \
    void tqt_run_rope_##NAME##_gfx950_async(const struct tqt_rope_params *params, void *stream)       \
    {                                                                                                 \
        check_run_rope<T>(params, as_stream(stream), "tqt_run_rope_" #NAME "_gfx950");                      \
    }                                                                                                 \
    void tqt_run_rope_##NAME##_gfx950(const struct tqt_rope_params *params)                           \
    {                                                                                                 \
        if (check_run_rope<T>(params, nullptr, "tqt_run_rope_" #NAME "_gfx950")) {                          \
            finish_sync(nullptr, "tqt_run_rope_" #NAME "_gfx950");                                    \
        }                                                                                             \
    }

TQT_ROPE_ENTRIES(f32, float)
TQT_ROPE_ENTRIES(f16, _Float16)
TQT_ROPE_ENTRIES(bf16, __bf16)

#define TQT_APPEND_ENTRIES(NAME, SRC, DST, CACHE)                                                     \
    const char *tqt_get_error_kv_append_rope_##NAME##_gfx950(                                         \
        const struct tqt_kv_append_rope_params *params)                                               \
    {                                                                                                 \
        return append_error(params, sizeof(CACHE), std::is_same<CACHE, int8_t>::value);               \
    }                                                                                                 \
    void tqt_run_kv_append_rope_##NAME##_gfx950_async(                                                \
        const struct tqt_kv_append_rope_params *params, void *stream)                                 \
    {                                                                                                 \
        check_run_append<SRC, DST, CACHE>(params, as_stream(stream),                                        \
                                    "tqt_run_kv_append_rope_" #NAME "_gfx950");                       \
    }                                                                                                 \
    void tqt_run_kv_append_rope_##NAME##_gfx950(const struct tqt_kv_append_rope_params *params)       \
    {                                                                                                 \
        if (check_run_append<SRC, DST, CACHE>(params, nullptr, "tqt_run_kv_append_rope_" #NAME "_gfx950")) { \
            finish_sync(nullptr, "tqt_run_kv_append_rope_" #NAME "_gfx950");                          \
        }                                                                                             \
    }

TQT_APPEND_ENTRIES(f16_f16, _Float16, _Float16, _Float16)
TQT_APPEND_ENTRIES(bf16_bf16, __bf16, __bf16, __bf16)
TQT_APPEND_ENTRIES(f16_f32, float, _Float16, _Float16)
TQT_APPEND_ENTRIES(bf16_f32, float, __bf16, __bf16)
TQT_APPEND_ENTRIES(qsi8dx_f16, _Float16, _Float16, int8_t)
TQT_APPEND_ENTRIES(qsi8dx_bf16, __bf16, __bf16, int8_t)

const char *tqt_get_error_rope_table_f32_gfx950(const struct tqt_rope_table_params *params)
{
    return table_error(params);
}

void tqt_run_rope_table_f32_gfx950_async(const struct tqt_rope_table_params *params, void *stream)
{
    run_table(params, as_stream(stream));
}

void tqt_run_rope_table_f32_gfx950(const struct tqt_rope_table_params *params)
{
    if (run_table(params, nullptr)) {
        finish_sync(nullptr, "tqt_run_rope_table_f32_gfx950");
    }
}

}  // extern "C"
