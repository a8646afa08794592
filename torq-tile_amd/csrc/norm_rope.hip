// The norm of heads with their rotation in the same pass on gfx950: alone, its gradient, and on the way into a
// paged cache. The forward kernels are those of rope_rows.hpp.
//
// Gradient: with u = dy turned back, f = weight + shift, m = x r,
//   dx = r (f u - m mean(f u m)),   dweight = sum over heads of u m.
// Bound by memory: x and dy are read once, dx is written once. The two sums of a head, x^2 and f u x, meet in one
// butterfly over its threads. A workgroup goes over every so many-th head, so that a thread keeps its 16 elements
// and their share of dweight stays in its registers; the workgroups' shares are joined in order by a second launch.
// 4099 tokens of 32 bf16 heads of 128 (101 MB) take 22.8-23.9 us, 4.2-4.4 TB/s, and 3 of join; loads a step ahead of
// their use gained 0.6 and cost 2.5 with f32 rows (registers), 512, 768 or 2048 workgroups took 1-4 more. Heads off the
// 16-element grid (a rotary_dim that is no multiple of 16 too) take a wave each, with loads of one element a lane: 2000
// tokens of 32 f32 heads of 80, 40 turned, 110 us forward and back.
#include "rope_rows.hpp"

namespace tqt {
namespace {

struct NormGradArgs
{
    const void *x, *dy;
    void *dx;
    float *part;  // [workgroups (waves)][head_dim]: shares of dweight, or nullptr
    long long x_ts, x_hs, dy_ts, dy_hs, dx_ts, dx_hs;
    const int32_t *positions;
    const float *table;
    const float *weight;
    float shift, eps;
    int max_pos, rotary_dim, interleaved;
    float sign;
    int head_dim;
    FastDiv heads;
    uint32_t rows;  // heads of all tokens
    int units;      // threads of a head, a power of two
};

// What one head's sums make of it.
struct NormGradHead
{
    float r;     // 1 / sqrt(mean(x^2) + eps)
    float mean;  // of f u m
};

__device__ __forceinline__ NormGradHead norm_grad_head(double squares, double products, const NormGradArgs &a)
{
    const double r = 1.0 / sqrt(squares / a.head_dim + a.eps);
    return {static_cast<float>(r), static_cast<float>(products * r / a.head_dim)};
}

// Turns the 8 pairs of two pieces.
__device__ __forceinline__ void turn8(bool interleaved, f32x8 c, f32x8 s, f32x8 &xa, f32x8 &xb)
{
    const f32x8 p = xa, q = xb;
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            xa[2 * i] = p[2 * i] * c[i] - p[2 * i + 1] * s[i];
            xa[2 * i + 1] = p[2 * i + 1] * c[i] + p[2 * i] * s[i];
            xb[2 * i] = q[2 * i] * c[i + 4] - q[2 * i + 1] * s[i + 4];
            xb[2 * i + 1] = q[2 * i + 1] * c[i + 4] + q[2 * i] * s[i + 4];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            xa[i] = p[i] * c[i] - q[i] * s[i];
            xb[i] = q[i] * c[i] + p[i] * s[i];
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kRopeThreads) void norm_grad_rows_kernel(NormGradArgs a)
{
    typedef typename Vec8<T>::type vec8;
    __shared__ float s_dw[16 * kRopeThreads];
    const int tid = threadIdx.x, unit = tid & (a.units - 1);
    const int heads_at_once = kRopeThreads / a.units, at = tid / a.units;
    const int r = a.rotary_dim, half = r >> 1;
    const bool turned = 16 * unit < r, on = 16 * unit < a.head_dim;
    int ea = 16 * unit, eb = ea + 8;
    if (turned && !a.interleaved) {
        ea = 8 * unit;
        eb = half + ea;
    }
    f32x8 fa = 1.0f, fb = 1.0f;
    if (on && a.weight != nullptr) {
        fa = *reinterpret_cast<const f32x8 *>(a.weight + ea) + a.shift;
        fb = *reinterpret_cast<const f32x8 *>(a.weight + eb) + a.shift;
    }
    f32x8 wa = 0.0f, wb = 0.0f;
    for (uint32_t row0 = blockIdx.x * heads_at_once; row0 < a.rows; row0 += gridDim.x * heads_at_once) {
        const bool live = on && row0 + at < a.rows;
        uint32_t head;
        const int token = static_cast<int>(fast_div(live ? row0 + at : 0u, a.heads, head));
        f32x8 xa = 0.0f, xb = 0.0f, ua = 0.0f, ub = 0.0f;
        if (live) {
            const T *x = static_cast<const T *>(a.x) + token * a.x_ts + head * a.x_hs;
            const T *dy = static_cast<const T *>(a.dy) + token * a.dy_ts + head * a.dy_hs;
            xa = __builtin_convertvector(*reinterpret_cast<const vec8 *>(x + ea), f32x8);
            xb = __builtin_convertvector(*reinterpret_cast<const vec8 *>(x + eb), f32x8);
            ua = __builtin_convertvector(*reinterpret_cast<const vec8 *>(dy + ea), f32x8);
            ub = __builtin_convertvector(*reinterpret_cast<const vec8 *>(dy + eb), f32x8);
            if (turned) {
                const int pos = a.positions[token];
                f32x8 c, s;
                if (pos >= 0 && pos < a.max_pos) {
                    const float *t = a.table + static_cast<long long>(pos) * r + 8 * unit;
                    c = *reinterpret_cast<const f32x8 *>(t);
                    s = *reinterpret_cast<const f32x8 *>(t + half);
                } else {
                    c = __builtin_nanf("");
                    s = c;
                }
                turn8(a.interleaved, c, s * a.sign, ua, ub);
            }
        }
        double squares = 0.0, products = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double p = xa[i], q = xb[i];
            squares = __builtin_fma(p, p, squares);
            squares = __builtin_fma(q, q, squares);
            products = __builtin_fma(static_cast<double>(fa[i] * ua[i]), p, products);
            products = __builtin_fma(static_cast<double>(fb[i] * ub[i]), q, products);
        }
        for (int off = a.units >> 1; off > 0; off >>= 1) {
            squares += __shfl_xor(squares, off);
            products += __shfl_xor(products, off);
        }
        if (live) {
            const NormGradHead h = norm_grad_head(squares, products, a);
            const f32x8 ma = xa * h.r, mb = xb * h.r;
            T *dx = static_cast<T *>(a.dx) + token * a.dx_ts + head * a.dx_hs;
            *reinterpret_cast<vec8 *>(dx + ea) = __builtin_convertvector((fa * ua - ma * h.mean) * h.r, vec8);
            *reinterpret_cast<vec8 *>(dx + eb) = __builtin_convertvector((fb * ub - mb * h.mean) * h.r, vec8);
            wa += ua * ma;
            wb += ub * mb;
        }
    }
    if (a.part == nullptr) {
        return;
    }
    const int width = 16 * a.units;
    if (on) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s_dw[at * width + ea + i] = wa[i];
            s_dw[at * width + eb + i] = wb[i];
        }
    }
    __syncthreads();
    for (int e = tid; e < a.head_dim; e += kRopeThreads) {
        double sum = 0.0;
        for (int i = 0; i < heads_at_once; ++i) {
            sum += s_dw[i * width + e];
        }
        a.part[static_cast<long long>(blockIdx.x) * a.head_dim + e] = static_cast<float>(sum);
    }
}

// Any head_dim, rotary_dim, stride and alignment: a wave goes over every so many-th head, a lane takes pairs,
// then elements past them, so that a lane's elements are the same in all of its heads.
template <typename T>
__global__ __launch_bounds__(kRopeThreads) void norm_grad_any_kernel(NormGradArgs a)
{
    const int lane = threadIdx.x & 63;
    const uint32_t wave = blockIdx.x * (kRopeThreads / 64) + (threadIdx.x >> 6);
    const uint32_t waves = gridDim.x * (kRopeThreads / 64);
    const int r = a.rotary_dim, half = r >> 1;
    float *part = a.part == nullptr ? nullptr : a.part + static_cast<long long>(wave) * a.head_dim;
    if (part != nullptr) {
        for (int i = lane; i < half; i += 64) {
            part[a.interleaved ? 2 * i : i] = 0.0f;
            part[a.interleaved ? 2 * i + 1 : half + i] = 0.0f;
        }
        for (int e = r + lane; e < a.head_dim; e += 64) {
            part[e] = 0.0f;
        }
    }
    for (uint32_t row = wave; row < a.rows; row += waves) {
        uint32_t head;
        const int token = static_cast<int>(fast_div(row, a.heads, head));
        const T *x = static_cast<const T *>(a.x) + token * a.x_ts + head * a.x_hs;
        const T *dy = static_cast<const T *>(a.dy) + token * a.dy_ts + head * a.dy_hs;
        T *dx = static_cast<T *>(a.dx) + token * a.dx_ts + head * a.dx_hs;
        const float *t = nullptr;
        if (r > 0) {
            const int pos = a.positions[token];
            t = pos >= 0 && pos < a.max_pos ? a.table + static_cast<long long>(pos) * r : nullptr;
        }
        auto factor = [&](int e) { return a.weight != nullptr ? a.weight[e] + a.shift : 1.0f; };
        // calls f with every element of this lane and its u
        auto each = [&](auto f) {
            for (int i = lane; i < half; i += 64) {
                const int e1 = a.interleaved ? 2 * i : i, e2 = a.interleaved ? 2 * i + 1 : half + i;
                const float p = static_cast<float>(dy[e1]), q = static_cast<float>(dy[e2]);
                const float c = t ? t[i] : __builtin_nanf("");
                const float s = (t ? t[half + i] : __builtin_nanf("")) * a.sign;
                const float x1 = static_cast<float>(x[e1]), x2 = static_cast<float>(x[e2]);
                f(e1, x1, p * c - q * s);
                f(e2, x2, q * c + p * s);
            }
            for (int e = r + lane; e < a.head_dim; e += 64) {
                f(e, static_cast<float>(x[e]), static_cast<float>(dy[e]));
            }
        };
        double squares = 0.0, products = 0.0;
        each([&](int e, float xe, float u) {
            squares = __builtin_fma(static_cast<double>(xe), static_cast<double>(xe), squares);
            products = __builtin_fma(static_cast<double>(factor(e) * u), static_cast<double>(xe), products);
        });
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            squares += __shfl_xor(squares, off);
            products += __shfl_xor(products, off);
        }
        const NormGradHead h = norm_grad_head(squares, products, a);
        each([&](int e, float xe, float u) {
            const float m = xe * h.r;
            dx[e] = static_cast<T>((factor(e) * u - m * h.mean) * h.r);
            if (part != nullptr) {
                part[e] += u * m;
            }
        });
    }
}

// dweight from `parts` shares of it: a workgroup takes 4 elements, 64 threads over the shares of each.
__global__ __launch_bounds__(256) void norm_grad_join_kernel(const float *part, int parts, int head_dim,
                                                             float *dweight)
{
    __shared__ double s_sum[64][4];
    const int e = blockIdx.x * 4 + (threadIdx.x & 3), at = threadIdx.x >> 2;
    double sum = 0.0;
    if (e < head_dim) {
        // 16 loads in flight whatever `parts` is: past the end they are the last share's (with a remainder's one by
        // one, the gradient of 500, 1000 tokens of 32 heads of 128 took 11.8, 17.2 us, now 10.0, 13.3)
        for (int i = at; i < parts; i += 64 * 16) {
            float x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                x[j] = part[static_cast<long long>(min(i + 64 * j, parts - 1)) * head_dim + e];
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                sum += i + 64 * j < parts ? x[j] : 0.0f;
            }
        }
    }
    s_sum[at][threadIdx.x & 3] = sum;
    for (int n = 32; n > 0; n >>= 1) {
        __syncthreads();
        if (at < n) {
            s_sum[at][threadIdx.x & 3] += s_sum[at + n][threadIdx.x & 3];
        }
    }
    if (at == 0 && e < head_dim) {
        dweight[e] = static_cast<float>(s_sum[0][threadIdx.x]);
    }
}

// ---------------------------------------------------------------------------------------------
// Checks and launches
// ---------------------------------------------------------------------------------------------

const char *norm_error(const tqt_head_norm &n)
{
    return n.eps > 0.0f && std::isfinite(n.eps) && std::isfinite(n.shift)
               ? nullptr
               : "eps is not a finite number > 0, or shift is not finite";
}

const char *norm_rope_error(const tqt_norm_rope_params *p)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    const char *e = rope_error(&p->rope);
    return e != nullptr || p->rope.tokens == 0 || p->rope.heads == 0 || p->rope.head_dim == 0 ? e
                                                                                              : norm_error(p->norm);
}

template <typename T>
bool run_norm_rope(const tqt_norm_rope_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = norm_rope_error(p);
    TQT_REQUIRE(error == nullptr, error);
    return run_rope<T, true>(&p->rope, &p->norm, stream, where);
}

const char *append_norm_error(const tqt_kv_append_norm_rope_params *p, size_t cache_bytes, bool quant)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    const char *e = append_error(&p->append, cache_bytes, quant);
    if (e == nullptr && p->append.tokens > 0) {
        e = norm_error(p->k_norm);
        e = e == nullptr && p->append.q_heads > 0 ? norm_error(p->q_norm) : e;
    }
    return e;
}

template <typename SRC, typename DST, typename CACHE>
bool run_append_norm(const tqt_kv_append_norm_rope_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = append_norm_error(p, sizeof(CACHE), std::is_same<CACHE, int8_t>::value);
    TQT_REQUIRE(error == nullptr, error);
    return run_append<SRC, DST, CACHE, true>(&p->append, &p->q_norm, &p->k_norm, stream, where);
}

// dX alone, with nothing to sum.
bool grad_empty(const tqt_rope_params &p)
{
    return p.tokens == 0 || p.heads == 0 || p.head_dim == 0;
}

const char *grad_error(const tqt_norm_rope_grad_params *p)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    const tqt_rope_params &f = p->forward.rope;
    if (f.tokens >= (1u << 31) || f.heads >= (1u << 20) || f.head_dim >= (1u << 20) ||
        f.tokens * f.heads >= (1u << 31)) {
        return "tokens, heads, tokens * heads or head_dim too large";
    }
    if (f.head_dim == 0 || (grad_empty(f) && p->dweight == nullptr)) {
        return nullptr;
    }
    if (!grad_empty(f)) {
        if (f.X == nullptr || p->dY == nullptr || p->dX == nullptr) {
            return "X / dY / dX == NULL";
        }
        if (const char *e = map_error(f.map, f.head_dim, f.positions)) {
            return e;
        }
        if (const char *e = norm_error(p->forward.norm)) {
            return e;
        }
    }
    const size_t need = tqt_get_workspace_size_norm_rope_grad_gfx950(p);
    if (p->workspace_size < need || (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace)))) {
        return "the workspace is too small or off the 16-byte grid";
    }
    return nullptr;
}

template <typename T>
bool run_grad(const tqt_norm_rope_grad_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = grad_error(p);
    TQT_REQUIRE(error == nullptr, error);
    const tqt_rope_params &f = p->forward.rope;
    if (f.head_dim == 0 || (grad_empty(f) && p->dweight == nullptr)) {
        return false;
    }
    NormGradArgs a = {};
    a.x = f.X;
    a.dy = p->dY;
    a.dx = p->dX;
    a.x_ts = f.x_token_stride;
    a.x_hs = f.x_head_stride;
    a.dy_ts = p->dy_token_stride;
    a.dy_hs = p->dy_head_stride;
    a.dx_ts = p->dx_token_stride;
    a.dx_hs = p->dx_head_stride;
    a.positions = f.positions;
    a.table = f.map.table;
    a.max_pos = static_cast<int>(f.map.max_pos);
    a.rotary_dim = static_cast<int>(f.map.rotary_dim);
    a.interleaved = f.map.interleaved != 0;
    a.sign = f.map.inverse != 0 ? 1.0f : -1.0f;  // turned back
    a.weight = p->forward.norm.weight;
    a.shift = p->forward.norm.shift;
    a.eps = p->forward.norm.eps;
    a.head_dim = static_cast<int>(f.head_dim);
    a.rows = static_cast<uint32_t>(f.tokens * f.heads);
    int blocks = 0;
    if (a.rows > 0) {
        a.heads = make_fast_div(static_cast<uint32_t>(f.heads));
        const bool rows = f.head_dim % 16 == 0 && f.map.rotary_dim % 16 == 0 && a.head_dim <= kNormMostDim &&
                          aligned16(a.table) && aligned16(a.weight) &&
                          on_grid(f.X, f.x_token_stride, f.x_head_stride, sizeof(T)) &&
                          on_grid(p->dY, p->dy_token_stride, p->dy_head_stride, sizeof(T)) &&
                          on_grid(p->dX, p->dx_token_stride, p->dx_head_stride, sizeof(T));
        const NormGradLaunch g = norm_grad_launch(a.rows, a.head_dim);
        a.part = p->dweight == nullptr ? nullptr : static_cast<float *>(p->workspace);
        a.units = g.units;
        if (rows) {
            blocks = g.row_blocks;
            hipLaunchKernelGGL((norm_grad_rows_kernel<T>), dim3(blocks), dim3(kRopeThreads), 0, stream, a);
        } else {
            blocks = 4 * g.any_blocks;
            hipLaunchKernelGGL((norm_grad_any_kernel<T>), dim3(g.any_blocks), dim3(kRopeThreads), 0, stream, a);
        }
        check_launch(where);
    }
    if (p->dweight != nullptr) {
        hipLaunchKernelGGL(norm_grad_join_kernel, dim3((a.head_dim + 3) / 4), dim3(256), 0, stream,
                           static_cast<const float *>(p->workspace), blocks, a.head_dim, p->dweight);
        check_launch(where);
    }
    return true;
}

}  // namespace
}  // namespace tqt

using namespace tqt;

extern "C" {

size_t tqt_get_workspace_size_norm_rope_grad_gfx950(const struct tqt_norm_rope_grad_params *params)
{
    if (params == nullptr || params->dweight == nullptr) {
        return 0;
    }
    const tqt_rope_params &f = params->forward.rope;
    if (grad_empty(f) || f.tokens >= (1u << 31) || f.heads >= (1u << 20) || f.head_dim >= (1u << 20) ||
        f.tokens * f.heads >= (1u << 31)) {
        return 0;
    }
    const NormGradLaunch g = norm_grad_launch(static_cast<long long>(f.tokens * f.heads),
                                              static_cast<long long>(f.head_dim));
    // either kernel may take the call: alignment decides
    return std::max(g.row_blocks, 4 * g.any_blocks) * f.head_dim * sizeof(float);
}

#define TQT_NORM_ROPE_ENTRIES(NAME, T)                                                                \
    const char *tqt_get_error_norm_rope_##NAME##_gfx950(const struct tqt_norm_rope_params *params)    \
    {                                                                                                 \
        return norm_rope_error(params);                                                               \
    }                                                                                                 \
    void tqt_run_norm_rope_##NAME##_gfx950_async(const struct tqt_norm_rope_params *params,           \
                                                 void *stream)                                        \
    {                                                                                                 \
        run_norm_rope<T>(params, as_stream(stream), "tqt_run_norm_rope_" #NAME "_gfx950");            \
    }                                                                                                 \
    void tqt_run_norm_rope_##NAME##_gfx950(const struct tqt_norm_rope_params *params)                 \
    {                                                                                                 \
        if (run_norm_rope<T>(params, nullptr, "tqt_run_norm_rope_" #NAME "_gfx950")) {                \
            finish_sync(nullptr, "tqt_run_norm_rope_" #NAME "_gfx950");                               \
        }                                                                                             \
    }                                                                                                 \
    const char *tqt_get_error_norm_rope_grad_##NAME##_gfx950(                                         \
        const struct tqt_norm_rope_grad_params *params)                                               \
    {                                                                                                 \
        return grad_error(params);                                                                    \
    }                                                                                                 \
    void tqt_run_norm_rope_grad_##NAME##_gfx950_async(const struct tqt_norm_rope_grad_params *params, \
                                                      void *stream)                                   \
    {                                                                                                 \
        run_grad<T>(params, as_stream(stream), "tqt_run_norm_rope_grad_" #NAME "_gfx950");            \
    }                                                                                                 \
    void tqt_run_norm_rope_grad_##NAME##_gfx950(const struct tqt_norm_rope_grad_params *params)       \
    {                                                                                                 \
        if (run_grad<T>(params, nullptr, "tqt_run_norm_rope_grad_" #NAME "_gfx950")) {                \
            finish_sync(nullptr, "tqt_run_norm_rope_grad_" #NAME "_gfx950");                          \
        }                                                                                             \
    }

TQT_NORM_ROPE_ENTRIES(f32, float)
TQT_NORM_ROPE_ENTRIES(f16, _Float16)
TQT_NORM_ROPE_ENTRIES(bf16, __bf16)

#define TQT_APPEND_NORM_ENTRIES(NAME, SRC, DST, CACHE)                                                \
    const char *tqt_get_error_kv_append_norm_rope_##NAME##_gfx950(                                    \
        const struct tqt_kv_append_norm_rope_params *params)                                          \
    {                                                                                                 \
        return append_norm_error(params, sizeof(CACHE), std::is_same<CACHE, int8_t>::value);          \
    }                                                                                                 \
    void tqt_run_kv_append_norm_rope_##NAME##_gfx950_async(                                           \
        const struct tqt_kv_append_norm_rope_params *params, void *stream)                            \
    {                                                                                                 \
        run_append_norm<SRC, DST, CACHE>(params, as_stream(stream),                                   \
                                         "tqt_run_kv_append_norm_rope_" #NAME "_gfx950");             \
    }                                                                                                 \
    void tqt_run_kv_append_norm_rope_##NAME##_gfx950(                                                 \
        const struct tqt_kv_append_norm_rope_params *params)                                          \
    {                                                                                                 \
        if (run_append_norm<SRC, DST, CACHE>(params, nullptr,                                         \
                                             "tqt_run_kv_append_norm_rope_" #NAME "_gfx950")) {       \
            finish_sync(nullptr, "tqt_run_kv_append_norm_rope_" #NAME "_gfx950");                     \
        }                                                                                             \
    }

TQT_APPEND_NORM_ENTRIES(f16_f16, _Float16, _Float16, _Float16)
TQT_APPEND_NORM_ENTRIES(bf16_bf16, __bf16, __bf16, __bf16)
TQT_APPEND_NORM_ENTRIES(f16_f32, float, _Float16, _Float16)
TQT_APPEND_NORM_ENTRIES(bf16_f32, float, __bf16, __bf16)
TQT_APPEND_NORM_ENTRIES(qsi8dx_f16, _Float16, _Float16, int8_t)
TQT_APPEND_NORM_ENTRIES(qsi8dx_bf16, __bf16, __bf16, int8_t)

}  // extern "C"
