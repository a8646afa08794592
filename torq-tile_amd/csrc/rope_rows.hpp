// What the kernels of rotary positions and of the append to a paged cache share with those that normalise the heads
// on the way: a call's arguments and its checks, the two kernels, and their launches.
//
//   y1 = x1 c - x2 s, y2 = x2 c + x1 s   for pairs (i, i + r / 2) or (2 i, 2 i + 1), i < r / 2
//
// with (c, s) of the token's position from a table, every product and sum in f32 rounded on its own (the
// library is built with -ffp-contract=off) and one rounding to the result's type; with a norm, x is
// x / sqrt(mean(x^2) + eps) * factor first. Bound by memory: each element is read once and written once; the table
// row of a token (4 r bytes) is shared by its heads.
//
// Split: one thread takes 16 elements of a head, the 8 + 8 of 8 pairs, as two 16-byte pieces (four for f32
// sources), so that a pair never crosses threads and the operation works in place. Threads of a token lie
// along its heads, so the 64 bytes of the table that a thread reads come from its CU's cache for all but the
// first of them (four heads a thread, which share them in registers, took 16.9 instead of 14.2 us for 1000
// tokens of 96 int8 heads and 26.6 instead of 24.2 for 4096 of 48 from f32: fewer waves have loads in flight).
// A norm, or an int8 row's maximum, is a sum over a head's threads, a power of two of them side by side: a
// butterfly of lane moves, whose instructions hide behind the loads (the kernels alone, without and with a norm: 4099
// tokens of 32 bf16 heads of 128, 64 turned, 15.4 and 15.6-16.7 us; 4096 tokens of 32 + 8 + 8 heads from f32 into an f16
// cache 23.0-24.5 and 28.5-30.2, 5.1 TB/s; calls in a row, into an int8 cache from bf16: those 4096 tokens 19.9 and 22.2,
// 4.2-4.7 TB/s, 1000 of 32 + 32 + 32 heads 11.0 and 13.1). The squares are summed in f64, which costs 4% at most (f32:
// 48.1 us where a training step's two calls now take 50.1; the append 33.6 and 34.4).
#pragma once

#include "fast_div.hpp"
#include "paged_kv.hpp"
#include "rope_route.hpp"
#include "tqt_hip_common.hpp"
#include "tqt_kv_append_norm_rope_gfx950.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tqt {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef int8_t i8x8 __attribute__((ext_vector_type(8)));

constexpr int kRopeThreads = 256;

template <typename T>
struct Vec8;
template <>
struct Vec8<float>
{
    typedef f32x8 type;
};
template <>
struct Vec8<_Float16>
{
    typedef f16x8 type;
};
template <>
struct Vec8<__bf16>
{
    typedef bf16x8 type;
};

// The tensors of a call: `rows` heads per token, q heads first, then k, then v (rope alone: q heads only).
struct RopeArgs
{
    const void *q, *k, *v;
    void *q_out;
    long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs;
    const int32_t *positions;
    const float *table;
    int max_pos, rotary_dim, interleaved;
    float sign;  // -1 for the inverse rotation
    int head_dim, q_heads, kv_heads;
    int tokens;
    FastDiv units, heads;  // threads per head, heads (rows) per token
    int rows;
    // the cache
    const int64_t *slots;
    void *ck, *cv;
    float *scale_k, *scale_v;
    long long num_slots, page_stride, token_stride, head_stride;
    FastDiv page;
    // the norm of q heads and of k heads
    struct Norm
    {
        const float *weight;
        float shift, eps;
    } q_norm, k_norm;
};

// A head's factor 1 / sqrt(mean + eps) from the sum of its squares. In 64 bits: squares of f32 values are exact and
// cannot overflow.
__device__ __forceinline__ float norm_factor(double squares, int head_dim, float eps)
{
    return static_cast<float>(1.0 / sqrt(squares / head_dim + eps));
}

// amax that keeps a NaN
__device__ __forceinline__ float nan_max(float m, float a)
{
    return a > m || a != a ? a : m;
}

// The scale of a row of an int8 cache, NaN for a row with a NaN or an infinity; `zero`: every q is 0 (a scale that
// is 0 in f32 too).
struct QuantRow
{
    float scale, inverse;
    bool zero, plain;
};

__device__ __forceinline__ QuantRow quant_row(float amax)
{
    QuantRow r;
    r.scale = amax < INFINITY ? amax * (1.0f / 127.0f) : __builtin_nanf("");
    r.zero = r.scale == 0.0f;
    if (r.zero) {
        r.scale = 1.0f;
    }
    r.inverse = 1.0f / r.scale;
    r.plain = r.scale >= 0x1p-80f && r.scale <= 0x1p100f;
    return r;
}

// nearbyint(x / scale). The quotient is correctly rounded without a division: from the correctly rounded inverse,
// two corrections by the exact remainder (the second starts within an ulp). A remainder underflows only for |x|
// below 2^-101, a quotient below 2^-20 here, which rounds to 0 either way.
__device__ __forceinline__ int8_t quant_value(float x, const QuantRow &r)
{
    float y;
    if (r.plain) {
        y = x * r.inverse;
        y = __builtin_fmaf(__builtin_fmaf(-y, r.scale, x), r.inverse, y);
        y = __builtin_fmaf(__builtin_fmaf(-y, r.scale, x), r.inverse, y);
    } else {
        y = x / r.scale;
    }
    const float q = fminf(fmaxf(rintf(y), -127.0f), 127.0f);
    return r.zero ? static_cast<int8_t>(0) : static_cast<int8_t>(q);
}

// Where a token's key and value go: a null slot is not written.
struct Slot
{
    bool used;
    long long base;         // element offset of the token's first head
    long long scale_base;   // its first head's scale
};

__device__ __forceinline__ Slot find_slot(const RopeArgs &a, int token)
{
    Slot s;
    const long long at = a.slots[token];
    s.used = at >= 0 && at < a.num_slots;
    uint32_t offset;
    const uint32_t page = fast_div(s.used ? static_cast<uint32_t>(at) : 0u, a.page, offset);
    s.base = page * a.page_stride + offset * a.token_stride;
    s.scale_base = static_cast<long long>(page) * a.kv_heads * a.page.d + offset;
    return s;
}

// One thread: 16 elements of a head. SRC: type of X (or Q, K, V); DST: type of Y; CACHE: the cache's type, void
// for rope alone; kNorm: heads of Q and K are normalised first.
template <typename SRC, typename DST, typename CACHE, bool kNorm>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeArgs a, int token0, uint32_t items)
{
    constexpr bool kCache = !std::is_same<CACHE, void>::value;
    constexpr bool kQuant = std::is_same<CACHE, int8_t>::value;
    typedef typename Vec8<SRC>::type src8;
    typedef typename Vec8<DST>::type dst8;

    const uint32_t index = blockIdx.x * kRopeThreads + threadIdx.x;
    const bool live = index < items;
    uint32_t unit, urow;
    const uint32_t rest = fast_div(live ? index : 0u, a.units, unit);
    const int token = token0 + static_cast<int>(fast_div(rest, a.heads, urow));
    const int row = static_cast<int>(urow);
    const bool query = !kCache || row < a.q_heads;
    const bool value = kCache && row >= a.q_heads + a.kv_heads;
    const int head = query ? row : (value ? row - a.q_heads - a.kv_heads : row - a.q_heads);
    const int r = a.rotary_dim, half = r >> 1;
    const bool turned = static_cast<int>(16 * unit) < r;
    int ea = 16 * unit, eb = ea + 8;  // first elements of the two pieces
    if (turned && !a.interleaved) {
        ea = 8 * unit;
        eb = half + ea;
    }
    Slot slot = {false, 0, 0};
    if (kCache && live && !query) {
        slot = find_slot(a, token);
    }
    // an int8 or normalised head has a power of two of threads, some of them past its end
    const bool on = live && static_cast<int>(16 * unit) < a.head_dim && (query || slot.used);
    f32x8 xa = 0.0f, xb = 0.0f;
    if (on) {
        const SRC *x = query ? static_cast<const SRC *>(a.q) + token * a.q_ts + head * a.q_hs
                             : (value ? static_cast<const SRC *>(a.v) + token * a.v_ts + head * a.v_hs
                                      : static_cast<const SRC *>(a.k) + token * a.k_ts + head * a.k_hs);
        xa = __builtin_convertvector(*reinterpret_cast<const src8 *>(x + ea), f32x8);
        xb = __builtin_convertvector(*reinterpret_cast<const src8 *>(x + eb), f32x8);
    }
    if constexpr (kNorm) {
        double squares = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            squares = __builtin_fma(static_cast<double>(xa[i]), static_cast<double>(xa[i]), squares);
            squares = __builtin_fma(static_cast<double>(xb[i]), static_cast<double>(xb[i]), squares);
        }
        for (uint32_t off = a.units.d >> 1; off > 0; off >>= 1) {
            squares += __shfl_xor(squares, static_cast<int>(off));
        }
        if (on && !value) {
            const RopeArgs::Norm &norm = query ? a.q_norm : a.k_norm;
            const float f = norm_factor(squares, a.head_dim, norm.eps);
            xa = xa * f;
            xb = xb * f;
            if (norm.weight != nullptr) {
                xa = xa * (*reinterpret_cast<const f32x8 *>(norm.weight + ea) + norm.shift);
                xb = xb * (*reinterpret_cast<const f32x8 *>(norm.weight + eb) + norm.shift);
            }
        }
    }
    if (on && turned && !value) {
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
        // (as a function, inlined, this takes the int8 instances 70 registers instead of 60 and 7 waves a SIMD instead of
        // 8: 4096 tokens of 32 + 8 + 8 heads of 128 19.95 instead of 19.85 us, with a norm 22.6 instead of 22.2)
        s = s * a.sign;
        const f32x8 p = xa, q = xb;
        if (a.interleaved) {
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
    QuantRow quant = {1.0f, 1.0f, true, true};
    if constexpr (kQuant) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            amax = nan_max(nan_max(amax, fabsf(xa[i])), fabsf(xb[i]));
        }
        for (uint32_t off = a.units.d >> 1; off > 0; off >>= 1) {
            amax = nan_max(amax, __shfl_xor(amax, static_cast<int>(off)));
        }
        quant = quant_row(amax);
    }
    if (!on) {
        return;
    }
    if (query) {
        DST *y = static_cast<DST *>(a.q_out) + token * a.qo_ts + head * a.qo_hs;
        *reinterpret_cast<dst8 *>(y + ea) = __builtin_convertvector(xa, dst8);
        *reinterpret_cast<dst8 *>(y + eb) = __builtin_convertvector(xb, dst8);
        return;
    }
    if constexpr (kCache) {
        CACHE *y = static_cast<CACHE *>(value ? a.cv : a.ck) + slot.base + head * a.head_stride;
        if constexpr (kQuant) {
            i8x8 qa, qb;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                qa[i] = quant_value(xa[i], quant);
                qb[i] = quant_value(xb[i], quant);
            }
            *reinterpret_cast<i8x8 *>(y + ea) = qa;
            *reinterpret_cast<i8x8 *>(y + eb) = qb;
            if (unit == 0) {
                (value ? a.scale_v : a.scale_k)[slot.scale_base +
                                                static_cast<long long>(head) * a.page.d] = quant.scale;
            }
        } else {
            typedef typename Vec8<CACHE>::type cache8;
            *reinterpret_cast<cache8 *>(y + ea) = __builtin_convertvector(xa, cache8);
            *reinterpret_cast<cache8 *>(y + eb) = __builtin_convertvector(xb, cache8);
        }
    }
}

// Any head_dim, rotary_dim, stride and alignment: a wave per head, a lane per pair, then per element past
// them. Both elements of a pair are read before either is written (in place).
template <typename SRC, typename DST, typename CACHE, bool kNorm>
__global__ __launch_bounds__(kRopeThreads) void rope_any_kernel(RopeArgs a, int token0, uint32_t items)
{
    constexpr bool kCache = !std::is_same<CACHE, void>::value;
    constexpr bool kQuant = std::is_same<CACHE, int8_t>::value;
    const int lane = threadIdx.x & 63;
    const uint32_t item = blockIdx.x * (kRopeThreads / 64) + (threadIdx.x >> 6);
    if (item >= items) {
        return;
    }
    uint32_t urow;
    const int token = token0 + static_cast<int>(fast_div(item, a.heads, urow));
    const int row = static_cast<int>(urow);
    const bool query = !kCache || row < a.q_heads;
    const bool value = kCache && row >= a.q_heads + a.kv_heads;
    const int head = query ? row : (value ? row - a.q_heads - a.kv_heads : row - a.q_heads);
    Slot slot = {false, 0, 0};
    if (kCache && !query) {
        slot = find_slot(a, token);
        if (!slot.used) {
            return;
        }
    }
    const SRC *x = query ? static_cast<const SRC *>(a.q) + token * a.q_ts + head * a.q_hs
                         : (value ? static_cast<const SRC *>(a.v) + token * a.v_ts + head * a.v_hs
                                  : static_cast<const SRC *>(a.k) + token * a.k_ts + head * a.k_hs);
    const int r = value ? 0 : a.rotary_dim, half = r >> 1;
    const float *t = nullptr;
    if (r > 0) {
        const int pos = a.positions[token];
        t = pos >= 0 && pos < a.max_pos ? a.table + static_cast<long long>(pos) * r : nullptr;
    }
    const RopeArgs::Norm &norm = query ? a.q_norm : a.k_norm;
    float f = 1.0f;
    if (kNorm && !value) {
        double squares = 0.0;
        for (int e = lane; e < a.head_dim; e += 64) {
            const double y = static_cast<double>(static_cast<float>(x[e]));
            squares = __builtin_fma(y, y, squares);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            squares += __shfl_xor(squares, off);
        }
        f = norm_factor(squares, a.head_dim, norm.eps);
    }
    auto get = [&](int e) {
        float y = static_cast<float>(x[e]);
        if (kNorm && !value) {
            y *= f;
            y = norm.weight != nullptr ? y * (norm.weight[e] + norm.shift) : y;
        }
        return y;
    };
    QuantRow quant = {1.0f, 1.0f, true, true};
    float amax = 0.0f;
    // an int8 row is gone through twice: its amax, then its values
    for (int pass = kQuant && !query ? 0 : 1; pass < 2; ++pass) {
        auto put = [&](int e, float y) {
            if (query) {
                (static_cast<DST *>(a.q_out) + token * a.qo_ts + head * a.qo_hs)[e] = static_cast<DST>(y);
            } else if constexpr (kQuant) {
                if (pass == 0) {
                    amax = nan_max(amax, fabsf(y));
                } else {
                    (static_cast<int8_t *>(value ? a.cv : a.ck) + slot.base + head * a.head_stride)[e] =
                        quant_value(y, quant);
                }
            } else if constexpr (kCache) {
                (static_cast<CACHE *>(value ? a.cv : a.ck) + slot.base + head * a.head_stride)[e] =
                    static_cast<CACHE>(y);
            }
        };
        for (int i = lane; i < half; i += 64) {
            const int e1 = a.interleaved ? 2 * i : i, e2 = a.interleaved ? 2 * i + 1 : half + i;
            const float p = get(e1), q = get(e2);
            const float c = t ? t[i] : __builtin_nanf("");
            const float s = (t ? t[half + i] : __builtin_nanf("")) * a.sign;
            put(e1, p * c - q * s);
            put(e2, q * c + p * s);
        }
        for (int e = r + lane; e < a.head_dim; e += 64) {
            put(e, get(e));
        }
        if (kQuant && pass == 0) {
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                amax = nan_max(amax, __shfl_xor(amax, off));
            }
            quant = quant_row(amax);
            if (lane == 0) {
                (value ? a.scale_v : a.scale_k)[slot.scale_base + static_cast<long long>(head) * a.page.d] =
                    quant.scale;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Checks
// ---------------------------------------------------------------------------------------------

const char *map_error(const tqt_rope_map &m, size_t head_dim, const int32_t *positions)
{
    if (m.rotary_dim == 0) {
        return nullptr;
    }
    if (m.rotary_dim % 2 != 0 || m.rotary_dim > head_dim) {
        return "rotary_dim is odd or > head_dim";
    }
    if (m.table == nullptr || positions == nullptr) {
        return "table / positions == NULL";
    }
    if (m.max_pos == 0 || m.max_pos >= (1u << 31)) {
        return "max_pos is 0 or exceeds 2^31-1";
    }
    return nullptr;
}

const char *rope_error(const tqt_rope_params *p)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    if (p->tokens >= (1u << 31) || p->heads >= (1u << 20) || p->head_dim >= (1u << 20)) {
        return "tokens, heads or head_dim too large";
    }
    if (p->tokens == 0 || p->heads == 0 || p->head_dim == 0) {
        return nullptr;
    }
    if (p->X == nullptr || p->Y == nullptr) {
        return "X / Y == NULL";
    }
    return map_error(p->map, p->head_dim, p->positions);
}

bool on_grid(const void *p, size_t ts, size_t hs, size_t bytes)
{
    return aligned16(p) && ts * bytes % 16 == 0 && hs * bytes % 16 == 0;
}

void set_map(RopeArgs &a, const tqt_rope_map &m, const int32_t *positions)
{
    a.positions = positions;
    a.table = m.table;
    a.max_pos = static_cast<int>(m.max_pos);
    a.rotary_dim = static_cast<int>(m.rotary_dim);
    a.interleaved = m.interleaved != 0;
    a.sign = m.inverse != 0 ? -1.0f : 1.0f;
}

// The norm of a call, nullptr for none; false if its weight keeps it from the fast kernel.
bool set_norm(RopeArgs::Norm &to, const tqt_head_norm *n)
{
    to = {};
    if (n != nullptr) {
        to = {n->weight, n->shift, n->eps};
    }
    return n == nullptr || aligned16(n->weight);
}

// Launches the rows of all tokens. grid16: they suit rope_rows_kernel.
template <typename SRC, typename DST, typename CACHE, bool kNorm>
void launch_rows(RopeArgs a, bool grid16, hipStream_t stream, const char *where)
{
    const RopeLaunch r = rope_launch(a.rows, a.head_dim, grid16 && (!kNorm || a.head_dim <= kNormMostDim),
                                     kNorm || std::is_same<CACHE, int8_t>::value);
    a.units = make_fast_div(static_cast<uint32_t>(r.per_head));
    a.heads = make_fast_div(a.rows);
    for (long long t0 = 0; t0 < a.tokens; t0 += r.tokens) {
        const long long n = std::min(r.tokens, a.tokens - t0);
        const uint32_t items = static_cast<uint32_t>(n * a.rows * r.per_head);
        const int per_block = r.rows ? kRopeThreads : kRopeThreads / 64;
        const dim3 grid((items + per_block - 1) / per_block);
        if (r.rows) {
            hipLaunchKernelGGL((rope_rows_kernel<SRC, DST, CACHE, kNorm>), grid, dim3(kRopeThreads), 0, stream, a,
                               static_cast<int>(t0), items);
        } else {
            hipLaunchKernelGGL((rope_any_kernel<SRC, DST, CACHE, kNorm>), grid, dim3(kRopeThreads), 0, stream, a,
                               static_cast<int>(t0), items);
        }
        check_launch(where);
    }
}

const char *append_error(const tqt_kv_append_rope_params *p, size_t cache_bytes, bool quant)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    if (p->tokens == 0) {
        return nullptr;
    }
    const tqt_paged_kv &c = p->kv;
    if (p->tokens >= (1u << 31) || p->q_heads >= (1u << 20)) {
        return "tokens or q_heads too large";
    }
    if (const char *e = paged_kv_error(c, cache_bytes, quant)) {
        return e;
    }
    if (p->K == nullptr || p->V == nullptr || p->slots == nullptr) {
        return "K / V / slots == NULL";
    }
    if (p->q_heads > 0 && (p->Q == nullptr || p->Q_out == nullptr)) {
        return "Q / Q_out == NULL";
    }
    return map_error(p->map, c.head_dim, p->positions);
}

// Runs a call that has been checked; false: there is nothing to do.
template <typename T, bool kNorm>
bool run_rope(const tqt_rope_params *p, const tqt_head_norm *norm, hipStream_t stream, const char *where)
{
    if (p->tokens == 0 || p->heads == 0 || p->head_dim == 0) {
        return false;
    }
    RopeArgs a = {};
    a.q = p->X;
    a.q_out = p->Y;
    a.q_ts = p->x_token_stride;
    a.q_hs = p->x_head_stride;
    a.qo_ts = p->y_token_stride;
    a.qo_hs = p->y_head_stride;
    set_map(a, p->map, p->positions);
    a.head_dim = static_cast<int>(p->head_dim);
    a.q_heads = a.rows = static_cast<int>(p->heads);
    a.tokens = static_cast<int>(p->tokens);
    const bool vec = set_norm(a.q_norm, norm) && p->head_dim % 16 == 0 && p->map.rotary_dim % 16 == 0 && aligned16(p->map.table) &&
                     on_grid(p->X, p->x_token_stride, p->x_head_stride, sizeof(T)) &&
                     on_grid(p->Y, p->y_token_stride, p->y_head_stride, sizeof(T));
    launch_rows<T, T, void, kNorm>(a, vec, stream, where);
    return true;
}

template <typename SRC, typename DST, typename CACHE, bool kNorm>
bool run_append(const tqt_kv_append_rope_params *p, const tqt_head_norm *q_norm, const tqt_head_norm *k_norm,
                hipStream_t stream, const char *where)
{
    if (p->tokens == 0) {
        return false;
    }
    const tqt_paged_kv &c = p->kv;
    RopeArgs a = {};
    a.q = p->Q;
    a.k = p->K;
    a.v = p->V;
    a.q_out = p->Q_out;
    a.q_ts = p->q_token_stride;
    a.q_hs = p->q_head_stride;
    a.k_ts = p->k_token_stride;
    a.k_hs = p->k_head_stride;
    a.v_ts = p->v_token_stride;
    a.v_hs = p->v_head_stride;
    a.qo_ts = p->qo_token_stride;
    a.qo_hs = p->qo_head_stride;
    set_map(a, p->map, p->positions);
    a.head_dim = static_cast<int>(c.head_dim);
    a.q_heads = static_cast<int>(p->q_heads);
    a.kv_heads = static_cast<int>(c.kv_heads);
    a.rows = a.q_heads + 2 * a.kv_heads;
    a.tokens = static_cast<int>(p->tokens);
    a.slots = p->slots;
    a.ck = c.k;
    a.cv = c.v;
    a.scale_k = c.scale_k;
    a.scale_v = c.scale_v;
    a.num_slots = static_cast<long long>(c.num_pages * c.page_size);
    a.page_stride = c.page_stride;
    a.token_stride = c.token_stride;
    a.head_stride = c.head_stride;
    a.page = make_fast_div(static_cast<uint32_t>(c.page_size));
    const bool k_fits = set_norm(a.k_norm, k_norm);
    const bool q_fits = set_norm(a.q_norm, p->q_heads > 0 ? q_norm : nullptr);
    const bool vec =
        k_fits && q_fits && p->map.rotary_dim % 16 == 0 && aligned16(p->map.table) &&
        on_grid(p->K, p->k_token_stride, p->k_head_stride, sizeof(SRC)) &&
        on_grid(p->V, p->v_token_stride, p->v_head_stride, sizeof(SRC)) &&
        (p->q_heads == 0 || (on_grid(p->Q, p->q_token_stride, p->q_head_stride, sizeof(SRC)) &&
                             on_grid(p->Q_out, p->qo_token_stride, p->qo_head_stride, sizeof(DST))));
    launch_rows<SRC, DST, CACHE, kNorm>(a, vec, stream, where);
    return true;
}

}  // namespace
}  // namespace tqt
