// Rotary positions and the append of keys and values to a paged cache on gfx950.
//
//   y1 = x1 c - x2 s, y2 = x2 c + x1 s   for pairs (i, i + r / 2) or (2 i, 2 i + 1), i < r / 2
//
// with (c, s) of the token's position from a table, every product and sum in f32 rounded on its own (the
// library is built with -ffp-contract=off) and one rounding to the result's type. Bound by memory: each
// element is read once and written once; the table row of a token (4 r bytes) is shared by its heads.
//
// Split: one thread takes 16 elements of a head, the 8 + 8 of 8 pairs, as two 16-byte pieces (four for f32
// sources), so that a pair never crosses threads and the operation works in place. Threads of a token lie
// along its heads, so the 64 bytes of the table that a thread reads come from its CU's cache for all but the
// first of them (four heads a thread, which share them in registers, took 16.9 instead of 14.2 us for 1000
// tokens of 96 int8 heads and 26.6 instead of 24.2 for 4096 of 48 from f32: fewer waves have loads in flight).
#include "fast_div.hpp"
#include "paged_kv.hpp"
#include "rope_route.hpp"
#include "tqt_hip_common.hpp"
#include "tqt_kv_append_rope_gfx950.h"

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
};

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
// for rope alone.
template <typename SRC, typename DST, typename CACHE>
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
    // an int8 head has a power of two of threads, some of them past its end
    const bool on = live && static_cast<int>(16 * unit) < a.head_dim && (query || slot.used);
    f32x8 xa = 0.0f, xb = 0.0f;
    if (on) {
        const SRC *x = query ? static_cast<const SRC *>(a.q) + token * a.q_ts + head * a.q_hs
                             : (value ? static_cast<const SRC *>(a.v) + token * a.v_ts + head * a.v_hs
                                      : static_cast<const SRC *>(a.k) + token * a.k_ts + head * a.k_hs);
        xa = __builtin_convertvector(*reinterpret_cast<const src8 *>(x + ea), f32x8);
        xb = __builtin_convertvector(*reinterpret_cast<const src8 *>(x + eb), f32x8);
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
template <typename SRC, typename DST, typename CACHE>
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
            const float p = static_cast<float>(x[e1]), q = static_cast<float>(x[e2]);
            const float c = t ? t[i] : __builtin_nanf("");
            const float s = (t ? t[half + i] : __builtin_nanf("")) * a.sign;
            put(e1, p * c - q * s);
            put(e2, q * c + p * s);
        }
        for (int e = r + lane; e < a.head_dim; e += 64) {
            put(e, static_cast<float>(x[e]));
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

// Launches the rows of all tokens. grid16: they suit rope_rows_kernel.
template <typename SRC, typename DST, typename CACHE>
void launch_rows(RopeArgs a, bool grid16, hipStream_t stream, const char *where)
{
    const RopeLaunch r = rope_launch(a.rows, a.head_dim, grid16, std::is_same<CACHE, int8_t>::value);
    a.units = make_fast_div(static_cast<uint32_t>(r.per_head));
    a.heads = make_fast_div(a.rows);
    for (long long t0 = 0; t0 < a.tokens; t0 += r.tokens) {
        const long long n = std::min(r.tokens, a.tokens - t0);
        const uint32_t items = static_cast<uint32_t>(n * a.rows * r.per_head);
        const int per_block = r.rows ? kRopeThreads : kRopeThreads / 64;
        const dim3 grid((items + per_block - 1) / per_block);
        if (r.rows) {
            hipLaunchKernelGGL((rope_rows_kernel<SRC, DST, CACHE>), grid, dim3(kRopeThreads), 0, stream, a,
                               static_cast<int>(t0), items);
        } else {
            hipLaunchKernelGGL((rope_any_kernel<SRC, DST, CACHE>), grid, dim3(kRopeThreads), 0, stream, a,
                               static_cast<int>(t0), items);
        }
        check_launch(where);
    }
}

template <typename T>
bool run_rope(const tqt_rope_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = rope_error(p);
    TQT_REQUIRE(error == nullptr, error);
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
    const bool vec = p->head_dim % 16 == 0 && p->map.rotary_dim % 16 == 0 && aligned16(p->map.table) &&
                     on_grid(p->X, p->x_token_stride, p->x_head_stride, sizeof(T)) &&
                     on_grid(p->Y, p->y_token_stride, p->y_head_stride, sizeof(T));
    launch_rows<T, T, void>(a, vec, stream, where);
    return true;
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

template <typename SRC, typename DST, typename CACHE>
bool run_append(const tqt_kv_append_rope_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = append_error(p, sizeof(CACHE), std::is_same<CACHE, int8_t>::value);
    TQT_REQUIRE(error == nullptr, error);
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
    const bool vec =
        p->map.rotary_dim % 16 == 0 && aligned16(p->map.table) &&
        on_grid(p->K, p->k_token_stride, p->k_head_stride, sizeof(SRC)) &&
        on_grid(p->V, p->v_token_stride, p->v_head_stride, sizeof(SRC)) &&
        (p->q_heads == 0 || (on_grid(p->Q, p->q_token_stride, p->q_head_stride, sizeof(SRC)) &&
                             on_grid(p->Q_out, p->qo_token_stride, p->qo_head_stride, sizeof(DST))));
    launch_rows<SRC, DST, CACHE>(a, vec, stream, where);
    return true;
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
        run_rope<T>(params, as_stream(stream), "tqt_run_rope_" #NAME "_gfx950");                      \
    }                                                                                                 \
    void tqt_run_rope_##NAME##_gfx950(const struct tqt_rope_params *params)                           \
    {                                                                                                 \
        if (run_rope<T>(params, nullptr, "tqt_run_rope_" #NAME "_gfx950")) {                          \
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
        run_append<SRC, DST, CACHE>(params, as_stream(stream),                                        \
                                    "tqt_run_kv_append_rope_" #NAME "_gfx950");                       \
    }                                                                                                 \
    void tqt_run_kv_append_rope_##NAME##_gfx950(const struct tqt_kv_append_rope_params *params)       \
    {                                                                                                 \
        if (run_append<SRC, DST, CACHE>(params, nullptr, "tqt_run_kv_append_rope_" #NAME "_gfx950")) { \
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
