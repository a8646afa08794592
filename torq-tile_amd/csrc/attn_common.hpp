// What the attention kernels over a paged cache share: a call's arguments, how a sequence and a key are
// found, the matrix instructions and conversions of the two 16-bit types.
#pragma once

#include <type_traits>

#include "attn_route.hpp"
#include "fast_div.hpp"
#include "paged_kv.hpp"
#include "tqt_hip_common.hpp"

namespace tqt {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct AttnArgs
{
    const void *q;
    void *d;
    float *lse;
    long long q_ts, q_hs, d_ts, d_hs;
    const int32_t *q_start, *kv_len, *table;
    long long ld_table;
    const void *k, *v;
    const float *scale_k, *scale_v;
    long long page_stride, token_stride, head_stride;
    int num_pages;
    FastDiv page, group;  // group: query heads per key head
    int batch, q_tokens, q_heads, kv_heads, head_dim, max_q_len, max_kv_len;
    // Scores are q . k times `scale` > 0, which holds log2(e) too; `sign` (-1, 0 or 1, times Q) is the
    // sign of the caller's scale.
    float scale, sign;
    int causal, window;  // window 0: none
    int few_rows;  // sequences of at most so many rows to a key head are the few-row kernel's
    // Parts of rows whose keys several workgroups have, in the workspace: f32 sums not divided by the sum of
    // probabilities, and (maximum in log2, sum). The few-row kernel's come first: workgroup w's are 2 w (of a
    // sequence that began before its run) and 2 w + 1 (of one that ends after it), kAttnFewRows rows each;
    // then the tile kernel's, [split][row of Q][query head], each of tile_chunk keys.
    float *part_o;   // [][head_dim]
    float *part_ml;  // [][2]
    int few_workgroups, tile_chunk, tile_rows;
};

// A sequence of the batch, with every length brought inside what the host checked.
struct AttnSeq
{
    int first;   // its first row of Q
    int q_len, kv_len;
    int nq;      // queries that are computed
    int pos0;    // position of query 0 (negative: the first queries see nothing)
};

__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, int b)
{
    AttnSeq s;
    s.first = min(max(a.q_start[b], 0), a.q_tokens);
    const int end = min(max(a.q_start[b + 1], s.first), a.q_tokens);
    s.q_len = end - s.first;
    s.kv_len = min(max(a.kv_len[b], 0), a.max_kv_len);
    s.nq = min(s.q_len, a.max_q_len);
    s.pos0 = s.kv_len - s.q_len;
    return s;
}

// One lane's sequence for the whole wave.
__device__ __forceinline__ AttnSeq attn_pick(const AttnSeq &x, int at)
{
    AttnSeq s;
    s.first = __builtin_amdgcn_readlane(x.first, at);
    s.q_len = __builtin_amdgcn_readlane(x.q_len, at);
    s.kv_len = __builtin_amdgcn_readlane(x.kv_len, at);
    s.nq = __builtin_amdgcn_readlane(x.nq, at);
    s.pos0 = __builtin_amdgcn_readlane(x.pos0, at);
    return s;
}

// The keys [lo, hi) that the query at `pos` may see.
__device__ __forceinline__ void attn_bounds(const AttnArgs &a, const AttnSeq &s, int pos, int &lo, int &hi)
{
    hi = a.causal ? min(max(pos + 1, 0), s.kv_len) : s.kv_len;
    lo = attn_first_key(pos, a.window);
}

// Workgroups that share the keys [first, last) of some rows.
__device__ __forceinline__ int attn_splits(int first, int last, int chunk)
{
    return last > first ? (last - first - 1) / chunk + 1 : 1;
}

// The keys that a tile of `m` rows may see, from a multiple of 64 on.
__device__ __forceinline__ void attn_tile_span(const AttnArgs &a, const AttnSeq &s, int tile, int m, int &first,
                                               int &last)
{
    int unused;
    const int end = min((tile + 1) * m, s.nq * static_cast<int>(a.group.d)) - 1;
    attn_bounds(a, s, s.pos0 + static_cast<int>(fast_div(tile * m, a.group)), first, unused);
    attn_bounds(a, s, s.pos0 + static_cast<int>(fast_div(end, a.group)), unused, last);
    first &= ~63;
}

// N elements of a row's sums from d0 on (d0 + N <= head_dim or d0 >= head_dim): the result where one
// workgroup has all of its keys (part < 0), else a part. sum == 0: no key, or scores of -infinity alone.
template <typename T, int N>
__device__ __forceinline__ void attn_put(const AttnArgs &a, long long part, int token, int head, int d0,
                                         const float (&acc)[N], float m, float sum)
{
    if (part >= 0) {
        if (d0 < a.head_dim) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                a.part_o[part * a.head_dim + d0 + e] = acc[e];
            }
        }
        if (d0 == 0) {
            a.part_ml[2 * part] = m;
            a.part_ml[2 * part + 1] = sum;
        }
        return;
    }
    if (d0 < a.head_dim) {
        typedef T out_vec __attribute__((ext_vector_type(N)));
        out_vec y;
        const float inv = 1.0f / sum;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            y[e] = static_cast<T>(sum == 0.0f ? 0.0f : acc[e] * inv);
        }
        *reinterpret_cast<out_vec *>(static_cast<T *>(a.d) + token * a.d_ts + head * a.d_hs + d0) = y;
    }
    if (a.lse != nullptr && d0 == 0) {
        a.lse[static_cast<long long>(token) * a.q_heads + head] =
            (m + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
    }
}

// The few-row kernel's work of one sequence: the keys [first, last) that its rows see, in units.
struct FewRowWork
{
    int first, last, units;  // units of one key head; 0: the sequence is not the few-row kernel's
};

__device__ __forceinline__ FewRowWork few_row_work(const AttnArgs &a, const AttnSeq &s)
{
    FewRowWork w;
    int unused;
    attn_bounds(a, s, s.pos0, w.first, unused);
    attn_bounds(a, s, s.pos0 + s.nq - 1, unused, w.last);
    const int rows = s.nq * static_cast<int>(a.group.d);
    w.units = rows == 0 || rows > a.few_rows ? 0 : attn_splits(w.first, w.last, kAttnFewRowUnit);
    return w;
}

// Sum of the lanes up to and with this one, of which those from n on hold 0 (and lane 63 the total).
__device__ __forceinline__ int wave_inclusive_sum(int x, int lane, int n)
{
    n = min(n, 64);
    for (int off = 1; off < n; off <<= 1) {
        const int y = __shfl_up(x, off);
        x += lane >= off ? y : 0;
    }
    return lane < n ? x : __builtin_amdgcn_readlane(x, n - 1);
}

// The few-row kernel's units of all sequences in order, each times kv_heads. A wave holds 64 sequences at a
// time, one a lane.
struct FewRowBatch
{
    AttnSeq s;       // sequence b0 + lane
    FewRowWork work;
    int b0;
    int upto;        // units of sequences up to and with this lane's
};

__device__ __forceinline__ void few_row_batch(const AttnArgs &a, int b0, int before, int lane, FewRowBatch &x)
{
    const bool in = b0 + lane < a.batch;
    x.s = attn_seq(a, in ? b0 + lane : 0);
    x.work = few_row_work(a, x.s);
    x.b0 = b0;
    x.upto = before + wave_inclusive_sum(in ? x.work.units * a.kv_heads : 0, lane, a.batch - b0);
}

// Units of a workgroup's run (all lanes of a wave call this); leaves the last 64 sequences in x.
__device__ __forceinline__ int few_row_run(const AttnArgs &a, int lane, int &total, FewRowBatch &x)
{
    total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        few_row_batch(a, b0, total, lane, x);
        total = __shfl(x.upto, 63);
    }
    return (total + a.few_workgroups - 1) / a.few_workgroups;
}

// One lane's sequence and work for the whole wave.
__device__ __forceinline__ void few_row_pick(const FewRowBatch &x, int at, AttnSeq &s, FewRowWork &w)
{
    s = attn_pick(x.s, at);
    w.first = __builtin_amdgcn_readlane(x.work.first, at);
    w.last = __builtin_amdgcn_readlane(x.work.last, at);
    w.units = __builtin_amdgcn_readlane(x.work.units, at);
}

// 512 zero bytes: a row of keys that are not there.
__device__ const u32x4 kAttnZeros[32] = {};

// Where a key's row of one key head is: its element offset, its page and the offset in it. Not kept: past the keys
// that are asked for, or on no page of the cache (then at is 0 and not read).
struct KeyRow
{
    long long at;
    int page, offset;
    bool kept;
};

// A key's page, asked for: the entry is on its way and nothing waits for it yet.
struct PageAsked
{
    int page, offset;
};

// For a key below the sequence's length.
__device__ __forceinline__ PageAsked attn_page_of(const AttnArgs &a, const int32_t *table, int j)
{
    uint32_t offset;
    const int page = table[fast_div(static_cast<uint32_t>(j), a.page, offset)];
    return {page, static_cast<int>(offset)};
}

__device__ __forceinline__ PageAsked attn_ask_page(const AttnArgs &a, const int32_t *table, int j, int hi)
{
    PageAsked r;
    uint32_t offset;
    const uint32_t pi = fast_div(static_cast<uint32_t>(j), a.page, offset);
    r.page = j < hi ? table[pi] : -1;
    r.offset = static_cast<int>(offset);
    return r;
}

__device__ __forceinline__ KeyRow attn_key(const AttnArgs &a, PageAsked p, int head)
{
    KeyRow r;
    r.page = p.page;
    r.offset = p.offset;
    r.kept = r.page >= 0 && r.page < a.num_pages;
    r.at = r.kept ? r.page * a.page_stride + r.offset * a.token_stride + head * a.head_stride : 0;
    return r;
}

__device__ __forceinline__ KeyRow attn_key(const AttnArgs &a, const int32_t *table, int head, int j, int hi)
{
    return attn_key(a, attn_ask_page(a, table, j, hi), head);
}

// 8 values of a 16-bit type as a matrix operand, and the two shapes of product used.
template <typename T>
struct Half8;
template <>
struct Half8<_Float16>
{
    typedef f16x8 type;
};
template <>
struct Half8<__bf16>
{
    typedef bf16x8 type;
};

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Four rows of a 16-bit matrix in LDS, read down a column: the 16 lanes of a group give the addresses of
// 4 rows x 16 columns (lane i: row i / 4, columns 4 (i % 4) ..) and lane i receives column i.
__device__ __forceinline__ u32x2 lds_read_column4(const void *p)
{
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)p));
}

// Orders a wave's own LDS writes before other lanes' reads of them (a wave's LDS operations complete in
// order; this holds the compiler to it).
__device__ __forceinline__ void wave_lds_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The larger of this lane's value and that of lane ^ 32. The swap is inline asm: with the builtin the compiler
// drops the maximum of its two results (each lane then has the lower half's value). Two wait states lie
// between a vector instruction's write and the swap.
__device__ __forceinline__ float max_across_halves(float x)
{
    float y = x;
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
#endif
    return fmaxf(x, y);
}

// Int8 values: the probability e = 2^(s - ref) of a key goes to the second product times its value's scale, in f16.
// `ref` follows a row's largest such term, not its largest score: it is the maximum of s + log2 |scale| over the
// keys that the row sees, less kValueLogUp. So no key that a row does not see changes its bits, and the largest
// term is 2^7 (2^28 down by 2^21): 2^-1 where the maximum is bounded from above by 2^8 (attn_tile.hpp), 2^15
// where ref follows it by steps of 2^8, below f16's 65504. Terms 2^13 times smaller than the largest, or more,
// keep all of f16's bits. What e (2^96 at most, of up to 2^30 keys) and its sums need of f32's range is what the
// constants leave: scales from 2^-60 up, those below losing bits as f16's subnormals do.
constexpr float kValueLogUp = 28.0f, kValueLogFloor = -60.0f;
constexpr float kValueLogLeast = kValueLogFloor - kValueLogUp;
constexpr float kValueDown = 0x1p-21f, kValueUp = 0x1p21f;

// What is kept of a value's scale: the factor of its key's e, and the summand of its score in the maximum. A row of
// zeros has a scale that says nothing (the append gives it 1): it counts as the smallest one. A scale that is no
// number makes the maximum infinite, which makes the rows that see the key NaN; its factor is 0, so that rows
// that do not see it take nothing from it.
struct ValueScale
{
    float factor, log;
};

__device__ __forceinline__ ValueScale value_scale(float scale, bool zeros)
{
    const float size = __builtin_fabsf(scale);
    const bool finite = size < INFINITY;  // false for a NaN
    ValueScale v;
    v.factor = finite && !zeros ? scale * kValueDown : 0.0f;
    v.log = fmaxf(__builtin_amdgcn_logf(zeros ? 0.0f : size), kValueLogFloor) - kValueLogUp;
    v.log = finite ? v.log : INFINITY;
    return v;
}

// What the sums so far are multiplied by when `ref` becomes `base`: `half` twice. In one factor it could
// leave f32's range where the sum does not (scales more than 2^126 apart). ref == base: 1.
__device__ __forceinline__ float value_half_step(float ref, float base)
{
    return __builtin_amdgcn_exp2f(0.5f * (ref - base));
}

// A part's sums times 2^(m - base): over int8 caches the sum of probabilities in two steps, as its reference may
// be further off than f32's range (value_half_step).
template <bool kQuant>
__device__ __forceinline__ float part_factor(float m, float base, float &sum)
{
    if constexpr (kQuant) {
        const float half = value_half_step(m, base);
        sum = sum * half * half;
        return half * half;
    } else {
        const float f = __builtin_amdgcn_exp2f(m - base);
        sum *= f;
        return f;
    }
}

// 16 int8 as 16-bit floats, exactly: [0] the first 8, [1] the others.
__device__ __forceinline__ void int8_to_half(u32x4 x, f16x8 (&y)[2])
{
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // value + 128 in the low bits of 1024.0's significand, then less 1152
        const uint32_t u = x[i] ^ 0x80808080u;
        const f16x2 base = {1152.0f16, 1152.0f16};
        w[2 * i] = __builtin_bit_cast(
            uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - base);
        w[2 * i + 1] = __builtin_bit_cast(
            uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - base);
    }
    __builtin_memcpy(&y[0], w, 16);
    __builtin_memcpy(&y[1], w + 4, 16);
}

__device__ __forceinline__ void int8_to_half(u32x4 x, bf16x8 (&y)[2])
{
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = static_cast<float>(static_cast<int8_t>(x[i] >> (8 * j)));
        }
        // whole numbers of 8 bits: the upper halves of the f32 hold them
        w[2 * i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[1]),
                                         __builtin_bit_cast(uint32_t, f[0]), 0x07060302u);
        w[2 * i + 1] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[3]),
                                             __builtin_bit_cast(uint32_t, f[2]), 0x07060302u);
    }
    __builtin_memcpy(&y[0], w, 16);
    __builtin_memcpy(&y[1], w + 4, 16);
}

// Whether any of 2 packed 16-bit values is an infinity or NaN (exponent bits all set).
template <typename T>
__device__ __forceinline__ bool any_not_finite(uint32_t x)
{
    constexpr uint32_t mask = std::is_same<T, _Float16>::value ? 0x7c00u : 0x7f80u;
    return (x & mask) == mask || ((x >> 16) & mask) == mask;
}

// Values that are no numbers, in a tile where some rows do not see some keys: 0 x infinity would reach
// them through the matrix product. The product takes 0 in their place (`clean`), and a second one, of
// `code` with 1 for every key a row sees, tells which of them each row meets: counts of +infinity,
// -infinity and NaN in steps of 1, 64 and 4096, which 32 keys do not overflow.
template <typename T>
__device__ __forceinline__ void split_not_finite(u32x4 x, u32x4 &clean, u32x4 &code)
{
    constexpr bool f16 = std::is_same<T, _Float16>::value;
    constexpr uint32_t mask = f16 ? 0x7c00u : 0x7f80u, mant = f16 ? 0x3ffu : 0x7fu;
    constexpr uint32_t one = f16 ? 0x3c00u : 0x3f80u, c64 = f16 ? 0x5400u : 0x4280u,
                       c4096 = f16 ? 0x6c00u : 0x4580u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        clean[i] = 0;
        code[i] = 0;
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
            const uint32_t v = (x[i] >> h) & 0xffffu;
            const bool bad = (v & mask) == mask;
            clean[i] |= (bad ? 0u : v) << h;
            code[i] |= (!bad ? 0u : (v & mant) ? c4096 : (v & 0x8000u) ? c64 : one) << h;
        }
    }
}

// What a row's sum becomes by the values that are no numbers it meets.
__device__ __forceinline__ float not_finite_term(float count)
{
    const int n = static_cast<int>(count);
    float t = 0.0f;
    if (n >= 4096) {
        t = __builtin_nanf("");
    }
    if ((n & 4095) >= 64) {
        t -= INFINITY;
    }
    if ((n & 63) > 0) {
        t += INFINITY;
    }
    return t;
}

}  // namespace tqt
