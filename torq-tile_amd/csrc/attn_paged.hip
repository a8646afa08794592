// Attention of new tokens over a paged cache on gfx950: the entry points and their checks.
#include "attn_common.hpp"
#include "attn_few_row.hpp"
#include "attn_join.hpp"
#include "tqt_attn_paged_gfx950.h"

#include <cmath>
#include <type_traits>

namespace tqt {
namespace {

// One wave per row: lanes along the head, keys one after another with the running maximum and sum.
template <typename T, typename C>
__global__ __launch_bounds__(256) void attn_row_kernel(AttnArgs a)
{
    const int lane = threadIdx.x & 63;
    const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (item >= static_cast<long long>(a.q_tokens) * a.q_heads) {
        return;
    }
    const int token = static_cast<int>(item / a.q_heads), head = static_cast<int>(item % a.q_heads);
    int b = 0;
    while (b < a.batch && a.q_start[b + 1] <= token) {
        ++b;
    }
    if (b == a.batch || token < a.q_start[b]) {
        return;
    }
    const AttnSeq s = attn_seq(a, b);
    const int i = token - s.first;
    if (i >= a.max_q_len || s.nq * static_cast<int>(a.group.d) <= kAttnFewRows) {
        return;
    }
    int lo, hi;
    attn_bounds(a, s, s.pos0 + i, lo, hi);
    const int kvh = fast_div(head, a.group);
    float q[4], o[4], m = -INFINITY, l = 0.0f;
    const T *qp = static_cast<const T *>(a.q) + token * a.q_ts + head * a.q_hs;
    for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        q[e] = d < a.head_dim ? static_cast<float>(qp[d]) * a.sign : 0.0f;
        o[e] = 0.0f;
    }
    for (int j = lo; j < hi; ++j) {
        uint32_t offset;
        const uint32_t pi = fast_div(j, a.page, offset);
        const int page = a.table[b * a.ld_table + pi];
        if (page < 0 || page >= a.num_pages) {
            continue;
        }
        const long long at = page * a.page_stride + offset * a.token_stride + kvh * a.head_stride;
        const C *kp = static_cast<const C *>(a.k) + at, *vp = static_cast<const C *>(a.v) + at;
        float dot = 0.0f;
        for (int e = 0; e < 4; ++e) {
            const int d = lane + 64 * e;
            dot += d < a.head_dim ? q[e] * static_cast<float>(kp[d]) : 0.0f;
        }
        for (int off = 32; off > 0; off >>= 1) {
            dot += __shfl_xor(dot, off);
        }
        float vs = 1.0f;
        if (std::is_same<C, int8_t>::value) {
            const long long sc = (static_cast<long long>(page) * a.kv_heads + kvh) * a.page.d + offset;
            dot *= a.scale_k[sc];
            vs = a.scale_v[sc];
        }
        dot *= a.scale;
        const float mn = dot > m ? dot : m;
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float alpha = exp2f(m - base), p = exp2f(dot - base);
        l = l * alpha + p;
        m = mn;
        for (int e = 0; e < 4; ++e) {
            const int d = lane + 64 * e;
            o[e] = o[e] * alpha + (d < a.head_dim ? p * vs * static_cast<float>(vp[d]) : 0.0f);
        }
    }
    T *dp = static_cast<T *>(a.d) + token * a.d_ts + head * a.d_hs;
    for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        if (d < a.head_dim) {
            dp[d] = static_cast<T>(l == 0.0f ? 0.0f : o[e] / l);
        }
    }
    if (a.lse != nullptr && lane == 0) {
        a.lse[static_cast<long long>(token) * a.q_heads + head] = (m + log2f(l)) * 0.69314718f;
    }
}

bool attn_empty(const tqt_attn_paged_params *p)
{
    return p->batch == 0 || p->q_tokens == 0 || p->q_heads == 0 || p->max_q_len == 0;
}

// The checks that the sizes alone decide.
const char *attn_size_error(const tqt_attn_paged_params *p)
{
    const size_t top = 1u << 31;
    if (p->batch >= (1u << 16) || p->q_tokens >= top || p->q_heads >= (1u << 16) || p->max_q_len >= top ||
        p->max_kv_len >= top || p->ld_table >= top || p->q_tokens * p->q_heads >= top) {
        return "batch, q_tokens, q_heads, max_q_len, max_kv_len or ld_table too large";
    }
    if (p->kv.head_dim == 0 || p->kv.kv_heads == 0 || p->q_heads % p->kv.kv_heads != 0) {
        return "q_heads % kv_heads != 0";
    }
    if (p->max_q_len * (p->q_heads / p->kv.kv_heads) >= top) {
        return "max_q_len * (q_heads / kv_heads) exceeds 2^31-1";
    }
    return nullptr;
}

const char *attn_error(const tqt_attn_paged_params *p, size_t cache_bytes, bool quant)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    if (attn_empty(p)) {
        return nullptr;
    }
    if (const char *e = paged_kv_error(p->kv, cache_bytes, quant)) {
        return e;
    }
    if (const char *e = attn_size_error(p)) {
        return e;
    }
    if (p->max_kv_len > p->ld_table * p->kv.page_size) {
        return "max_kv_len > ld_table * page_size";
    }
    if (p->Q == nullptr || p->D == nullptr || p->q_start == nullptr || p->kv_len == nullptr ||
        (p->block_table == nullptr && p->max_kv_len > 0)) {
        return "Q / D / q_start / kv_len / block_table == NULL";
    }
    if (!aligned16(p->Q) || !aligned16(p->D) || p->q_token_stride % 8 != 0 || p->q_head_stride % 8 != 0 ||
        p->d_token_stride % 8 != 0 || p->d_head_stride % 8 != 0) {
        return "rows of Q or D are off the 16-byte grid";
    }
    if (!std::isfinite(p->scale)) {
        return "scale is not finite";
    }
    if (p->window > 0 && p->causal == 0) {
        return "a window needs causal";
    }
    const size_t need = tqt_get_workspace_size_attn_paged_gfx950(p);
    if (p->workspace_size < need || (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace)))) {
        return "the workspace is too small or off the 16-byte grid";
    }
    return nullptr;
}

// What a call launches, from its sizes (which have been checked).
struct AttnPlan
{
    bool run_few, run_tile;
    AttnSplit few;
    int splits;      // of the kernel that has more
    long long rows;  // of Q, times query heads
};

AttnPlan attn_plan(const tqt_attn_paged_params *p)
{
    AttnPlan plan;
    const long long group = p->q_heads / p->kv.kv_heads;
    const long long window = static_cast<long long>(std::min<size_t>(p->window, 1u << 31));
    plan.rows = static_cast<long long>(p->q_tokens) * p->q_heads;
    plan.run_few = group <= kAttnFewRows;
    plan.run_tile = static_cast<long long>(p->max_q_len) * group > kAttnFewRows;
    const long long few_q = std::min<long long>(p->max_q_len, std::max(1ll, kAttnFewRows / group));
    plan.few = attn_few_row_split(p->batch, p->kv.kv_heads, attn_span(few_q, p->max_kv_len, window));
    plan.splits = plan.run_few ? plan.few.splits : 1;
    return plan;
}

template <typename T, typename C>
bool run_attn(const tqt_attn_paged_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = attn_error(p, sizeof(C), std::is_same<C, int8_t>::value);
    TQT_REQUIRE(error == nullptr, error);
    if (attn_empty(p)) {
        return false;
    }
    AttnArgs a = {};
    a.q = p->Q;
    a.d = p->D;
    a.lse = p->lse;
    a.q_ts = p->q_token_stride;
    a.q_hs = p->q_head_stride;
    a.d_ts = p->d_token_stride;
    a.d_hs = p->d_head_stride;
    a.q_start = p->q_start;
    a.kv_len = p->kv_len;
    a.table = p->block_table;
    a.ld_table = p->ld_table;
    a.k = p->kv.k;
    a.v = p->kv.v;
    a.scale_k = p->kv.scale_k;
    a.scale_v = p->kv.scale_v;
    a.page_stride = p->kv.page_stride;
    a.token_stride = p->kv.token_stride;
    a.head_stride = p->kv.head_stride;
    a.num_pages = static_cast<int>(p->kv.num_pages);
    a.page = make_fast_div(static_cast<uint32_t>(p->kv.page_size));
    a.group = make_fast_div(static_cast<uint32_t>(p->q_heads / p->kv.kv_heads));
    a.batch = static_cast<int>(p->batch);
    a.q_tokens = static_cast<int>(p->q_tokens);
    a.q_heads = static_cast<int>(p->q_heads);
    a.kv_heads = static_cast<int>(p->kv.kv_heads);
    a.head_dim = static_cast<int>(p->kv.head_dim);
    a.max_q_len = static_cast<int>(p->max_q_len);
    a.max_kv_len = static_cast<int>(p->max_kv_len);
    a.sign = p->scale > 0.0f ? 1.0f : p->scale < 0.0f ? -1.0f : 0.0f;
    a.scale = p->scale == 0.0f ? 1.0f : std::fabs(p->scale) * 1.4426950408889634f;
    a.causal = p->causal != 0;
    // a window past every length is none
    a.window = p->window < (1u << 31) ? static_cast<int>(p->window) : 0;
    const AttnPlan plan = attn_plan(p);
    a.few_chunk = plan.few.chunk;
    a.part_o = static_cast<float *>(p->workspace);
    a.part_ml = a.part_o + plan.rows * plan.splits * a.head_dim;
    if (plan.run_few) {
        const dim3 grid(plan.few.splits, a.kv_heads, a.batch);
        if (a.head_dim <= 64) {
            hipLaunchKernelGGL((attn_few_row_kernel<T, C, 64>), grid, dim3(256), 0, stream, a);
        } else if (a.head_dim <= 128) {
            hipLaunchKernelGGL((attn_few_row_kernel<T, C, 128>), grid, dim3(256), 0, stream, a);
        } else {
            hipLaunchKernelGGL((attn_few_row_kernel<T, C, 256>), grid, dim3(256), 0, stream, a);
        }
        check_launch(where);
    }
    if (plan.run_tile) {
        const long long rows = static_cast<long long>(a.q_tokens) * a.q_heads;
        hipLaunchKernelGGL((attn_row_kernel<T, C>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256),
                           0, stream, a);
        check_launch(where);
    }
    if (plan.splits > 1) {
        hipLaunchKernelGGL((attn_join_kernel<T>), dim3(a.q_tokens, a.q_heads), dim3(256), 0, stream, a);
    }
    check_launch(where);
    return true;
}

}  // namespace
}  // namespace tqt

using namespace tqt;

extern "C" {

size_t tqt_get_workspace_size_attn_paged_gfx950(const struct tqt_attn_paged_params *params)
{
    if (params == nullptr || attn_size_error(params) != nullptr || attn_empty(params)) {
        return 0;
    }
    const AttnPlan plan = attn_plan(params);
    // a part of every row and split: its sums, its maximum and its sum of probabilities
    return plan.splits > 1 ? static_cast<size_t>(plan.rows) * plan.splits * (params->kv.head_dim + 2) * 4 : 0;
}

#define TQT_ATTN_ENTRIES(NAME, T, C)                                                                  \
    const char *tqt_get_error_attn_paged_##NAME##_gfx950(const struct tqt_attn_paged_params *params)  \
    {                                                                                                 \
        return attn_error(params, sizeof(C), std::is_same<C, int8_t>::value);                         \
    }                                                                                                 \
    void tqt_run_attn_paged_##NAME##_gfx950_async(const struct tqt_attn_paged_params *params,         \
                                                  void *stream)                                       \
    {                                                                                                 \
        run_attn<T, C>(params, as_stream(stream), "tqt_run_attn_paged_" #NAME "_gfx950");             \
    }                                                                                                 \
    void tqt_run_attn_paged_##NAME##_gfx950(const struct tqt_attn_paged_params *params)               \
    {                                                                                                 \
        if (run_attn<T, C>(params, nullptr, "tqt_run_attn_paged_" #NAME "_gfx950")) {                 \
            finish_sync(nullptr, "tqt_run_attn_paged_" #NAME "_gfx950");                              \
        }                                                                                             \
    }

TQT_ATTN_ENTRIES(f16_f16, _Float16, _Float16)
TQT_ATTN_ENTRIES(bf16_bf16, __bf16, __bf16)
TQT_ATTN_ENTRIES(f16_qsi8dx, _Float16, int8_t)
TQT_ATTN_ENTRIES(bf16_qsi8dx, __bf16, int8_t)

}  // extern "C"
