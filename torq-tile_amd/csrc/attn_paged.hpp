// Attention of new tokens over a paged cache on gfx950: the checks of a call, what it launches, and the entry
// points of one type (each in a file of its own: the kernels' instances take the compiler a minute).
#pragma once

#include "attn_common.hpp"
#include "attn_few_row.hpp"
#include "attn_join.hpp"
#include "attn_tile.hpp"
#include "tqt_attn_tree_gfx950.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tqt {
namespace {

bool attn_empty(const tqt_attn_paged_params *p)
{
    return p->batch == 0 || p->q_tokens == 0 || p->q_heads == 0 || p->max_q_len == 0;
}

// What scores are multiplied by for powers of 2.
float attn_log2_scale(float scale)
{
    return std::fabs(scale) * 1.4426950408889634f;
}

// The checks that the sizes alone decide.
const char *attn_size_error(const tqt_attn_paged_params *p)
{
    const size_t top = 1u << 31;
    if (p->batch >= (1u << 16) || p->q_tokens >= top || p->q_heads >= (1u << 16) || p->max_q_len >= top ||
        p->max_kv_len >= top / 2 || p->ld_table >= top || p->q_tokens * p->q_heads >= top) {
        return "batch, q_tokens, q_heads, max_q_len, max_kv_len or ld_table too large";
    }
    if (p->kv.head_dim == 0 || p->kv.kv_heads == 0 || p->q_heads % p->kv.kv_heads != 0) {
        return "q_heads % kv_heads != 0";
    }
    const size_t group = p->q_heads / p->kv.kv_heads;
    if (p->max_q_len * group >= top - 256) {
        return "max_q_len * (q_heads / kv_heads) too large";
    }
    // units of the few-row kernel in 32 bits, with the end of the last of up to 512 equal runs, which is up to 511
    // past theirs, and grids of fewer than 2^32 work-items
    if (p->batch * p->kv.kv_heads * (p->max_kv_len / kAttnFewRowUnit + 1) >= top - 512 ||
        p->batch * p->kv.kv_heads * kAttnFewRows >= (1u << 26)) {
        return "batch * kv_heads or batch * kv_heads * max_kv_len too large";
    }
    if (attn_tiles(p->batch, p->q_tokens, p->max_q_len, group) * static_cast<long long>(p->kv.kv_heads) >=
        (1 << 24)) {
        return "too many rows";
    }
    return nullptr;
}

// The checks of a call, `need` bytes of workspace apart.
const char *attn_call_error(const tqt_attn_paged_params *p, size_t cache_bytes, bool quant)
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
    if (!std::isfinite(attn_log2_scale(p->scale))) {
        return "scale times log2(e) is not finite";
    }
    if (p->window > 0 && p->causal == 0) {
        return "a window needs causal";
    }
    return nullptr;
}

const char *attn_space_error(const tqt_attn_paged_params *p, size_t need)
{
    if (p->workspace_size < need || (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace)))) {
        return "the workspace is too small or off the 16-byte grid";
    }
    return nullptr;
}

inline const char *attn_error(const tqt_attn_paged_params *p, size_t cache_bytes, bool quant)
{
    const char *e = attn_call_error(p, cache_bytes, quant);
    return e != nullptr || attn_empty(p) ? e : attn_space_error(p, tqt_get_workspace_size_attn_paged_gfx950(p));
}

inline const char *attn_tree_error(const tqt_attn_tree_params *p, size_t cache_bytes, bool quant)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    const char *e = attn_call_error(&p->attn, cache_bytes, quant);
    if (e != nullptr || attn_empty(&p->attn)) {
        return e;
    }
    if (p->attn.causal != 1) {
        return "trees need causal == 1";
    }
    if (p->mask == nullptr) {
        return "mask == NULL";
    }
    if (p->ld_mask >= (1u << 25) || p->ld_mask * 32 < p->attn.max_q_len) {
        return "ld_mask words hold fewer than max_q_len bits, or are too many";
    }
    // the join's grid, as in attn_size_error
    if (p->attn.batch * p->attn.kv.kv_heads * 32 >= (1u << 26)) {
        return "batch * kv_heads too large";
    }
    return attn_space_error(&p->attn, tqt_get_workspace_size_attn_tree_gfx950(p));
}

// What a call launches, from its sizes (which have been checked).
struct AttnPlan
{
    bool run_few, run_tile;
    int few_workgroups;    // 0: no few-row kernel
    int few_columns;       // of 16 rows
    bool few_whole;        // keys of a sequence and key head are not split
    bool few_many;         // parts for a row of the few-row kernel
    long long few_tokens;  // of a sequence of the few-row kernel, at most
    long long tiles;
    AttnSplit tile;
    int even_parts;   // trees: attn_even_parts
    long long span;   // keys that a row sees at most
    long long parts;  // rows of the workspace
};

// mask_bits: of a row, with trees, whose rows see the window before the context's end and all new tokens
// that have a bit; else 0.
AttnPlan attn_plan(const tqt_attn_paged_params *p, long long mask_bits = 0)
{
    const int head_dim = static_cast<int>(p->kv.head_dim);
    const int few_rows = mask_bits > 0 ? attn_few_rows<AttnTreeArgs>(head_dim) : kAttnFewRows;
    AttnPlan plan = {};
    const long long group = p->q_heads / p->kv.kv_heads;
    const long long window = static_cast<long long>(std::min<size_t>(p->window, 1u << 31));
    // where the bounds say that every sequence has max_q_len tokens, or there is one, its length decides;
    // a shorter one after all is the tile kernel's
    const bool alike = p->batch == 1 || p->q_tokens == p->batch * p->max_q_len;
    plan.run_few = group <= few_rows && (!alike || static_cast<long long>(p->max_q_len) * group <= few_rows);
    plan.run_tile = static_cast<long long>(p->max_q_len) * group > few_rows;
    plan.few_tokens = std::min<long long>(p->max_q_len, std::max(1ll, few_rows / group));
    if (plan.run_few) {
        plan.few_columns = static_cast<long long>(p->max_q_len) * group <= 16 ? 1 : few_rows / 16;
        const long long heads = static_cast<long long>(p->batch) * p->kv.kv_heads;
        const long long span = attn_span(mask_bits > 0 ? mask_bits + 1 : plan.few_tokens, p->max_kv_len, window);
        plan.few_whole = mask_bits > 0 && span <= attn_tree_whole(heads);
        plan.few_workgroups = attn_few_row_workgroups(
            heads * (plan.few_whole ? 1 : std::max(1ll, (span + kAttnFewRowUnit - 1) / kAttnFewRowUnit)),
            attn_few_row_per_cu(head_dim, plan.few_columns));
        plan.few_many = plan.few_workgroups > heads * kAttnJoinManyParts;
    }
    plan.tiles = attn_tiles(p->batch, p->q_tokens, p->max_q_len, group);
    plan.tile = attn_call_split(plan.tiles, p->kv.kv_heads,
                                attn_span(mask_bits > 0 ? mask_bits + 1
                                                        : std::min<long long>(p->max_q_len,
                                                                              kAttnTileRows / group + 2),
                                          p->max_kv_len, window),
                                static_cast<long long>(p->kv.head_dim),
                                static_cast<long long>(p->q_tokens * p->q_heads));
    plan.parts = plan.few_whole ? 0 : 2ll * plan.few_workgroups * few_rows;
    const long long rows = static_cast<long long>(p->q_tokens) * p->q_heads;
    if (plan.run_tile && mask_bits > 0) {
        plan.span = attn_span(mask_bits + 1, p->max_kv_len, window);
        plan.even_parts = attn_even_parts(p->batch, plan.tiles * p->kv.kv_heads, plan.tile, plan.span, head_dim, rows);
        plan.tile.splits = std::max(plan.tile.splits, plan.even_parts);
    }
    if (plan.run_tile && plan.tile.splits > 1) {
        // and 4 rows for the equal spans, 64 whole numbers
        plan.parts += plan.tile.splits * rows + (plan.even_parts > 0 ? 4 : 0);
    }
    return plan;
}

// Calls f with the first of the sizes that holds head_dim, and whether it is the head's own.
template <int kSize, int... kMore, typename F>
void by_head_dim(int head_dim, F f)
{
    if constexpr (sizeof...(kMore) > 0) {
        if (head_dim > kSize) {
            by_head_dim<kMore...>(head_dim, f);
            return;
        }
    }
    if (head_dim == kSize) {
        f(std::integral_constant<int, kSize>(), std::true_type());
    } else {
        f(std::integral_constant<int, kSize>(), std::false_type());
    }
}

// Everything of a call but what its plan says.
void set_attn(AttnArgs &a, const tqt_attn_paged_params *p)
{
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
    a.scale = p->scale == 0.0f ? 1.0f : attn_log2_scale(p->scale);
    a.causal = p->causal != 0;
    // a window past every length is none
    a.window = p->window < (1u << 31) ? static_cast<int>(p->window) : 0;
}

template <typename T, typename C, typename A>
void launch_attn(A a, const AttnPlan &plan, const tqt_attn_paged_params *p, hipStream_t stream, const char *where)
{
    a.few_workgroups = plan.few_workgroups;
    a.tile_chunk = plan.tile.chunk;
    a.tile_rows = kAttnTileRows;
    a.few_rows = plan.run_few ? attn_few_rows<A>(a.head_dim) : 0;
    a.part_o = static_cast<float *>(p->workspace);
    a.part_ml = a.part_o + plan.parts * a.head_dim;
    if (plan.run_few) {
        by_head_dim<64, 128, 256>(a.head_dim, [&](auto dp, auto full) {
            constexpr int kMost = attn_few_rows<A>(dp.value) / 16;
            const dim3 grid(plan.few_workgroups), block(64 * kAttnFewRowWaves);
            if (plan.few_columns < kMost) {
                hipLaunchKernelGGL((attn_few_row_kernel<T, C, dp.value, full.value, A, 1>), grid, block, 0, stream, a);
            } else {
                hipLaunchKernelGGL((attn_few_row_kernel<T, C, dp.value, full.value, A, kMost>), grid, block, 0,
                                   stream, a);
            }
        });
        check_launch(where);
    }
    if (plan.run_tile) {
        dim3 grid(static_cast<unsigned>(plan.tiles * a.kv_heads), plan.tile.splits);
        if (plan.even_parts > 0) {
            // at most two rounds, and a workgroup at least for each tile
            grid = dim3(static_cast<unsigned>(2 * attn_tile_workgroups(a.head_dim) / a.kv_heads * a.kv_heads));
        }
        by_head_dim<64, 96, 128, 192, 256>(a.head_dim, [&](auto dp, auto full) {
            hipLaunchKernelGGL((attn_tile_kernel<T, C, dp.value, 4, full.value, A>), grid, dim3(256), 0, stream,
                               a);
        });
        check_launch(where);
    }
    constexpr bool kQuant = std::is_same<C, int8_t>::value;
    const bool join_tile = plan.run_tile && plan.tile.splits > 1;
    const bool join_few = plan.few_workgroups > 1 && !plan.few_whole;
    if (join_few || join_tile) {
        const int each = static_cast<int>(plan.few_tokens), few = join_few ? a.batch * each : 0;
        const int rows = few + (join_tile ? a.q_tokens : 0);
        if (plan.few_many || plan.tile.splits > kAttnJoinManyParts) {
            hipLaunchKernelGGL((attn_join_many_kernel<T, kQuant, A>), dim3(static_cast<unsigned>(rows) * a.q_heads),
                               dim3(256), 0, stream, a, few, each);
        } else {
            const int per_wave = 256 / a.head_dim;
            const long long items = static_cast<long long>(rows) * ((a.q_heads + per_wave - 1) / per_wave);
            hipLaunchKernelGGL((attn_join_few_kernel<T, kQuant, A>), dim3(static_cast<unsigned>((items + 3) / 4)),
                               dim3(256), 0, stream, a, few, each, rows);
        }
    }
    check_launch(where);
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
    set_attn(a, p);
    launch_attn<T, C>(a, attn_plan(p), p, stream, where);
    return true;
}

template <typename T, typename C>
bool run_attn_tree(const tqt_attn_tree_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = attn_tree_error(p, sizeof(C), std::is_same<C, int8_t>::value);
    TQT_REQUIRE(error == nullptr, error);
    if (attn_empty(&p->attn)) {
        return false;
    }
    AttnTreeArgs a = {};
    set_attn(a, &p->attn);
    a.causal = 0;
    a.mask = p->mask;
    a.ld_mask = static_cast<int>(p->ld_mask);
    const AttnPlan plan = attn_plan(&p->attn, 32 * static_cast<long long>(p->ld_mask));
    a.few_unit = plan.few_whole ? 1 << 30 : kAttnFewRowUnit;
    a.even_parts = plan.even_parts;
    if (plan.even_parts > 0) {
        const long long longest = plan.span + 63;  // a tile's keys begin at a multiple of 64
        a.even_round = static_cast<int>(attn_tile_workgroups(a.head_dim));
        a.even_least = static_cast<int>(std::max<long long>(
            kAttnTileLeast, ((longest + plan.even_parts - 1) / plan.even_parts + 63) / 64 * 64));
        a.even_most = static_cast<int>((longest + 127) / 64 * 64);
        a.even_chunk = reinterpret_cast<int *>(static_cast<float *>(p->attn.workspace) + (plan.parts - 4) * a.head_dim);
    }
    launch_attn<T, C>(a, plan, &p->attn, stream, where);
    return true;
}

}  // namespace
}  // namespace tqt

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


#define TQT_ATTN_TREE_ENTRIES(NAME, T, C)                                                             \
    const char *tqt_get_error_attn_tree_##NAME##_gfx950(const struct tqt_attn_tree_params *params)    \
    {                                                                                                 \
        return attn_tree_error(params, sizeof(C), std::is_same<C, int8_t>::value);                    \
    }                                                                                                 \
    void tqt_run_attn_tree_##NAME##_gfx950_async(const struct tqt_attn_tree_params *params,           \
                                                 void *stream)                                        \
    {                                                                                                 \
        run_attn_tree<T, C>(params, as_stream(stream), "tqt_run_attn_tree_" #NAME "_gfx950");         \
    }                                                                                                 \
    void tqt_run_attn_tree_##NAME##_gfx950(const struct tqt_attn_tree_params *params)                 \
    {                                                                                                 \
        if (run_attn_tree<T, C>(params, nullptr, "tqt_run_attn_tree_" #NAME "_gfx950")) {             \
            finish_sync(nullptr, "tqt_run_attn_tree_" #NAME "_gfx950");                               \
        }                                                                                             \
    }
