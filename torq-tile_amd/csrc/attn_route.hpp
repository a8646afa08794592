// Rules of the attention over a paged cache: which kernel takes a sequence, and how its keys are split.
// Plain C++ without HIP, so that a host program can evaluate them as the launcher does.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace tqt {

// Rows of one key head that the few-row kernel takes: (new tokens) x (query heads per key head), as many
// as its matrix instruction has columns.
constexpr int kAttnFewRows = 16;

// Keys that the queries of one sequence may see at most.
constexpr long long attn_span(long long max_q_len, long long max_kv_len, long long window)
{
    return window > 0 ? std::min(max_kv_len, window + max_q_len - 1) : max_kv_len;
}

// The first key that a query at position `pos` sees through a window of `window` keys (0: none). Queries that
// stand before every key have negative positions, down to 1 - 2^31, and a window may be 2^31 - 1: only the
// difference of two positions that are not negative is formed.
constexpr int attn_first_key(int pos, int window)
{
    return window > 0 && pos >= window ? pos - window + 1 : 0;
}

// The few-row kernel reads each key once, so it is bound by the cache's bytes: every CU should have them in
// flight all the time, whatever the lengths are. Its keys are cut into units of so many for each key head, and
// the workgroups that fit the chip at once take equal runs of units, across sequences.
constexpr int kAttnFewRowWaves = 4;
constexpr int kAttnFewRowUnit = 32 * kAttnFewRowWaves;

// Workgroups of the few-row kernel for a call of at most so many units.
inline int attn_few_row_workgroups(long long units, int per_cu)
{
    return static_cast<int>(std::max(1ll, std::min(units, 256ll * per_cu)));
}

// Whether the join of the few-row kernel's parts takes four waves for a row instead of one: at more parts
// than so many.
constexpr int kAttnJoinManyParts = 16;

// The tile kernel is bound by instructions. Workgroups that a CU's registers hold (a prompt of 4096, 32 / 8
// heads of 64, bf16: three 105 us, two 117):
constexpr int kAttnTileRows = 128;
constexpr int attn_tile_per_cu(size_t cache_element, int head_dim)
{
    return head_dim > 128 ? 1 : head_dim > 64 || cache_element == 1 ? 2 : 3;
}

// Where the tiles are fewer than fill the chip, their keys are split, in spans of at least 256, for so many
// workgroups: 512, or 256 where a CU holds one (512 tokens of 32 / 8 heads over 8000 keys: d 128 in four parts
// 83 us and 10 of join; d 256 173 us with 256 workgroups, 189 with 512). Heads of 64 are not faster with 768
// (256 tokens over 16384 keys 60 us, 58 with 512).
constexpr int kAttnTileLeast = 256;
constexpr long long attn_tile_workgroups(long long head_dim)
{
    return head_dim > 128 ? 256 : 512;
}

// Tiles of all sequences at most, from the host's bounds.
inline long long attn_tiles(long long batch, long long q_tokens, long long max_q_len, long long group)
{
    const long long each = (max_q_len * group + kAttnTileRows - 1) / kAttnTileRows;
    return std::min(batch * each, q_tokens * group / kAttnTileRows + batch);
}

struct AttnSplit
{
    int chunk, splits;
};

// What the parts and their join cost, in keys that a workgroup has meanwhile; a split that takes less from the
// longest workgroup is not made. 32 / 8 heads of 128 (256), us with and without a split: 300 tokens from an
// empty cache 18.3, 13.6 (29.3, 24.6), 512: 22.5, 17.4 (34.5, 31.5), 1000: 39, 27; 512 tokens over 1024
// keys 33, 26 (46.6, 48.1), 256 over 1024 24.9, 25.8; 64 over 512 17.4, 16.9 (26.8, 30.9).
constexpr long long attn_split_cost(long long workgroups, long long head_dim)
{
    return head_dim > 128 ? 128 + 200 * workgroups / 256 : 256 + 800 * workgroups / 512;
}

inline AttnSplit attn_tile_split(long long tiles, long long kv_heads, long long span,
                                 long long head_dim = 128)
{
    const long long whole = std::max(1ll, tiles * kv_heads);
    const long long want = std::max(1ll, attn_tile_workgroups(head_dim) / whole);
    const long long chunk = std::max<long long>(kAttnTileLeast, ((span + want - 1) / want + 63) / 64 * 64);
    // a tile's span begins at a multiple of 64: up to 63 keys more
    const long long splits = (span + 63 + chunk - 1) / chunk;
    if (want == 1 || span - chunk < attn_split_cost(whole * splits, head_dim)) {
        return {static_cast<int>((span + 127) / 64 * 64), 1};
    }
    return {static_cast<int>(chunk), static_cast<int>(splits)};
}

// The parts and their join are laid out for every row of Q, `rows` (token, query head) pairs, whether a sequence has
// it or not: q_tokens may be a buffer's. From so many rows on keys are not split, so that the join's grid stays
// below 2^32 work-items (256 a row). A call of so few tiles that they are split has 2^15 rows of its own at most.
constexpr long long kAttnJoinRows = 1 << 23;

inline AttnSplit attn_call_split(long long tiles, long long kv_heads, long long span, long long head_dim,
                                 long long rows)
{
    const AttnSplit s = attn_tile_split(tiles, kv_heads, span, head_dim);
    return rows < kAttnJoinRows ? s : AttnSplit{static_cast<int>((span + 127) / 64 * 64), 1};
}

}  // namespace tqt
