// What the append to a paged cache and the attention over it share: the checks of its geometry.
#pragma once

#include "tqt_hip_common.hpp"
#include "tqt_kv_append_rope_gfx950.h"

namespace tqt {

constexpr size_t kMaxHeadDim = 256;

// NULL, or why the cache's geometry is refused. `bytes`: of an element; `quant`: int8 with scales. Rows on
// the 16-byte grid let every kernel move 16 bytes at a time; fewer than 2^31 tokens keep slot arithmetic in
// 32 bits (element offsets are 64-bit).
inline const char *paged_kv_error(const tqt_paged_kv &c, size_t bytes, bool quant)
{
    if (c.head_dim == 0 || c.head_dim % 16 != 0 || c.head_dim > kMaxHeadDim) {
        return "head_dim is not a multiple of 16 from 16 to 256";
    }
    if (c.kv_heads == 0 || c.kv_heads >= (1u << 16)) {
        return "kv_heads is 0 or too large";
    }
    if (c.page_size == 0 || c.page_size >= (1u << 31) || c.num_pages >= (1u << 31) ||
        c.num_pages * c.page_size >= (1u << 31)) {
        return "page_size is 0, or the cache holds 2^31 tokens or more";
    }
    if (c.num_pages > 0 && (c.k == nullptr || c.v == nullptr)) {
        return "kv.k / kv.v == NULL";
    }
    if (quant && c.num_pages > 0 && (c.scale_k == nullptr || c.scale_v == nullptr)) {
        return "kv.scale_k / kv.scale_v == NULL for an int8 cache";
    }
    if (!aligned16(c.k) || !aligned16(c.v) || c.page_stride * bytes % 16 != 0 ||
        c.token_stride * bytes % 16 != 0 || c.head_stride * bytes % 16 != 0) {
        return "the cache's rows are off the 16-byte grid";
    }
    return nullptr;
}

}  // namespace tqt
