// Attention of trees of new tokens over a paged cache with bf16 queries: the entry points.
#include "attn_paged.hpp"

using namespace tqt;

extern "C" {

TQT_ATTN_TREE_ENTRIES(bf16_bf16, __bf16, __bf16)
TQT_ATTN_TREE_ENTRIES(bf16_qsi8dx, __bf16, int8_t)

}  // extern "C"
