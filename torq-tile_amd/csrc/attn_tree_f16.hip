// Attention of trees of new tokens over a paged cache with f16 queries: the entry points, and the workspace's size
// for all types.
#include "attn_paged.hpp"

using namespace tqt;

extern "C" {

size_t tqt_get_workspace_size_attn_tree_gfx950(const struct tqt_attn_tree_params *params)
{
    if (params == nullptr || params->ld_mask >= (1u << 25) || attn_size_error(&params->attn) != nullptr ||
        attn_empty(&params->attn)) {
        return 0;
    }
    const AttnPlan plan = attn_plan(&params->attn, 32 * static_cast<long long>(params->ld_mask));
    return static_cast<size_t>(plan.parts) * (params->attn.kv.head_dim + 2) * 4;
}

TQT_ATTN_TREE_ENTRIES(f16_f16, _Float16, _Float16)
TQT_ATTN_TREE_ENTRIES(f16_qsi8dx, _Float16, int8_t)

}  // extern "C"
