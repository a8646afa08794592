// Attention over a paged cache with f16 queries: the entry points, and the workspace's size for all types.
#include "attn_paged.hpp"

using namespace tqt;

extern "C" {

size_t tqt_get_workspace_size_attn_paged_gfx950(const struct tqt_attn_paged_params *params)
{
    if (params == nullptr || attn_size_error(params) != nullptr || attn_empty(params)) {
        return 0;
    }
    const AttnPlan plan = attn_plan(params);
    return static_cast<size_t>(plan.parts) * (params->kv.head_dim + 2) * 4;
}

TQT_ATTN_ENTRIES(f16_f16, _Float16, _Float16)
TQT_ATTN_ENTRIES(f16_qsi8dx, _Float16, int8_t)

}  // extern "C"
