// What the attention kernels over a paged cache share: a call's arguments and how a sequence is found.
#pragma once

#include "fast_div.hpp"
#include "paged_kv.hpp"
#include "tqt_hip_common.hpp"

namespace tqt {

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
    float scale;
    int causal, window;  // window 0: none
};

// A sequence of the batch, with every length brought inside what the host checked.
struct AttnSeq
{
    int first;   // its first row of Q
    int q_len, kv_len;
    int pos0;    // position of query 0 (negative: the first queries see nothing)
};

__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, int b)
{
    AttnSeq s;
    s.first = min(max(a.q_start[b], 0), a.q_tokens);
    const int end = min(max(a.q_start[b + 1], s.first), a.q_tokens);
    s.q_len = end - s.first;
    s.kv_len = min(max(a.kv_len[b], 0), a.max_kv_len);
    s.pos0 = s.kv_len - s.q_len;
    return s;
}

// The keys [lo, hi) that the query at `pos` may see.
__device__ __forceinline__ void attn_bounds(const AttnArgs &a, const AttnSeq &s, int pos, int &lo, int &hi)
{
    hi = a.causal ? min(pos + 1, s.kv_len) : s.kv_len;
    lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
}

}  // namespace tqt
