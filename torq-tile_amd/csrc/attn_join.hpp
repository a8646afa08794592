// Joining the parts that several workgroups have of a row: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, with
// the parts taken in the order of the keys. Bound by latency at few rows, by the parts' bytes (at most 3% of the
// cache's at 256 keys a split) at many.
#pragma once

#include "attn_common.hpp"

namespace tqt {
namespace {

// One workgroup per row; head_dim / 4 threads along the row, as many such groups as fit over the splits. The
// first `few` workgroups of a head are the rows that the few-row kernel may have (its sequences have at most
// a.few_rows / group tokens), the others are all rows of Q, for the tile kernel's.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int few)
{
    __shared__ int s_seq;
    __shared__ f32x4 s_acc[256];
    __shared__ float s_sum[256];
    const int tid = threadIdx.x, head = static_cast<int>(blockIdx.y);
    const int heads = static_cast<int>(a.group.d);
    int b, token;
    const bool tiles = static_cast<int>(blockIdx.x) >= few;
    if (tiles) {
        token = static_cast<int>(blockIdx.x) - few;
        if (tid == 0) {
            s_seq = -1;
        }
        __syncthreads();
        for (int x = tid; x < a.batch; x += 256) {
            if (a.q_start[x] <= token && token < a.q_start[x + 1]) {
                s_seq = x;
            }
        }
        __syncthreads();
        b = s_seq;
        if (b < 0) {
            return;
        }
    } else {
        const int each = few / a.batch;
        b = static_cast<int>(blockIdx.x) / each;
        token = static_cast<int>(blockIdx.x) - b * each;
    }
    const AttnSeq s = attn_seq(a, b);
    if (tiles) {
        token -= s.first;
    }
    if (token >= s.nq || (s.nq * heads > a.few_rows) != tiles) {
        return;
    }
    int first, last, unused, chunk = a.few_chunk;
    if (tiles) {
        uint32_t head_in_group;
        fast_div(head, a.group, head_in_group);
        attn_tile_span(a, s, (token * heads + static_cast<int>(head_in_group)) / a.tile_rows, a.tile_rows,
                       first, last);
        chunk = a.tile_chunk;
    } else {
        attn_bounds(a, s, s.pos0, first, unused);
        attn_bounds(a, s, s.pos0 + s.nq - 1, unused, last);
    }
    const int splits = attn_splits(first, last, chunk);
    if (splits == 1) {
        return;
    }
    token += s.first;
    const long long row = static_cast<long long>(token) * a.q_heads + head;
    const long long step = static_cast<long long>(a.q_tokens) * a.q_heads;
    const int across = a.head_dim / 4, groups = 256 / across;
    const int group = tid / across, at = tid - group * across;
    float m = -INFINITY;
    for (int k = tid & 63; k < splits; k += 64) {
        m = fmaxf(m, a.part_ml[2 * (k * step + row)]);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        m = fmaxf(m, __shfl_xor(m, off));
    }
    const float base = m == -INFINITY ? 0.0f : m;
    f32x4 acc = 0.0f;
    float sum = 0.0f;
    if (group < groups) {
        // consecutive splits to one group: the sums' order is that of the keys
        const int each = (splits + groups - 1) / groups;
        const int k1 = min(splits, (group + 1) * each);
#pragma unroll 4
        for (int k = group * each; k < k1; ++k) {
            const long long r = k * step + row;
            const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * r] - base);
            sum += a.part_ml[2 * r + 1] * f;
            acc += *reinterpret_cast<const f32x4 *>(a.part_o + r * a.head_dim + 4 * at) * f;
        }
    }
    s_acc[tid] = acc;
    s_sum[tid] = sum;
    __syncthreads();
    if (tid >= across) {
        return;
    }
    for (int k = 1; k < groups; ++k) {
        acc += s_acc[k * across + tid];
        sum += s_sum[k * across + tid];
    }
    const float out[4] = {acc[0], acc[1], acc[2], acc[3]};
    attn_put<T, 4>(a, 0, 1, token, head, 4 * tid, out, m, sum);
}

}  // namespace
}  // namespace tqt
