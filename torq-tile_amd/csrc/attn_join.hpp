// Joining the parts that several workgroups have of a row: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, with
// the parts taken in the order of the keys. Bound by latency at few rows, by the parts' bytes (at most 3% of the
// cache's at 256 keys a split) at many.
#pragma once

#include "attn_common.hpp"

namespace tqt {
namespace {

// kWaves waves per row, head_dim / 4 threads along it and as many such groups as fit over the splits: one wave
// (four rows a workgroup) where the parts are few, four where they are many. The first `few` rows of a head are
// those that the few-row kernel may have (`each` tokens of every sequence), the others are all rows of Q, for
// the tile kernel's.
template <typename T, int kWaves>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int few, int each, int rows)
{
    __shared__ f32x4 s_acc[kWaves > 1 ? 256 : 1];
    __shared__ float s_sum[kWaves > 1 ? 256 : 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const int heads = static_cast<int>(a.group.d);
    const int item = __builtin_amdgcn_readfirstlane(
        static_cast<int>(blockIdx.x) * (4 / kWaves) + (kWaves > 1 ? 0 : tid >> 6));
    if (item >= rows * a.q_heads) {
        return;
    }
    const int at_row = item / a.q_heads, head = item - at_row * a.q_heads;
    const bool tiles = at_row >= few;
    AttnSeq s;
    int token, units = 0, run = 1, before = 0;
    if (tiles) {
        token = at_row - few;
        int b = -1;
        for (int x0 = 0; x0 < a.batch && b < 0; x0 += 64) {
            const int x = x0 + lane;
            const unsigned long long here =
                __ballot(x < a.batch && a.q_start[x] <= token && token < a.q_start[x + 1]);
            b = here != 0 ? x0 + __builtin_ctzll(here) : -1;
        }
        if (b < 0) {
            return;
        }
        s = attn_seq(a, b);
        token -= s.first;
    } else {
        const int b = at_row / each;
        token = at_row - b * each;
        FewRowBatch batch;
        FewRowWork work;
        int total;
        run = few_row_run(a, lane, total, batch);
        for (int b0 = 0; a.batch > 64 && b0 <= b; b0 += 64) {
            few_row_batch(a, b0, before, lane, batch);
            before = __shfl(batch.upto, 63);
        }
        few_row_pick(batch, b & 63, s, work);
        units = work.units;
        before = __builtin_amdgcn_readlane(batch.upto, b & 63) - units * a.kv_heads;
    }
    if (token >= s.nq || (s.nq * heads > a.few_rows) != tiles) {
        return;
    }
    // the row's parts: part0, then from part1 on every `step` rows of the workspace
    uint32_t in_group;
    const int kvh = static_cast<int>(fast_div(head, a.group, in_group));
    int parts;
    long long part0, part1, step;
    if (tiles) {
        int first, last;
        attn_tile_span(a, s, (token * heads + static_cast<int>(in_group)) / a.tile_rows, a.tile_rows, first,
                       last);
        parts = attn_splits(first, last, a.tile_chunk);
        step = static_cast<long long>(a.q_tokens) * a.q_heads;
        part0 = 2ll * a.few_workgroups * kAttnFewRows +
                static_cast<long long>(s.first + token) * a.q_heads + head;
        part1 = part0 + step;
    } else {
        before += kvh * units;
        const int w0 = before / run, w1 = (before + units - 1) / run;
        parts = w1 - w0 + 1;
        const int r = token * heads + static_cast<int>(in_group);
        part0 = (2ll * w0 + 1) * kAttnFewRows + r;
        part1 = 2ll * (w0 + 1) * kAttnFewRows + r;
        step = 2 * kAttnFewRows;
    }
    if (parts == 1) {
        return;
    }
    token += s.first;
    const int across = a.head_dim / 4, groups = 64 * kWaves / across;
    const int me = kWaves > 1 ? tid : lane;
    const int group = me / across, at = me - group * across;
    float m = -INFINITY;
    for (int k = lane; k < parts; k += 64) {
        m = fmaxf(m, a.part_ml[2 * (k == 0 ? part0 : part1 + (k - 1) * step)]);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        m = fmaxf(m, __shfl_xor(m, off));
    }
    const float base = m == -INFINITY ? 0.0f : m;
    f32x4 acc = 0.0f;
    float sum = 0.0f;
    if (group < groups) {
        // consecutive parts to one group: the sums' order is that of the keys
        const int per = (parts + groups - 1) / groups;
        const int k1 = min(parts, (group + 1) * per);
#pragma unroll 8
        for (int k = group * per; k < k1; ++k) {
            const long long r = k == 0 ? part0 : part1 + (k - 1) * step;
            const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * r] - base);
            sum += a.part_ml[2 * r + 1] * f;
            acc += *reinterpret_cast<const f32x4 *>(a.part_o + r * a.head_dim + 4 * at) * f;
        }
    }
    if constexpr (kWaves > 1) {
        s_acc[tid] = acc;
        s_sum[tid] = sum;
        __syncthreads();
    }
    const f32x4 own = acc;
    const float own_sum = sum;
    for (int k = 1; k < groups; ++k) {
        if constexpr (kWaves > 1) {
            if (tid < across) {
                acc += s_acc[k * across + tid];
                sum += s_sum[k * across + tid];
            }
        } else {
            // every group's sums in turn, to the first
            const int from = k * across + at;
            sum += __shfl(own_sum, from);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[e] += __shfl(own[e], from);
            }
        }
    }
    if (me >= across) {
        return;
    }
    const float out[4] = {acc[0], acc[1], acc[2], acc[3]};
    attn_put<T, 4>(a, -1, token, head, 4 * at, out, m, sum);
}

}  // namespace
}  // namespace tqt
