// Joining the parts that several workgroups have of a row: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s,
// with the parts taken in the order of the keys. Bound by latency at few rows (the batch's lengths, then the
// parts), by the parts' bytes at many.
#pragma once

#include "attn_common.hpp"

namespace tqt {
namespace {

// A row's parts: part0, then from part1 on every `step` rows of the workspace.
struct JoinRow
{
    int parts;
    long long part0, part1, step;
    int token;  // row of Q
};

__device__ __forceinline__ long long join_part(const JoinRow &j, int k)
{
    return k == 0 ? j.part0 : j.part1 + (k - 1) * j.step;
}

// The parts of row `at_row` (the same for the whole wave) and query head `head` (a lane's own). The first `few`
// rows are those that the few-row kernel may have (`each` tokens of every sequence), the others are all rows
// of Q, for the tile kernel's. parts <= 1: nothing to join.
template <typename A>
__device__ __forceinline__ JoinRow join_row(const A &a, int few, int each, int at_row, int head, int lane)
{
    JoinRow j = {0, 0, 0, 0, 0};
    const int heads = static_cast<int>(a.group.d);
    const bool tiles = at_row >= few;
    AttnSeq s;
    int token, units = 0, run = 1, before = 0, b = -1;
    if (tiles) {
        token = at_row - few;
        for (int x0 = 0; x0 < a.batch && b < 0; x0 += 64) {
            const int x = x0 + lane;
            const unsigned long long here =
                __ballot(x < a.batch && a.q_start[x] <= token && token < a.q_start[x + 1]);
            b = here != 0 ? x0 + __builtin_ctzll(here) : -1;
        }
        if (b < 0) {
            return j;
        }
        s = attn_seq(a, b);
        token -= s.first;
    } else {
        b = at_row / each;
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
        return j;
    }
    j.token = s.first + token;
    uint32_t in_group;
    const int kvh = static_cast<int>(fast_div(head, a.group, in_group));
    const int r = token * heads + static_cast<int>(in_group);
    if (tiles) {
        const AttnKeys keys = attn_tile_keys(a, s, r / a.tile_rows, a.tile_rows);
        j.parts = attn_splits(keys.first, keys.last, attn_tile_span(a, b));
        j.step = static_cast<long long>(a.q_tokens) * a.q_heads;
        j.part0 = attn_few_parts(a) + static_cast<long long>(j.token) * a.q_heads + head;
        j.part1 = j.part0 + j.step;
    } else {
        before += kvh * units;
        const int w0 = before / run, w1 = (before + units - 1) / run;
        j.parts = w1 - w0 + 1;
        j.part0 = (2ll * w0 + 1) * attn_few_rows<A>(a.head_dim) + r;
        j.part1 = 2ll * (w0 + 1) * attn_few_rows<A>(a.head_dim) + r;
        j.step = 2 * attn_few_rows<A>(a.head_dim);
    }
    return j;
}

// Few parts: a wave takes as many heads of a row as fit at 4 elements a lane.
template <typename T, bool kQuant, typename A>
__global__ __launch_bounds__(256) void attn_join_few_kernel(A a, int few, int each, int rows)
{
    const int lane = threadIdx.x & 63;
    const int across = a.head_dim / 4, per_wave = 64 / across;
    const int blocks = (a.q_heads + per_wave - 1) / per_wave;
    const int item =
        __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6));
    if (item >= rows * blocks) {
        return;
    }
    const int at_row = item / blocks, group = lane / across, at = lane - group * across;
    const int head = (item - at_row * blocks) * per_wave + group;
    const bool mine = group < per_wave && head < a.q_heads;
    const JoinRow j = join_row(a, few, each, at_row, mine ? head : 0, lane);
    if (!mine || j.parts <= 1) {
        return;
    }
    float m = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < j.parts; ++k) {
        m = fmaxf(m, a.part_ml[2 * join_part(j, k)]);
    }
    const float base = m == -INFINITY ? 0.0f : m;
    f32x4 acc = 0.0f;
    float sum = 0.0f;
#pragma unroll 4
    for (int k = 0; k < j.parts; ++k) {
        const long long r = join_part(j, k);
        float part = a.part_ml[2 * r + 1];
        const float f = part_factor<kQuant>(a.part_ml[2 * r], base, part);
        sum += part;
        acc += *reinterpret_cast<const f32x4 *>(a.part_o + r * a.head_dim + 4 * at) * f;
    }
    const float out[4] = {acc[0], acc[1], acc[2], acc[3]};
    attn_put<T, 4>(a, -1, j.token, head, 4 * at, out, m, sum);
}

// Many parts: a workgroup takes one row, head_dim / 4 threads along it and as many such groups as fit over the
// parts.
template <typename T, bool kQuant, typename A>
__global__ __launch_bounds__(256) void attn_join_many_kernel(A a, int few, int each)
{
    __shared__ f32x4 s_acc[256];
    __shared__ float s_sum[256];
    const int tid = threadIdx.x, lane = tid & 63;
    const int at_row = static_cast<int>(blockIdx.x) / a.q_heads;
    const int head = static_cast<int>(blockIdx.x) - at_row * a.q_heads;
    const JoinRow j = join_row(a, few, each, at_row, head, lane);
    if (j.parts <= 1) {
        return;
    }
    const int across = a.head_dim / 4, groups = 256 / across;
    const int group = tid / across, at = tid - group * across;
    float m = -INFINITY;
    for (int k = lane; k < j.parts; k += 64) {
        m = fmaxf(m, a.part_ml[2 * join_part(j, k)]);
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
        const int per = (j.parts + groups - 1) / groups;
        const int k1 = min(j.parts, (group + 1) * per);
#pragma unroll 8
        for (int k = group * per; k < k1; ++k) {
            const long long r = join_part(j, k);
            float part = a.part_ml[2 * r + 1];
            const float f = part_factor<kQuant>(a.part_ml[2 * r], base, part);
            sum += part;
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
    attn_put<T, 4>(a, -1, j.token, head, 4 * at, out, m, sum);
}

}  // namespace
}  // namespace tqt
