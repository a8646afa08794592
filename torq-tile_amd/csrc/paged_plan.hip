// The bookkeeping of a step over a paged cache on gfx950: pages, block tables, lengths, slots, positions, tree masks.
//
// Bound by latency: some 30 bytes a token. What a sequence gets depends on all before it (rows, returned pages,
// needs are running sums over the batch), so one workgroup goes over the batch, a thread a sequence; the rows
// follow, a thread each, which finds its sequence by bisection: in the same workgroup where they are few (one launch
// instead of two), by a grid of their own else. A row's page comes from the block table or, for pages taken in this
// step, from the stack, by an index that follows from the sums alone; the row at a taken page's start writes the
// table's entry, so that no thread walks over a sequence's pages. 64 sequences with 1014 rows in trees take 9.3-9.6
// us in one launch; 256 with 32056 rows 7.8-8.2 and 2.4-3.5 (a workgroup of 256 threads: 14).
#include "fast_div.hpp"
#include "paged_route.hpp"
#include "tqt_hip_common.hpp"
#include "tqt_paged_plan_gfx950.h"

#include <algorithm>
#include <type_traits>

namespace tqt {
namespace {

constexpr int kPlanMostLen = 1 << 30;
constexpr int kPlanStarts = 2048;  // sequences whose first rows the rows' workgroups hold in LDS

// What the rows of a sequence need to know.
struct PlanSeq
{
    int kv_len;
    int held;        // entries of the block table that it had; -1: refused
    uint32_t fresh;  // entry j >= held comes from place fresh - j of the stack
    int unused;
};

struct PlanArgs
{
    const int32_t *new_len, *kv_len, *held, *free_count;
    int32_t *kv_len_out, *held_out, *free_count_out, *refused;
    int32_t *table, *free_pages, *q_start, *positions;
    int64_t *slots;
    const int32_t *parent;
    uint32_t *mask;
    PlanSeq *seqs;  // [batch], or nullptr: in LDS
    long long ld_table;
    int batch, tokens, num_pages, free_capacity, ld_mask;
    FastDiv page;
};

// A row: its sequence follows from q_start and seqs (these and parent are the call's or copies of them in LDS).
__device__ __forceinline__ void plan_row(const PlanArgs &a, int row, int total, const int32_t *q_start,
                                         const PlanSeq *seqs, const int32_t *parent)
{
    if (row >= total) {
        a.slots[row] = -1;
        a.positions[row] = 0;
        for (int w = 0; w < a.ld_mask; ++w) {
            a.mask[static_cast<long long>(row) * a.ld_mask + w] = 0;
        }
        return;
    }
    // the last sequence that begins at or before the row
    int b = 0;
    for (int end = a.batch; end - b > 1;) {
        const int mid = (b + end) >> 1;
        if (q_start[mid] <= row) {
            b = mid;
        } else {
            end = mid;
        }
    }
    const int first = q_start[b], i = row - first;
    const PlanSeq s = seqs[b];
    uint32_t offset;
    const uint32_t col = fast_div(static_cast<uint32_t>(s.kv_len + i), a.page, offset);
    long long slot = -1;
    if (s.held >= 0) {
        int32_t *entry = a.table + b * a.ld_table + col;
        int page;
        if (static_cast<int>(col) < s.held) {
            page = *entry;
        } else {
            page = a.free_pages[s.fresh - col];
            if (offset == 0) {
                *entry = page;
            }
        }
        if (page >= 0 && page < a.num_pages) {
            slot = static_cast<long long>(page) * a.page.d + offset;
        }
    }
    a.slots[row] = slot;
    if (a.parent == nullptr) {
        a.positions[row] = s.kv_len + i;
        return;
    }
    // up the tree: numbers fall, so the mask's words are done from the last to the first
    auto above = [&](int t) {
        const int p = parent[first + t];
        return p < t ? max(p, -1) : -1;
    };
    int t = i, depth = -1;
    for (; (t >> 5) >= a.ld_mask; t = above(t)) {
        ++depth;
    }
    for (int w = a.ld_mask - 1; w >= 0; --w) {
        uint32_t word = 0;
        for (; t >= 0 && (t >> 5) == w; t = above(t)) {
            word |= 1u << (t & 31);
            ++depth;
        }
        a.mask[static_cast<long long>(row) * a.ld_mask + w] = word;
    }
    a.positions[row] = s.kv_len + depth;
}

// Sum of the lanes up to and with this one, by moves between lanes (row_shr and row_bcast: shuffles go through LDS, and
// each of their six steps waits some hundred cycles).
__device__ __forceinline__ long long plan_wave_sum(long long x)
{
    auto add = [&](auto ctrl, auto rows) {
        const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), ctrl.value, rows.value, 0xf, false);
        const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(x >> 32), ctrl.value, rows.value, 0xf, false);
        x += static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 |
                                    static_cast<uint32_t>(lo));
    };
    typedef std::integral_constant<int, 0xf> All;
    add(std::integral_constant<int, 0x111>(), All());
    add(std::integral_constant<int, 0x112>(), All());
    add(std::integral_constant<int, 0x114>(), All());
    add(std::integral_constant<int, 0x118>(), All());
    add(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());
    add(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
    return x;
}

__device__ __forceinline__ long long plan_lane(long long x, int lane)
{
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), lane);
    return static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(
                                      __builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane)))
                                      << 32 |
                                  lo);
}

// The sum of the workgroup's threads up to and with this one, and of all of them. Every thread calls it.
// `on`: whether the wave has sequences, the same for all of its lanes; others only meet the barriers.
__device__ __forceinline__ long long plan_sum(long long x, bool on, long long (&s_wave)[kPlanThreads / 64],
                                              long long &all)
{
    constexpr int kWaves = kPlanThreads / 64;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const long long upto = on ? plan_wave_sum(x) : 0;
    __syncthreads();
    if (lane == 63) {
        s_wave[wave] = upto;
    }
    __syncthreads();
    const long long other = plan_wave_sum(lane < kWaves ? s_wave[lane] : 0);
    all = plan_lane(other, kWaves - 1);
    return upto + (wave > 0 ? plan_lane(other, wave - 1) : 0);
}

// Pages of an ended sequence that a lane keeps from counting them to putting them on the stack.
constexpr int kPlanHeld = 8;

// Sequences, a thread each, kPlanThreads at a time; with kRows also the rows (then batch <= kPlanThreads). Bound by
// what its waves issue and by the rows' chains of reads: waves without sequences skip the sums, but take rows. 64
// sequences, five of them ended, with 1014 rows in trees take 9.5 us so, 10.4 where all waves do all, 14.1 with 256
// threads, and 14.8 with shuffles, two sums more and the parents read from global memory.
template <bool kRows>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a)
{
    __shared__ long long s_wave[kPlanThreads / 64];
    __shared__ int s_list[kPlanThreads], s_held[kPlanThreads];
    __shared__ long long s_upto[kPlanThreads];
    __shared__ unsigned long long s_taken;
    __shared__ int s_refused;
    __shared__ int32_t s_start[kRows ? kPlanThreads + 1 : 1];
    __shared__ PlanSeq s_seqs[kRows ? kPlanThreads : 1];
    __shared__ int32_t s_parent[kRows ? kPlanRowsOfOne : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // what the first round of threads reads is asked for together: each wait for memory takes a microsecond
    const int first_count = a.free_count[0];
    const bool first_in = tid < a.batch;
    const int first_new = first_in ? a.new_len[tid] : 0, first_held = first_in ? a.held[tid] : 0;
    const int first_kv = first_in ? a.kv_len[tid] : 0;
    auto new_len = [&](int b) { return b < kPlanThreads ? first_new : b < a.batch ? a.new_len[b] : 0; };
    auto held_pages = [&](int b) { return b < kPlanThreads ? first_held : b < a.batch ? a.held[b] : 0; };
    auto kv_tokens = [&](int b) {
        return min(max(b < kPlanThreads ? first_kv : b < a.batch ? a.kv_len[b] : 0, 0), kPlanMostLen);
    };
    // the pages of so many tokens
    auto pages_of = [&](int n) {
        uint32_t rest;
        const long long pages = fast_div(static_cast<uint32_t>(n), a.page, rest);
        return pages + (rest > 0);
    };
    if constexpr (kRows) {
        // the way up a tree is a chain of reads
        if (a.parent != nullptr) {
            for (int row = tid; row < a.tokens; row += kPlanThreads) {
                s_parent[row] = a.parent[row];
            }
        }
    }
    if (tid == 0) {
        s_taken = 0;
        s_refused = 0;
    }
    const int count = min(max(first_count, 0), a.free_capacity);

    // 1. pages of ended sequences
    long long top = count;
    for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
        const bool on = b0 + 64 * wave < a.batch;
        int held = 0;
        if (on && new_len(b0 + tid) < 0) {
            held = static_cast<int>(
                min(max(static_cast<long long>(held_pages(b0 + tid)), pages_of(kv_tokens(b0 + tid))), a.ld_table));
        }
        if (!__syncthreads_or(held > 0)) {
            continue;
        }
        long long n;
        const int at = static_cast<int>(plan_sum(held > 0, on, s_wave, n)) - 1;
        if (held > 0) {
            s_list[at] = b0 + tid;
            s_held[at] = held;
        }
        __syncthreads();
        // a wave counts the kept pages of every so many-th of them; those of its first are at hand afterwards
        int pages[kPlanHeld];
        for (int k = wave; k < n; k += kPlanThreads / 64) {
            const int32_t *table = a.table + s_list[k] * a.ld_table;
            int kept = 0;
            if (k == wave) {
#pragma unroll
                for (int i = 0; i < kPlanHeld; ++i) {
                    pages[i] = 64 * i + lane < s_held[k] ? table[64 * i + lane] : -1;
                    kept += pages[i] >= 0 && pages[i] < a.num_pages;
                }
            }
            for (int j = (k == wave ? 64 * kPlanHeld : 0) + lane; j < s_held[k]; j += 64) {
                const int page = table[j];
                kept += page >= 0 && page < a.num_pages;
            }
            const long long all = plan_lane(plan_wave_sum(kept), 63);
            if (lane == 0) {
                s_upto[k] = all;
            }
        }
        __syncthreads();
        long long returned;
        const long long mine = tid < n ? s_upto[tid] : 0;
        const long long upto = plan_sum(mine, 64 * wave < n, s_wave, returned);
        if (tid < n) {
            s_upto[tid] = upto - mine;
        }
        __syncthreads();
        for (int k = wave; k < n; k += kPlanThreads / 64) {
            const int32_t *table = a.table + s_list[k] * a.ld_table;
            long long to = top + s_upto[k];
            auto put = [&](int page) {
                const bool kept = page >= 0 && page < a.num_pages;
                const unsigned long long all = __ballot(kept);
                const long long here = to + __builtin_popcountll(all & ((1ull << lane) - 1));
                if (kept && here < a.free_capacity) {
                    a.free_pages[here] = page;
                }
                to += __builtin_popcountll(all);
            };
            if (k == wave) {
#pragma unroll
                for (int i = 0; i < kPlanHeld; ++i) {
                    put(pages[i]);
                }
            }
            for (int j0 = k == wave ? 64 * kPlanHeld : 0; j0 < s_held[k]; j0 += 64) {
                put(j0 + lane < s_held[k] ? table[j0 + lane] : -1);
            }
        }
        top += returned;
        __syncthreads();
    }
    top = min(top, static_cast<long long>(a.free_capacity));

    // 2., 3. what the others need and get. Sequences whose rows do not fit come after all whose rows do, so that the
    // sums may count their pages. Those that get pages come before all that get none: the last one's sum is what
    // is taken.
    long long rows = 0, needed = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
        const int b = b0 + tid;
        const bool in = b < a.batch;
        if (b0 + 64 * wave >= a.batch) {
            long long all;
            plan_sum(0, false, s_wave, all);
            rows += all;
            plan_sum(0, false, s_wave, all);
            continue;
        }
        const int given = new_len(b), has = held_pages(b);
        const int kv_len = kv_tokens(b);
        const bool ended = given < 0;
        const int n = min(max(given, 0), kPlanMostLen);
        const long long own = pages_of(kv_len);
        const long long held = min(max(static_cast<long long>(has), own), a.ld_table);
        long long need = 0;
        bool fits = in && !ended && own <= a.ld_table && kv_len + static_cast<long long>(n) <= kPlanMostLen;
        if (fits) {
            need = max(pages_of(kv_len + n) - held, 0ll);
            fits = held + need <= a.ld_table;
            need = fits ? need : 0;
        }
        long long all;
        const long long rows_upto = rows + plan_sum(n, true, s_wave, all);
        rows += all;
        const long long upto = needed + plan_sum(need, true, s_wave, all);
        needed += all;
        const bool served = fits && (n == 0 || rows_upto <= a.tokens) && (need == 0 || upto <= top);
        if (served && need > 0) {
            atomicMax(&s_taken, static_cast<unsigned long long>(upto));
        }
        const unsigned long long refused = __ballot(in && !ended && !served);
        if (lane == 0 && refused != 0) {
            atomicAdd(&s_refused, static_cast<int>(__builtin_popcountll(refused)));
        }
        if (in) {
            a.kv_len_out[b] = ended ? 0 : served ? kv_len + n : kv_len;
            a.held_out[b] = static_cast<int32_t>(ended ? 0 : served ? held + need : held);
            const int32_t start = static_cast<int32_t>(min(rows_upto - n, static_cast<long long>(a.tokens)));
            const PlanSeq s = {kv_len, served ? static_cast<int>(held) : -1,
                               static_cast<uint32_t>(top - 1 - (upto - need) + held), 0};
            a.q_start[b] = start;
            if constexpr (kRows) {
                s_start[tid] = start;
                s_seqs[tid] = s;
            } else {
                a.seqs[b] = s;
            }
        }
    }
    const int total = static_cast<int>(min(rows, static_cast<long long>(a.tokens)));
    __syncthreads();
    if (tid == 0) {
        a.q_start[a.batch] = total;
        a.free_count_out[0] = static_cast<int32_t>(top - static_cast<long long>(s_taken));
        a.refused[0] = s_refused;
    }
    if constexpr (kRows) {
        for (int row = tid; row < a.tokens; row += kPlanThreads) {
            plan_row(a, row, total, s_start, s_seqs, s_parent);
        }
    }
}

__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a)
{
    __shared__ int32_t s_start[kPlanStarts];
    const int row = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
    const int total = a.q_start[a.batch];
    const int32_t *q_start = a.q_start;
    if (a.batch <= kPlanStarts) {
        for (int b = threadIdx.x; b < a.batch; b += 256) {
            s_start[b] = a.q_start[b];
        }
        __syncthreads();
        q_start = s_start;
    }
    if (row < a.tokens) {
        plan_row(a, row, total, q_start, a.seqs, a.parent);
    }
}

const char *plan_error(const tqt_paged_plan_params *p)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    if (p->batch >= (1u << 16) || p->tokens >= (1u << 30) || p->ld_table >= (1u << 31) ||
        p->free_capacity >= (1u << 31) || p->ld_mask >= (1u << 25)) {
        return "batch, tokens, ld_table, free_capacity or ld_mask too large";
    }
    if (p->page_size == 0 || p->page_size >= (1u << 31) || p->num_pages >= (1u << 31) ||
        p->num_pages * p->page_size >= (1u << 31)) {
        return "page_size is 0, or the cache holds 2^31 tokens or more";
    }
    if (p->free_count == nullptr || p->free_count_out == nullptr || p->refused == nullptr ||
        p->q_start == nullptr || (p->free_pages == nullptr && p->free_capacity > 0)) {
        return "free_count / free_count_out / refused / q_start / free_pages == NULL";
    }
    if (p->batch > 0 && (p->new_len == nullptr || p->kv_len == nullptr || p->kv_len_out == nullptr ||
                         p->held == nullptr || p->held_out == nullptr ||
                         (p->block_table == nullptr && p->ld_table > 0))) {
        return "new_len / kv_len / kv_len_out / held / held_out / block_table == NULL";
    }
    if (p->tokens > 0 && (p->positions == nullptr || p->slots == nullptr)) {
        return "positions / slots == NULL";
    }
    if (p->parent == nullptr ? p->mask != nullptr || p->ld_mask > 0
                             : p->mask == nullptr || p->ld_mask == 0) {
        return "trees need parent, mask and ld_mask together";
    }
    const size_t need = tqt_get_workspace_size_paged_plan_gfx950(p);
    if (p->workspace_size < need || (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace)))) {
        return "the workspace is too small or off the 16-byte grid";
    }
    return nullptr;
}

bool run_plan(const tqt_paged_plan_params *p, hipStream_t stream, const char *where)
{
    if (p == nullptr) {
        return false;
    }
    const char *error = plan_error(p);
    TQT_REQUIRE(error == nullptr, error);
    PlanArgs a = {};
    a.new_len = p->new_len;
    a.kv_len = p->kv_len;
    a.held = p->held;
    a.free_count = p->free_count;
    a.kv_len_out = p->kv_len_out;
    a.held_out = p->held_out;
    a.free_count_out = p->free_count_out;
    a.refused = p->refused;
    a.table = p->block_table;
    a.free_pages = p->free_pages;
    a.q_start = p->q_start;
    a.positions = p->positions;
    a.slots = p->slots;
    a.parent = p->parent;
    a.mask = p->mask;
    a.seqs = static_cast<PlanSeq *>(p->workspace);
    a.ld_table = static_cast<long long>(p->ld_table);
    a.batch = static_cast<int>(p->batch);
    a.tokens = static_cast<int>(p->tokens);
    a.num_pages = static_cast<int>(p->num_pages);
    a.free_capacity = static_cast<int>(p->free_capacity);
    a.ld_mask = static_cast<int>(p->ld_mask);
    a.page = make_fast_div(static_cast<uint32_t>(p->page_size));
    if (plan_one_launch(a.batch, a.tokens)) {
        hipLaunchKernelGGL((plan_kernel<true>), dim3(1), dim3(kPlanThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((plan_kernel<false>), dim3(1), dim3(kPlanThreads), 0, stream, a);
        check_launch(where);
        if (a.tokens > 0) {
            hipLaunchKernelGGL(plan_rows_kernel, dim3((a.tokens + 255) / 256), dim3(256), 0, stream, a);
        }
    }
    check_launch(where);
    return true;
}

}  // namespace
}  // namespace tqt

using namespace tqt;

extern "C" {

size_t tqt_get_workspace_size_paged_plan_gfx950(const struct tqt_paged_plan_params *params)
{
    if (params == nullptr || params->batch >= (1u << 16) || params->tokens >= (1u << 30) ||
        plan_one_launch(static_cast<long long>(params->batch), static_cast<long long>(params->tokens))) {
        return 0;
    }
    return params->batch * sizeof(PlanSeq);
}

const char *tqt_get_error_paged_plan_gfx950(const struct tqt_paged_plan_params *params)
{
    return plan_error(params);
}

void tqt_run_paged_plan_gfx950_async(const struct tqt_paged_plan_params *params, void *stream)
{
    run_plan(params, as_stream(stream), "tqt_run_paged_plan_gfx950");
}

void tqt_run_paged_plan_gfx950(const struct tqt_paged_plan_params *params)
{
    if (run_plan(params, nullptr, "tqt_run_paged_plan_gfx950")) {
        finish_sync(nullptr, "tqt_run_paged_plan_gfx950");
    }
}

}  // extern "C"
