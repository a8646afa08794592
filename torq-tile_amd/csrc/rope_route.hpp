// Rules of the rotary positions and the append to a paged cache: which kernel takes a call, and the launches it is
// cut into. Plain C++ without HIP, so that a host program can evaluate them as the launcher does.
#pragma once

#include <algorithm>

namespace tqt {

// Work-items of one launch: of 2^32 at most along a grid's dimension, and of indexes that FastDiv takes.
constexpr long long kRopeMostThreads = 1ll << 30;

// Heads of more elements than a wave's lanes take (16 each) are normalised by rope_any_kernel.
constexpr long long kNormMostDim = 16 * 64;

struct RopeLaunch
{
    bool rows;           // rope_rows_kernel (a thread for 16 elements), else rope_any_kernel (a wave for a head)
    long long per_head;  // its threads of a head, or 1 wave
    long long tokens;    // of one launch
};

// A call with `heads` heads of `head_dim` elements per token. grid16: its rows suit rope_rows_kernel; the append to an
// int8 cache and the norm of heads pad a head's threads to a power of two (`pow2`), which exchange their maxima or sums
// in a butterfly. A token
// of more threads than a launch has goes to the waves: fewer than 2^21 heads of them fit.
inline RopeLaunch rope_launch(long long heads, long long head_dim, bool grid16, bool pow2)
{
    long long threads = head_dim / 16;
    if (pow2) {
        long long p = 1;
        while (p < threads) {
            p *= 2;
        }
        threads = p;
    }
    const bool rows = grid16 && heads * threads <= kRopeMostThreads;
    const long long per_token = rows ? heads * threads : heads * 64;
    return {rows, rows ? threads : 1, std::max(1ll, kRopeMostThreads / per_token)};
}

// The gradient of the norm: workgroups of 256 threads that go over the heads, `units` threads a head (of up to
// kNormMostDim elements) or a wave, with a share of the weight's gradient for each workgroup, or for each wave (four a
// workgroup, of 2^22 elements together unless a head has more).
struct NormGradLaunch
{
    int units, row_blocks, any_blocks;
};

constexpr long long kNormGradBlocks = 1024;

inline NormGradLaunch norm_grad_launch(long long rows, long long head_dim)
{
    long long units = 1;
    while (units < 64 && 16 * units < head_dim) {
        units *= 2;
    }
    const long long at_once = 256 / units, waves = std::max(1ll, std::min(4096ll, (1ll << 22) / head_dim));
    return {static_cast<int>(units),
            static_cast<int>(std::min(kNormGradBlocks, (rows + at_once - 1) / at_once)),
            static_cast<int>(std::min((rows + 3) / 4, (waves + 3) / 4))};
}

}  // namespace tqt
