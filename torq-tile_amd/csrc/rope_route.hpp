// Rules of the rotary positions and the append to a paged cache: which kernel takes a call, and the launches it is
// cut into. Plain C++ without HIP, so that a host program can evaluate them as the launcher does.
#pragma once

#include <algorithm>

namespace tqt {

// Work-items of one launch: of 2^32 at most along a grid's dimension, and of indexes that FastDiv takes.
constexpr long long kRopeMostThreads = 1ll << 30;

struct RopeLaunch
{
    bool rows;           // rope_rows_kernel (a thread for 16 elements), else rope_any_kernel (a wave for a head)
    long long per_head;  // its threads of a head, or 1 wave
    long long tokens;    // of one launch
};

// A call with `heads` heads of `head_dim` elements per token. grid16: its rows suit rope_rows_kernel; the append to an
// int8 cache pads a head's threads to a power of two (`pow2`), which exchange their maxima in a butterfly. A token
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

}  // namespace tqt
