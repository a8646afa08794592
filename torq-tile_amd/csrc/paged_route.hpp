// Rules of the bookkeeping of a paged cache: how a call is launched. Plain C++ without HIP, so that a host program can
// evaluate them as the launcher does.
#pragma once

namespace tqt {

// Threads of the workgroup that goes over the batch.
constexpr int kPlanThreads = 1024;

// Whether that workgroup does the rows too: with so many at most, and every sequence in its shared memory. (us in one
// and in two launches: 256 sequences with 1818 rows 9.3, 10.0; 64 with 1547 9.5, 10.4, with 2497 in trees 13.4, 12.4.)
constexpr long long kPlanRowsOfOne = 2048;

inline bool plan_one_launch(long long batch, long long tokens)
{
    return batch <= kPlanThreads && tokens <= kPlanRowsOfOne;
}

}  // namespace tqt
