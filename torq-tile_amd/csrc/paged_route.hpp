// Rules of the bookkeeping of a paged cache: how a call is launched. Plain C++ without HIP, so that a host program can
// evaluate them as the launcher does.
#pragma once

namespace tqt {

// Threads of the workgroup that goes over the batch.
constexpr int kPlanThreads = 1024;

// Whether that workgroup does the rows too: with so many at most, and every sequence in its shared memory.
constexpr long long kPlanRowsOfOne = 4 * kPlanThreads;

inline bool plan_one_launch(long long batch, long long tokens)
{
    return batch <= kPlanThreads && tokens <= kPlanRowsOfOne;
}

}  // namespace tqt
