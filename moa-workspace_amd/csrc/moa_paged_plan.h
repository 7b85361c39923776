// moa_paged_plan.h -- decisions of the paged cache's kernels in plain arithmetic, for the device and for host tests.
#pragma once

#ifdef __HIPCC__
#define MOA_PLAN_FN __host__ __device__ __forceinline__
#else
#define MOA_PLAN_FN inline
#endif

namespace moa {

// Whether a sequence's rows [row0, end) lie within a call's `rows`, at most max_rows of them. Row starts are device memory and
// may hold anything: the difference is taken only of values that are in range, since elsewhere it can pass 32 bits and look small.
MOA_PLAN_FN bool rows_in_range(int row0, int end, int rows, int max_rows) {
    return row0 >= 0 && row0 <= end && end <= rows && end - row0 <= max_rows;
}

// A counter that the parts of a split sequence arrive at: a launch adds kJoinTurn in all (the first part what the others leave), so
// the arrival that completes a turn is the last one, nothing is set back, and the counter stands at a multiple of kJoinTurn after
// every launch, whatever it held: calls that overlapped against the contract spoil their own results and no later call's.
constexpr unsigned kJoinTurn = 32;
MOA_PLAN_FN unsigned join_share(bool first, int parts) { return first ? kJoinTurn + 1 - (unsigned)parts : 1; }
MOA_PLAN_FN bool join_last(unsigned before, unsigned share) { return (before + share) % kJoinTurn == 0; }

}  // namespace moa
