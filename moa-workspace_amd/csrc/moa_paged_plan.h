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
MOA_PLAN_FN unsigned join_share(bool first, int parts, unsigned turn = kJoinTurn) { return first ? turn + 1 - (unsigned)parts : 1; }
MOA_PLAN_FN bool join_last(unsigned before, unsigned share, unsigned turn = kJoinTurn) { return (before + share) % turn == 0; }

// Units of a part of a split tile, such that tiles of more units, in ceil(units / part) parts each, have at most `items` parts in all: a
// tile has less than 2 units / part of them, so part >= 2 total / items will do. `total` is an f32 sum of one product per
// sequence, over up to 1024 terms a lane and 6 across the wave: short by at most 1 + 1024 + 6 roundings of 2^-24, 6.15e-5 of it,
// and the three operations here by 3 more. A part in ten thousand more covers them all; the 1 covers the fraction that is cut off.
// No tile has 1e9 units.
constexpr int kChunkMinUnits = 4;
MOA_PLAN_FN int chunk_part_units(float total, int items) {
    const float part = 2.0002f * total / (float)items + 1.0f;
    const int whole = (int)(part < 1e9f ? part : 1e9f);
    return whole > kChunkMinUnits ? whole : kChunkMinUnits;
}

}  // namespace moa
