// The paged cache's decisions (moa-workspace_amd/csrc/moa_paged_plan.h) for host tests, by C names.
#include "moa_paged_plan.h"

extern "C" {
int rows_in_range(int row0, int end, int rows, int max_rows) { return moa::rows_in_range(row0, end, rows, max_rows); }
unsigned join_turn() { return moa::kJoinTurn; }
unsigned join_share(int first, int parts) { return moa::join_share(first != 0, parts); }
int join_last(unsigned before, unsigned share) { return moa::join_last(before, share); }
int chunk_part_units(float total, int items) { return moa::chunk_part_units(total, items); }
}
