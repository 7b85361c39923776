// The counters that a launch's parts join at (moa-workspace_amd/csrc/moa_paged_plan.h), with turns of any length, for host tests.
#include "moa_paged_plan.h"

extern "C" {
unsigned join_share(int first, int parts, unsigned turn) { return moa::join_share(first != 0, parts, turn); }
int join_last(unsigned before, unsigned share, unsigned turn) { return moa::join_last(before, share, turn); }
}
