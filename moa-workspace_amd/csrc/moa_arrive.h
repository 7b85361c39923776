// moa_arrive.h -- workgroups that share a piece of work: the last of them to arrive at a counter goes on, no other waits.
#pragma once

#include "moa_device.h"
#include "moa_internal.h"
#include "moa_paged_plan.h"

namespace moa {
namespace {

// The turn of the counters behind the first kSearchRows of the search tickets: a row's parts, a call's rows, a sequence's workgroups.
constexpr unsigned kRowTurn = 512;

// Whether this workgroup is the last of `parts` to arrive at a counter; what the others published before is then there to
// collect. kTurn: a power of two above any number of parts.
template <unsigned kTurn>
__device__ bool arrive_last(uint32_t* ticket, bool first, int parts) {
    __shared__ uint32_t flag;
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t share = join_share(first, parts, kTurn);
        flag = join_last(__hip_atomic_fetch_add(ticket, share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), share, kTurn);
    }
    __syncthreads();
    return flag;
}

}  // namespace
}  // namespace moa
