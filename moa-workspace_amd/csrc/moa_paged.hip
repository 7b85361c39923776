// moa_paged.hip -- the paged KV cache (include/moa_paged.h): argument checks, the calls that change its
// state (reserve, fork, free, compact, a tree's commit, reorder), the append of new rows, and the copies of pages.
//
// State changes that are all or nothing are planned by one workgroup that reads the lengths and the reference counts, checks the whole
// call, and only then writes: that makes a call all or nothing and its result independent of any order between
// workgroups. Pages are copied by a second launch over the plan's list of moves.
#include <algorithm>
#include <string>

#include "../../include/moa_paged.h"
#include "moa_arrive.h"
#include "moa_checks.h"
#include "moa_device.h"
#include "moa_paged.h"

namespace moa {
namespace {

constexpr int kPlanBlock = 1024;
constexpr int kPlanWaves = kPlanBlock / kWave;

// ------------------------------------------------------------------ one workgroup's sums and ranks

// The sum of v over the workgroup, in every thread.
__device__ uint64_t block_sum(uint64_t v, uint64_t* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) t += lds[w];
    return t;
}

// The sum of v over the threads before this one; *total: over all of them.
__device__ int block_before(int v, int* lds, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(x, o, kWave);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? lds[w] : 0;
        all += lds[w];
    }
    *total = all;
    return before + x - v;
}

// The last of kPlanBlock ascending numbers, the first of which is 0, that is at most r.
__device__ __forceinline__ int last_at_most(const int* numbers, int r) {
    int lo = 0;
#pragma unroll
    for (int step = kPlanBlock / 2; step > 0; step /= 2)
        if (numbers[lo + step] <= r) lo += step;
    return lo;
}

// kPer pages a thread and step, so that a step's loads go out together.
constexpr int kPer = 8;
constexpr int kStepPages = kPlanBlock * kPer;

struct Counts { int32_t r[kPer]; };  // reference counts of the thread's pages of one step (0 behind the last)
__device__ __forceinline__ Counts counts_at(const PagedView& c, int base) {
    Counts v;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int p = base + j * kPlanBlock + (int)threadIdx.x;
        v.r[j] = p < c.pages ? c.refs[p] : 0;
    }
    return v;
}

// Calls f(page, rank, count) for the pages of [from, to) that are free (want_free) or live, in ascending order of rank, until
// `most` of them; returns how many there were. first: counts_at(c, 0), asked for ahead of the work that leads here.
template <class F>
__device__ int each_page(const PagedView& c, const Counts& first, int from, int to, bool want_free, int most, int* lds, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int found = 0;
    for (int base = from / kStepPages * kStepPages; base < to && found < most; base += kStepPages) {
        Counts v = first;
        if (base) v = counts_at(c, base);
        uint64_t b[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int p = base + j * kPlanBlock + (int)threadIdx.x;
            b[j] = __ballot(p >= from && p < to && (v.r[j] > 0) != want_free);
        }
        __syncthreads();  // the step before has read the counts
        if (lane < kPer) {
            uint64_t mine = b[0];
#pragma unroll
            for (int j = 1; j < kPer; ++j) mine = lane == j ? b[j] : mine;
            lds[lane * kPlanWaves + wave] = __popcll(mine);
        }
        __syncthreads();
        // every wave scans the step's kPer * kPlanWaves = 128 counts, two a lane
        const int c0 = lds[2 * lane], c1 = lds[2 * lane + 1];
        int x = c0 + c1;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int y = __shfl_up(x, o, kWave);
            if (lane >= o) x += y;
        }
        const int all = __shfl(x, 63, kWave);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int at = j * kPlanWaves + wave;  // counts before it: the scan of the lane that holds it
            const int upto = __shfl(x, at >> 1, kWave), odd = __shfl(c1, at >> 1, kWave), even = __shfl(c0, at >> 1, kWave);
            const int before = upto - odd - ((at & 1) ? 0 : even);
            const int rank = found + before + __popcll(b[j] & ((1ull << lane) - 1));
            if ((b[j] >> lane & 1) && rank < most) f(base + j * kPlanBlock + (int)threadIdx.x, rank, v.r[j]);
        }
        found += all;
    }
    __syncthreads();  // what f wrote is seen by the workgroup
    return min(found, most);
}
static_assert(kPer * kPlanWaves == 2 * kWave, "each_page scans two counts a lane");

// A list of pages by rank: the first kFew in LDS, the others in global memory.
constexpr int kFew = 2 * kPlanBlock;
struct PageList {
    int *few; int32_t* more;
    __device__ void put(int rank, int p) const {
        if (rank < kFew) few[rank] = p;
        else more[rank] = p;
    }
    __device__ int get(int rank) const { return rank < kFew ? few[rank] : more[rank]; }
};

__device__ __forceinline__ int pages_of(const PagedView& c, int n) { return (int)page_of(c, (uint32_t)(n + (int)c.slots - 1)); }

__device__ __forceinline__ void raise(const PagedView& c) { atomicOr(c.err, kErrPaged); }

// ------------------------------------------------------------------------------------------ reserve

// Thread t takes sequences t, t + 1024, ...: a first pass checks them and counts the pages they need, then the lowest
// free pages are listed, and a second pass hands them out, 1024 sequences at a time: each thread takes pages by their rank and
// finds their sequence among the prefix sums of the needs. Bound by its chain of memory round trips and barriers (7.3 us with
// lengths, counts and the list fetched one after the other, 6.7 with lengths and counts asked for at once and a short list in LDS).
__global__ __launch_bounds__(kPlanBlock) void paged_reserve_kernel(PagedView c, const int32_t* fresh, int32_t* list) {
    __shared__ uint64_t sums[kPlanWaves];
    __shared__ int lds[2 * kWave], before[kPlanBlock], old[kPlanBlock], few[kFew];
    const PageList free_pages = {few, list};
    const int cap = paged_capacity(c);
    const Counts first = counts_at(c, 0);
    const int len0 = (int)threadIdx.x < c.sequences ? c.lens[threadIdx.x] : 0, n0 = (int)threadIdx.x < c.sequences ? fresh[threadIdx.x] : 0;
    uint64_t need = 0;
    bool bad = false;
    for (int s = threadIdx.x; s < c.sequences; s += kPlanBlock) {
        const int len = s < kPlanBlock ? len0 : c.lens[s], n = s < kPlanBlock ? n0 : fresh[s];
        if (n < 0 || len < 0 || len > cap || n > cap - len) bad = true;
        else need += pages_of(c, len + n) - pages_of(c, len);
    }
    bad = __syncthreads_or(bad);
    need = block_sum(need, sums);
    if (bad || need > (uint64_t)c.pages ||
        each_page(c, first, 0, c.pages, true, (int)need, lds, [&](int p, int rank, int) { free_pages.put(rank, p); }) < (int)need) {
        if (threadIdx.x == 0) raise(c);
        return;
    }
    int given = 0;
    for (int base = 0; base < c.sequences; base += kPlanBlock) {
        const int s = base + (int)threadIdx.x, t = threadIdx.x;
        const int len = base == 0 ? len0 : (s < c.sequences ? c.lens[s] : 0), n = base == 0 ? n0 : (s < c.sequences ? fresh[s] : 0);
        const int had = pages_of(c, len);
        int all = 0;
        before[t] = block_before(pages_of(c, len + n) - had, lds, &all);
        old[t] = had;
        if (n > 0) c.lens[s] = len + n;
        __syncthreads();
        for (int r = t; r < all; r += kPlanBlock) {
            const int lo = last_at_most(before, r);  // the sequence whose pages start at or before rank r: one with pages
            const int p = free_pages.get(given + r);
            c.table[(base + lo) * c.table_stride + old[lo] + r - before[lo]] = p;
            c.refs[p] = 1;
        }
        given += all;
        __syncthreads();  // the next sequences' sums
    }
}

// --------------------------------------------------------------------------------------- page copies

// Moves (source page, target page) of every layer's K and V; a negative source is no move. A unit of work is up to
// kCopyBytes of one page of one tensor: 256 threads, four 16-byte loads each before the first store, so a workgroup
// has 16 KB in flight. Bound by memory: 870 MB read and written in 175 us, 5 TB/s.
constexpr int kCopyBlock = 256;
constexpr int kCopyBytes = kCopyBlock * 16 * 4;

// Where 16-byte chunk i of a page lies. Dense: slots and heads fill the page without gaps, in either order.
__device__ __forceinline__ int64_t chunk_at(bool dense, uint32_t i, uint32_t per_row, uint32_t heads, int64_t slot, int64_t head) {
    if (dense) return (int64_t)i * 16;
    const uint32_t row = i / per_row, in = i - row * per_row, s = row / heads, h = row - s * heads;
    return s * slot + h * head + in * 16;
}

__device__ void copy_pages(const PagedView& c, const int32_t* src, const int32_t* dst, int moves, int elem, int dense_k,
                           int dense_v, int wg, int wgs) {
    const uint32_t per_row = (uint32_t)(c.head_dim * elem / 16), chunks = c.slots * (uint32_t)c.kv_heads * per_row;
    const uint32_t parts = (chunks + kCopyBytes / 16 - 1) / (kCopyBytes / 16);
    const uint64_t per_move = (uint64_t)parts * 2 * c.layers;
    for (uint64_t u = wg; u < per_move * moves; u += wgs) {
        const int m = (int)(u / per_move);
        const uint32_t r = (uint32_t)(u - m * per_move), tensor = r / parts, part = r - tensor * parts;
        const int from = src[m], to = dst[m];
        if (from < 0) continue;
        const bool v = tensor & 1;
        uint8_t* base = v ? c.v + (int64_t)(tensor >> 1) * c.v_layer : c.k + (int64_t)(tensor >> 1) * c.k_layer;
        const int64_t page = v ? c.v_page : c.k_page, slot = v ? c.v_slot : c.k_slot, head = v ? c.v_head : c.k_head;
        const uint8_t* a = base + from * page;
        uint8_t* b = base + to * page;
        const bool dense = v ? dense_v : dense_k;
        const uint32_t i0 = part * (kCopyBytes / 16) + threadIdx.x;
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * kCopyBlock < chunks)
                w[j] = ld16(a + chunk_at(dense, i0 + j * kCopyBlock, per_row, c.kv_heads, slot, head));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * kCopyBlock < chunks)
                *reinterpret_cast<uint4*>(b + chunk_at(dense, i0 + j * kCopyBlock, per_row, c.kv_heads, slot, head)) = w[j];
    }
}

// --------------------------------------------------------------------------------------------- fork

// What the plan needs of fork f: lengths are -1 where an index is out of range.
struct Fork { int parent, child, len, child_len, full, page; };
__device__ __forceinline__ Fork fork_at(const PagedView& c, const int32_t* parents, const int32_t* children, int count, int f) {
    Fork x = {-1, -1, -1, -1, 0, -1};
    if (f >= count) return x;
    x.parent = parents[f], x.child = children[f];
    if (x.parent >= 0 && x.parent < c.sequences) x.len = c.lens[x.parent];
    if (x.child >= 0 && x.child < c.sequences) x.child_len = c.lens[x.child];
    if (x.len >= 0 && x.len <= paged_capacity(c)) {
        x.full = (int)page_of(c, x.len);
        if (x.full * (int)c.slots < x.len) x.page = c.table[x.parent * c.table_stride + x.full];
    }
    return x;
}

// Checks the whole call, the tables of the parents included (each parent's once, 1024 forks' entries at a time dealt out to the
// threads, as the reserve plan deals out pages), then hands out the pages of the partly filled last pages. src, dst: per fork the
// page to copy (-1: none) and its copy; result: the number of forks, 0 if the call is refused. Bound by its chain of memory round
// trips, as the reserve plan: the first 1024 forks' values are fetched once (one fork 9.8 us, 36 of 9 parents 11; the tables
// are 3 to 4 us of that).
__global__ __launch_bounds__(kPlanBlock) void paged_fork_plan_kernel(PagedView c, const int32_t* parents, const int32_t* children,
                                                                     int count, int32_t* src, int32_t* dst, int32_t* result) {
    __shared__ int lds[2 * kWave], few[kFew], before[kPlanBlock], row[kPlanBlock];
    __shared__ uint32_t child[kPagedMaxSequences / 32], parent[kPagedMaxSequences / 32];
    const PageList free_pages = {few, dst + kPagedMaxSequences};
    const Counts first = counts_at(c, 0);
    const Fork mine = fork_at(c, parents, children, count, threadIdx.x);
    if (threadIdx.x == 0) *result = 0;
    for (int i = threadIdx.x; i < (c.sequences + 31) / 32; i += kPlanBlock) child[i] = 0, parent[i] = 0;
    __syncthreads();
    bool bad = false;
    for (int f = threadIdx.x; f < count; f += kPlanBlock) {
        const Fork x = f < kPlanBlock ? mine : fork_at(c, parents, children, count, f);
        if (x.child_len != 0) bad = true;
        else bad |= (atomicOr(&child[x.child >> 5], 1u << (x.child & 31)) >> (x.child & 31) & 1) != 0;
    }
    bad = __syncthreads_or(bad);
    int need = 0;
    if (!bad) {
        for (int f = threadIdx.x; f < count; f += kPlanBlock) {
            const Fork x = f < kPlanBlock ? mine : fork_at(c, parents, children, count, f);
            if (x.len < 0 || x.len > paged_capacity(c) || (child[x.parent >> 5] >> (x.parent & 31) & 1)) {
                bad = true;
            } else if (x.full * (int)c.slots < x.len) {
                bad |= x.page < 0 || x.page >= c.pages;
                ++need;
            }
        }
        bad = __syncthreads_or(bad);
    }
    if (!bad) {
        const int t = threadIdx.x;
        for (int base = 0; base < count; base += kPlanBlock) {
            const int f = base + t;
            const Fork x = base == 0 ? mine : fork_at(c, parents, children, count, f);
            const bool first_of = f < count && !(atomicOr(&parent[x.parent >> 5], 1u << (x.parent & 31)) >> (x.parent & 31) & 1);
            int all = 0;
            before[t] = block_before(first_of ? x.full : 0, lds, &all);  // at most 2^20 a fork
            row[t] = x.parent;
            __syncthreads();
#pragma unroll 4
            for (int r = t; r < all; r += kPlanBlock) {
                const int lo = last_at_most(before, r);
                const int p = c.table[row[lo] * c.table_stride + r - before[lo]];
                bad |= p < 0 || p >= c.pages;
            }
            __syncthreads();  // the next forks' entries
        }
        bad = __syncthreads_or(bad);
    }
    int total = 0;
    (void)block_before(need, lds, &total);
    if (bad || total > c.pages ||
        each_page(c, first, 0, c.pages, true, total, lds, [&](int p, int rank, int) { free_pages.put(rank, p); }) < total) {
        if (threadIdx.x == 0) raise(c);
        return;
    }
    int given = 0;
    for (int base = 0; base < count; base += kPlanBlock) {
        const int f = base + (int)threadIdx.x;
        const Fork x = base == 0 ? mine : fork_at(c, parents, children, count, f);
        const bool part = f < count && x.full * (int)c.slots < x.len;
        int all = 0;
        const int at = given + block_before(part, lds, &all);
        if (f < count) {
            src[f] = -1;
            if (part) {
                const int p = free_pages.get(at);
                src[f] = x.page;
                dst[f] = p;
                c.table[x.child * c.table_stride + x.full] = p;
                c.refs[p] = 1;
            }
            c.lens[x.child] = x.len;
        }
        given += all;
    }
    if (threadIdx.x == 0) *result = count;
}

// The first `count` workgroups each copy one child's table row and count its references; all of them copy pages.
__global__ __launch_bounds__(kCopyBlock) void paged_fork_kernel(PagedView c, const int32_t* parents, const int32_t* children,
                                                                const int32_t* src, const int32_t* dst, const int32_t* result,
                                                                int elem, int dense_k, int dense_v) {
    const int count = *result;
    for (int f = blockIdx.x; f < count; f += gridDim.x) {
        const int s = parents[f], ch = children[f], full = (int)page_of(c, c.lens[ch]);
        for (int i = threadIdx.x; i < full; i += kCopyBlock) {
            const int p = c.table[s * c.table_stride + i];  // the plan has checked it
            c.table[ch * c.table_stride + i] = p;
            atomicAdd(c.refs + p, 1);
        }
    }
    copy_pages(c, src, dst, count, elem, dense_k, dense_v, blockIdx.x, gridDim.x);
}

// --------------------------------------------------------------------------------------------- free

// One workgroup per listed sequence; the first to take its length (an exchange with 0 of what it has checked) gives its pages back.
__global__ __launch_bounds__(kCopyBlock) void paged_free_kernel(PagedView c, const int32_t* sequences, int count) {
    __shared__ int had;
    for (int f = blockIdx.x; f < count; f += gridDim.x) {
        const int s = sequences[f];
        __syncthreads();
        if (threadIdx.x == 0) {
            const int len = s >= 0 && s < c.sequences ? c.lens[s] : -1;
            const bool bad = len < 0 || len > paged_capacity(c);
            if (bad) raise(c);
            had = bad || atomicCAS(c.lens + s, len, 0) != len ? 0 : len;  // taken by an equal entry: nothing is left
        }
        __syncthreads();
        const int len = had;
        for (int i = threadIdx.x; i < pages_of(c, len); i += kCopyBlock) {
            const int p = c.table[s * c.table_stride + i];
            if (p < 0 || p >= c.pages) raise(c);
            else if (atomicSub(c.refs + p, 1) <= 0) {  // the count was wrong: a free page stays at 0
                atomicAdd(c.refs + p, 1);
                raise(c);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------- compact

// list: place[p] for every page from the number of live pages on (where page p goes, itself if it does not move), and
// behind kPagedMaxPages the targets and sources of the moves; result: the number of live pages, and of moves. A length that is
// out of range refuses the call: nobody could say which entries of that table follow their pages.
__global__ __launch_bounds__(kPlanBlock) void paged_compact_plan_kernel(PagedView c, int32_t* place, int32_t* src, int32_t* dst,
                                                                        int32_t* result) {
    __shared__ uint64_t sums[kPlanWaves];
    __shared__ int lds[2 * kWave], few[kFew];
    const PageList targets = {few, dst};
    const Counts first = counts_at(c, 0);
    bool bad = false;
    for (int s = threadIdx.x; s < c.sequences; s += kPlanBlock) bad |= c.lens[s] < 0 || c.lens[s] > paged_capacity(c);
    uint64_t n = 0;
    for (int base = 0; base < c.pages; base += kStepPages) {
        Counts v = first;
        if (base) v = counts_at(c, base);
#pragma unroll
        for (int j = 0; j < kPer; ++j) n += v.r[j] > 0;
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) {
            result[1] = 0;
            raise(c);
        }
        return;
    }
    const int live = (int)block_sum(n, sums);
    for (int p = live + (int)threadIdx.x; p < c.pages; p += kPlanBlock) place[p] = p;
    const int moves = each_page(c, first, 0, live, true, live, lds, [&](int p, int rank, int) {
        targets.put(rank, p);
        if (rank < kFew) dst[rank] = p;
    });
    // as many live pages lie behind `live` as free ones before it
    each_page(c, first, live, c.pages, false, moves, lds, [&](int p, int rank, int count) {
        const int to = targets.get(rank);
        src[rank] = p;
        place[p] = to;
        c.refs[to] = count;
        c.refs[p] = 0;
    });
    if (threadIdx.x == 0) {
        result[0] = live;
        result[1] = moves;
    }
}

__global__ __launch_bounds__(kCopyBlock) void paged_compact_kernel(PagedView c, const int32_t* place, const int32_t* src,
                                                                   const int32_t* dst, const int32_t* result, int elem,
                                                                   int dense_k, int dense_v) {
    const int live = result[0], moves = result[1];
    if (!moves) return;
    for (int s = blockIdx.x; s < c.sequences; s += gridDim.x) {
        const int pages = pages_of(c, c.lens[s]);
        for (int i = threadIdx.x; i < pages; i += kCopyBlock) {
            const int p = c.table[s * c.table_stride + i];
            if (p < 0 || p >= c.pages) raise(c);
            else if (p >= live) c.table[s * c.table_stride + i] = place[p];
        }
    }
    copy_pages(c, src, dst, moves, elem, dense_k, dense_v, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------------------------------- commit

// A workgroup has a thread per node of its sequence: the nodes that the accepted one sees, in order, become positions base, base + 1, ... of the
// sequence, base the positions before the tree. The first of them may be there already (`still` of them); the others move, one after the
// other and eight at a time read before they are written: a target lies before its source, and so before every later source. A unit of
// work is a layer's K or V and 256 chunks of 16 bytes of a position: its chunks of all moves are the same lanes', so no lane waits for another.
// Every workgroup of a sequence finds the moves for itself; the last of them to arrive, when all have read the state, writes it: the length,
// and the counts of the pages behind it, which are the sequence's alone. A sequence that breaks a rule has no moves and keeps its state.
// Latency bounds it: starts, then the leaf's mask and the pages, their counts, the moves, the arrival. 8 layers of one path 5.6 us, 60 paths of 10
// layers, 20 MB read and written, 8.8; a plan and the moves as two launches 3.3 + 4.0 and 4.0 + 6.3, and 15.5 us a call for 12.5 by the host.
__host__ __device__ inline int commit_units(const PagedView& c, int elem) {
    return 2 * c.layers * ((c.kv_heads * c.head_dim * elem / 16 + kCopyBlock - 1) / kCopyBlock);
}

__global__ __launch_bounds__(kCopyBlock) void paged_commit_kernel(PagedView c, const int32_t* starts, const uint64_t* masks, int words,
                                                                  const int32_t* leaves, int rows, int first, uint32_t* tickets, int elem) {
    static_assert(kCopyBlock == kTreeMaxNodes, "a thread per node");
    __shared__ int2 place[kTreeMaxNodes];  // page and slot of every node
    __shared__ uint8_t from[kTreeMaxNodes];  // the nodes that move
    const int s = first + blockIdx.y, i = threadIdx.x;
    const int row0 = starts[s], end = starts[s + 1], len = c.lens[s], leaf = leaves[s];
    if (row0 == end) return;
    // (in this order: differences only of values that are in range)
    if (!rows_in_range(row0, end, rows, 64 * words) || len < end - row0 || len > paged_capacity(c) || leaf < -1 || leaf >= end - row0) {
        if (i == 0 && blockIdx.x == 0) raise(c);
        return;
    }
    const int n = end - row0, base = len - n;
    const int32_t* table = c.table + s * c.table_stride;
    int rank = 0, kept = 0;
    bool mine = false, bad = false;
    for (int w = 0; w < words && leaf >= 0; ++w) {
        uint64_t m = masks[(int64_t)(row0 + leaf) * words + w];
        const int left = n - 64 * w;
        m &= left >= 64 ? ~0ull : (left > 0 ? (1ull << left) - 1 : 0);
        kept += __popcll(m);
        if (i >> 6 > w) rank += __popcll(m);
        if (i >> 6 == w) rank += __popcll(m & ((1ull << (i & 63)) - 1)), mine = m >> (i & 63) & 1;
    }
    if (i < n) {
        const int column = (int)page_of(c, base + i), page = table[column];
        bad = page < 0 || page >= c.pages || c.refs[page] != 1;
        place[i] = make_int2(page, base + i - column * (int)c.slots);
    }
    bad = __syncthreads_or(bad);
    // (a rank is at most the node's number, and once below stays below)
    const int still = __syncthreads_count(mine && rank == i), moves = bad ? 0 : kept - still;
    if (mine && rank != i) from[rank - still] = (uint8_t)i;
    __syncthreads();
    const int units = commit_units(c, elem), parts = units / (2 * c.layers), per_head = c.head_dim * elem / 16;
    for (int u = blockIdx.x; u < units && moves; u += gridDim.x) {
        const int tensor = u / parts, chunk = (u - tensor * parts) * kCopyBlock + i;
        if (chunk >= c.kv_heads * per_head) continue;
        const bool v = tensor & 1;
        const int h = chunk / per_head;
        uint8_t* at = (v ? c.v + (int64_t)(tensor >> 1) * c.v_layer + h * c.v_head : c.k + (int64_t)(tensor >> 1) * c.k_layer + h * c.k_head) +
                      (chunk - h * per_head) * 16;
        const int64_t page = v ? c.v_page : c.k_page, slot = v ? c.v_slot : c.k_slot;
        for (int m0 = 0; m0 < moves; m0 += 8) {
            uint4 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int2 x = place[from[min(m0 + j, moves - 1)]];
                w[j] = ld16(at + x.x * page + x.y * slot);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int2 x = place[still + min(m0 + j, moves - 1)];
                if (m0 + j < moves) *reinterpret_cast<uint4*>(at + x.x * page + x.y * slot) = w[j];
            }
        }
    }
    if (!arrive_last<kRowTurn>(tickets + (int64_t)blockIdx.y * kTicketStride, blockIdx.x == 0, gridDim.x)) return;
    if (bad) {
        if (i == 0) raise(c);
        return;
    }
    if (i == 0) c.lens[s] = base + kept;
    for (int x = pages_of(c, base + kept) + i; x < pages_of(c, len); x += kTreeMaxNodes) c.refs[table[x]] = 0;
}

// ------------------------------------------------------------------------------------------ reorder

// Scratch of a reorder, in the page lists: the lengths before it; of every sequence the copy of its parent's last page that it gets
// (-1: none); source, target and slots in use of every copy; pages of dropped sequences and free ones behind the first kFew.
struct ReorderLists {
    int32_t *lens, *copy, *src, *dst, *used, *more, *result;
    __device__ explicit ReorderLists(int32_t* list)
        : lens(list), copy(list + kPagedMaxSequences), src(list + 2 * kPagedMaxSequences), dst(list + 3 * kPagedMaxSequences),
          used(list + 4 * kPagedMaxSequences), more(list + 5 * kPagedMaxSequences), result(list + 2 * kPagedMaxPages) {}
};
static_assert(7 * kPagedMaxSequences < 2 * kPagedMaxPages, "a reorder's lists fit the page lists");

// One workgroup, whole groups of beams at a time. A parent's partly filled last page stays with its keeper: the parent itself if it is its
// own child, else its first child. Every other child gets a copy, in the order of the sequences: in the partly filled last pages of the
// sequences that are nobody's parents, where those were theirs alone, then in the lowest free pages. result: the copies, or -1. Latency bounds
// it, a chain of lengths, table entries, counts and the workgroup's scans: 6.8 us for 4 beams, 8.4 for 12 groups of 8. Taking the pages that
// dropped sequences leave first spares the pass over the pool's counts while beams are as long as each other.
struct Beam { int parent, len, parent_len, last; bool copies, dropped; };

__global__ __launch_bounds__(kPlanBlock) void paged_reorder_plan_kernel(PagedView c, const int32_t* parents, int count, int beams, int32_t* list) {
    __shared__ int lds[2 * kWave], few[kFew], par[kPlanBlock], len[kPlanBlock];
    const ReorderLists l(list);
    const PageList pages = {few, l.more};
    const Counts first = counts_at(c, 0);
    const int t = threadIdx.x, step = kPlanBlock / beams * beams;
    // sequence base + t's part; the workgroup's lists are those of the step
    auto beam_at = [&](int base, bool* bad) {
        Beam b = {-1, 0, 0, -1, false, false};
        const int s = base + t;
        const bool in = t < step && s < count;
        __syncthreads();  // the step before has read the lists
        if (in) {
            b.parent = parents[s];
            b.len = c.lens[s];
            const int g = s / beams * beams;
            if (b.parent < g || b.parent >= g + beams || b.len < 0 || b.len > paged_capacity(c)) {
                *bad = true;
                b.parent = s;
                b.len = 0;
            }
            par[t] = b.parent;
            len[t] = b.len;
        }
        __syncthreads();
        if (!in) return b;
        const int g = t / beams * beams, p = b.parent - base;
        bool chosen = false;
        b.copies = b.parent != s && par[p] == b.parent;
        for (int i = g; i < g + beams; ++i) {
            chosen |= par[i] == s;
            b.copies |= i < t && par[i] == b.parent && b.parent != s;
        }
        b.parent_len = len[p];
        b.copies &= b.parent_len % (int)c.slots != 0;
        b.dropped = !chosen && b.len % (int)c.slots != 0;
        if (b.copies) {
            b.last = c.table[b.parent * c.table_stride + b.parent_len / (int)c.slots];
            *bad |= b.last < 0 || b.last >= c.pages;
        }
        return b;
    };
    bool bad = false;
    int copies = 0, dropped = 0;
    Beam b = {-1, 0, 0, -1, false, false};
    for (int base = 0; base < count; base += step) {
        b = beam_at(base, &bad);
        int page = -1, all = 0;
        if (b.dropped) {
            page = c.table[(base + t) * c.table_stride + b.len / (int)c.slots];
            if (page < 0 || page >= c.pages || c.refs[page] != 1) page = -1;
        }
        const int at = dropped + block_before(page >= 0, lds, &all);
        if (page >= 0) pages.put(at, page);
        dropped += all;
        (void)block_before(b.copies, lds, &all);
        copies += all;
        if (t < step && base + t < count) l.lens[base + t] = b.len;
    }
    bad = __syncthreads_or(bad);
    const int more = copies - dropped;
    if (bad || (more > 0 && each_page(c, first, 0, c.pages, true, more, lds, [&](int p, int rank, int) { pages.put(dropped + rank, p); }) < more)) {
        if (t == 0) {
            *l.result = -1;
            raise(c);
        }
        return;
    }
    int given = 0;
    for (int base = 0; base < count; base += step) {
        if (count > step) b = beam_at(base, &bad);  // (the only step's are still here)
        int all = 0;
        const int at = given + block_before(b.copies, lds, &all);
        if (t < step && base + t < count) {
            const int p = b.copies ? pages.get(at) : -1;
            l.copy[base + t] = p;
            if (b.copies) {
                l.src[at] = b.last;
                l.dst[at] = p;
                l.used[at] = b.parent_len % (int)c.slots;
            }
            if (b.parent != base + t) c.lens[base + t] = b.parent_len;  // (the step's lengths have been read)
        }
        given += all;
    }
    if (t == 0) *l.result = copies;
}

constexpr int kReorderColumns = 64;

// A workgroup takes 64 columns of a group's table rows, all of them read before any is written; a page's count follows the entries that
// name it. All workgroups copy the slots in use of the pages that are copied, 16 KB in flight each (12 groups of 8 over 6 layers, 79 MB read
// and written, 18.8 us).
__global__ __launch_bounds__(kCopyBlock) void paged_reorder_kernel(PagedView c, const int32_t* parents, int count, int beams, int32_t* list, int elem) {
    __shared__ int32_t entry[kMaxBeams][kReorderColumns];
    __shared__ int par[kMaxBeams], len[kMaxBeams];
    const ReorderLists l(list);
    const int copies = *l.result;
    if (copies < 0) return;
    const int slices = (c.columns + kReorderColumns - 1) / kReorderColumns, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tables = (int64_t)(count / beams) * slices;
    for (int64_t u = blockIdx.x; u < tables; u += gridDim.x) {
        const int g = (int)(u / slices) * beams, i = (int)(u % slices) * kReorderColumns + lane;
        __syncthreads();
        bool moves = false;
        if ((int)threadIdx.x < beams) {
            par[threadIdx.x] = parents[g + threadIdx.x] - g;
            len[threadIdx.x] = l.lens[g + threadIdx.x];
            moves = par[threadIdx.x] != (int)threadIdx.x;
        }
        if (!__syncthreads_or(moves)) continue;
        for (int b = wave; b < beams; b += 4)
            entry[b][lane] = i < pages_of(c, len[b]) ? c.table[(g + b) * c.table_stride + i] : -1;
        __syncthreads();
        for (int b = wave; b < beams; b += 4) {
            const int p = par[b];
            if (p == b) continue;
            const int had = pages_of(c, len[b]), has = pages_of(c, len[p]), copy = l.copy[g + b];
            const int old = entry[b][lane], now = copy >= 0 && i == has - 1 ? copy : entry[p][lane];
            if (i < has) c.table[(g + b) * c.table_stride + i] = now;
            if (i < had && i < has && old == now) continue;
            if (i < has) {
                if (now < 0 || now >= c.pages) raise(c);
                else atomicAdd(c.refs + now, 1);
            }
            if (i < had) {
                if (old < 0 || old >= c.pages) raise(c);
                else if (atomicSub(c.refs + old, 1) <= 0) {  // the count was wrong: a free page stays at 0
                    atomicAdd(c.refs + old, 1);
                    raise(c);
                }
            }
        }
    }
    const uint32_t per_row = (uint32_t)(c.head_dim * elem / 16), chunks = c.slots * (uint32_t)c.kv_heads * per_row;
    const uint32_t parts = (chunks + kCopyBytes / 16 - 1) / (kCopyBytes / 16);
    const uint64_t per_move = (uint64_t)parts * 2 * c.layers;
    for (uint64_t u = blockIdx.x; u < per_move * copies; u += gridDim.x) {
        const int m = (int)(u / per_move);
        const uint32_t r = (uint32_t)(u - m * per_move), tensor = r / parts, i0 = (r - tensor * parts) * (kCopyBytes / 16) + threadIdx.x;
        const uint32_t used = l.used[m] * (uint32_t)c.kv_heads * per_row;
        const bool v = tensor & 1;
        uint8_t* base = v ? c.v + (int64_t)(tensor >> 1) * c.v_layer : c.k + (int64_t)(tensor >> 1) * c.k_layer;
        const int64_t page = v ? c.v_page : c.k_page, slot = v ? c.v_slot : c.k_slot, head = v ? c.v_head : c.k_head;
        const uint8_t* a = base + l.src[m] * page;
        uint8_t* b = base + l.dst[m] * page;
        const bool dense = head == c.head_dim * elem && slot == (int64_t)c.kv_heads * head;
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * kCopyBlock < used) w[j] = ld16(a + chunk_at(dense, i0 + j * kCopyBlock, per_row, c.kv_heads, slot, head));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * kCopyBlock < used)
                *reinterpret_cast<uint4*>(b + chunk_at(dense, i0 + j * kCopyBlock, per_row, c.kv_heads, slot, head)) = w[j];
    }
}

// -------------------------------------------------------------------------------------------- append

// One wave per row: it finds the row's sequence, then moves K and V, 8 elements a lane and step. Bound by memory: 10500
// rows of 8 heads of 128 into E4M3 pages (65 MB) 17 us a layer, 3.8 TB/s; the other waves of a CU hide a wave's own steps
// (loads sent ahead of the search, or a residual step in the division's place: 1 us more).
template <bool E4M3>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedView c, const uint16_t* k, int64_t k_row, const uint16_t* v,
                                                           int64_t v_row, const int32_t* starts, int rows) {
    const int lane = threadIdx.x & 63, m = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (m >= rows) return;
    const int s = sequence_of(starts, c.sequences, m);
    if (s < 0 || s >= c.sequences) return;
    const int end = starts[s + 1], len = c.lens[s], cap = paged_capacity(c);
    // (end <= m: starts that descend. Only then is the difference sure to fit.)
    const int t = end > m && end <= rows && len >= 0 && len <= cap ? len - (end - m) : -1;
    if (t < 0) {
        if (lane == 0) raise(c);
        return;
    }
    const uint32_t i = page_of(c, t), slot = t - i * c.slots;
    const int p = c.table[s * c.table_stride + i];
    if (p < 0 || p >= c.pages) {
        if (lane == 0) raise(c);
        return;
    }
    const int log = __builtin_ctz(c.head_dim / 8), chunks = c.kv_heads << log;  // head_dim / 8 chunks a head
    uint8_t* kp = c.k + p * c.k_page + slot * c.k_slot;
    uint8_t* vp = c.v + p * c.v_page + slot * c.v_slot;
    for (int x = lane; x < 2 * chunks; x += 64) {
        const bool is_v = x >= chunks;
        const int y = is_v ? x - chunks : x, h = y >> log, at = (y - (h << log)) * 8;
        const uint4 w = ld16((is_v ? v + m * v_row : k + m * k_row) + (int64_t)y * 8);
        uint8_t* to = is_v ? vp + h * c.v_head : kp + h * c.k_head;
        if (!E4M3) {
            *reinterpret_cast<uint4*>(to + at * 2) = w;
        } else {
            const float f = is_v ? c.v_scale[h] : c.k_scale[h];
            float e[8];
            bf16x8_to_f32(w, e);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                e[j] = __fdiv_rn(e[j], f);
                e[j] = e[j] > 448.0f ? 448.0f : (e[j] < -448.0f ? -448.0f : e[j]);  // a NaN stays one
            }
            uint32_t lo = __builtin_amdgcn_cvt_pk_fp8_f32(e[0], e[1], 0, false);
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(e[2], e[3], lo, true);
            uint32_t hi = __builtin_amdgcn_cvt_pk_fp8_f32(e[4], e[5], 0, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(e[6], e[7], hi, true);
            *reinterpret_cast<uint2*>(to + at) = make_uint2(lo, hi);
        }
    }
}

// ------------------------------------------------------------------------------------ host: the checks

int elem_bytes(const moa_paged_cache* c) { return c->element == MOA_PAGES_BF16 ? 2 : 1; }

// Strides of one tensor: multiples of 16 bytes, at least a head, within 2^46 elements over the whole tensor.
int check_strides(const int64_t* st, const moa_paged_cache* c, const char* name) {
    static const char* dims[4] = {"layer", "page", "slot", "head"};
    const int64_t size[4] = {c->layers, c->pages, c->slots, c->kv_heads};
    for (int i = 0; i < 4; ++i) {
        if (size[i] == 1) continue;
        if (st[i] < c->head_dim || st[i] % (16 / elem_bytes(c)) || st[i] > (int64_t(1) << 46) / size[i])
            return bad_value(std::string(name) + ": the " + dims[i] + " stride must be a multiple of 16 bytes, at least head_dim, got " +
                             std::to_string(st[i]) + " elements");
    }
    return MOA_SUCCESS;
}

// The checks of a cache and, with the call's layer, the view its kernels get.
int cache_view(const moa_paged_cache* c, int layer, PagedView* v) {
    if (!c) return bad_value("cache is NULL");
    int e;
    if ((e = check_range(c->layers, 1, 1024, "layers")) || (e = check_range(c->pages, 1, kPagedMaxPages, "pages")) ||
        (e = check_range(c->slots, 1, 65536, "slots")) || (e = check_range(c->kv_heads, 1, 256, "kv_heads")) ||
        (e = check_range(c->element, MOA_PAGES_BF16, MOA_PAGES_E4M3, "element")) ||
        (e = check_range(c->sequences, 1, kPagedMaxSequences, "sequences")) ||
        (e = check_range(c->columns, 1, 1 << 20, "columns")) || (e = check_range(layer, 0, c->layers - 1, "layer")))
        return e;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256 && c->head_dim != 512)
        return bad_value("head_dim must be 64, 128, 256 or 512, got " + std::to_string(c->head_dim));
    if ((int64_t)c->columns * c->slots > (1 << 30)) return bad_value("columns * slots must be at most 2^30");
    if (c->table_stride < c->columns || c->table_stride > (int64_t(1) << 40))
        return bad_value("table_stride must be at least columns, got " + std::to_string(c->table_stride));
    if ((e = check_ptr(c->k_pages, "k_pages", 16)) || (e = check_ptr(c->v_pages, "v_pages", 16)) ||
        (e = check_ptr(c->page_table, "page_table", 4)) || (e = check_ptr(c->seq_lens, "seq_lens", 4)) ||
        (e = check_ptr(c->ref_counts, "ref_counts", 4)))
        return e;
    if (c->element == MOA_PAGES_E4M3) {
        if ((e = check_ptr(c->k_scale, "k_scale", 4)) || (e = check_ptr(c->v_scale, "v_scale", 4))) return e;
    } else if (c->k_scale || c->v_scale) {
        return bad_value("bf16 pages have no scales: k_scale and v_scale must be NULL");
    }
    if ((e = check_strides(c->k_stride, c, "k_pages")) || (e = check_strides(c->v_stride, c, "v_pages"))) return e;
    const int b = elem_bytes(c);
    const bool e4 = c->element == MOA_PAGES_E4M3;
    v->k_layer = c->k_stride[0] * b, v->k_page = c->k_stride[1] * b, v->k_slot = c->k_stride[2] * b, v->k_head = c->k_stride[3] * b;
    v->v_layer = c->v_stride[0] * b, v->v_page = c->v_stride[1] * b, v->v_slot = c->v_stride[2] * b, v->v_head = c->v_stride[3] * b;
    v->k = static_cast<uint8_t*>(c->k_pages) + layer * v->k_layer;
    v->v = static_cast<uint8_t*>(c->v_pages) + layer * v->v_layer;
    v->k_scale = e4 ? c->k_scale + (size_t)layer * c->kv_heads : nullptr;
    v->v_scale = e4 ? c->v_scale + (size_t)layer * c->kv_heads : nullptr;
    v->table = c->page_table, v->lens = c->seq_lens, v->refs = c->ref_counts;
    v->table_stride = c->table_stride;
    v->slots = (uint32_t)c->slots;
    uint32_t log = 0;
    while ((1 << log) < c->slots) ++log;
    v->shift = 31 + log;
    v->magic = (uint32_t)((uint64_t(1) << v->shift) / (uint32_t)c->slots + 1);
    v->layers = c->layers, v->pages = c->pages, v->kv_heads = c->kv_heads, v->head_dim = c->head_dim;
    v->sequences = c->sequences, v->columns = c->columns;
    auto reach = [&](const int64_t* st) {  // bytes from the first element of a layer to behind its last
        return ((c->pages - 1) * st[1] + (c->slots - 1) * st[2] + (c->kv_heads - 1) * st[3] + c->head_dim) * b;
    };
    v->near = reach(c->k_stride) < (int64_t(1) << 32) && reach(c->v_stride) < (int64_t(1) << 32);
    v->alike = v->k_page == v->v_page && v->k_slot == v->v_slot;
    v->err = nullptr;
    return MOA_SUCCESS;
}

// Whether a page's rows fill it without gaps, slots outside heads or heads outside slots.
int dense_page(const moa_paged_cache* c, const int64_t* st) {
    const int64_t d = c->head_dim;
    const int64_t slot = c->slots == 1 ? c->kv_heads * d : st[2], head = c->kv_heads == 1 ? d : st[3];
    return (head == d && slot == c->kv_heads * d) || (slot == d && st[3] == c->slots * d);
}

int64_t copy_units(const moa_paged_cache* c, int64_t moves) {
    const int64_t bytes = (int64_t)c->slots * c->kv_heads * c->head_dim * elem_bytes(c);
    return moves * ((bytes + kCopyBytes - 1) / kCopyBytes) * 2 * c->layers;
}

// Workgroups of a copy launch: one per unit of work, up to the eight of 256 threads that a CU holds; more would
// only wait.
int copy_grid(int64_t units, int cus) {
    const int64_t most = (int64_t)cus * 8;
    return (int)(units < 1 ? 1 : (units < most ? units : most));
}

// The checks of both attention calls; of a call without rows only those of its numbers.
int check_attention(const uint16_t* q, int64_t q_row_stride, const moa_paged_cache* cache, const int32_t* row_starts, const uint16_t* out,
                    int64_t out_row_stride, int rows, int q_heads, int layer, int window, float scale, int max_rows, PagedView* v) {
    int e;
    if ((e = cache_view(cache, layer, v)) || (e = check_range(rows, 0, 1 << 20, "rows")) ||
        (e = check_range(q_heads, 1, 1 << 15, "q_heads")) || (e = check_range(window, 0, 1 << 30, "window")))
        return e;
    if (q_heads % v->kv_heads || q_heads / v->kv_heads > 128)
        return bad_value("q_heads must be kv_heads times 1 .. 128, got " + std::to_string(q_heads) + " and " + std::to_string(v->kv_heads));
    if (!(scale > -1e30f && scale < 1e30f)) return bad_value("scale must be finite and below 1e30");
    if (rows == 0) return MOA_SUCCESS;
    if ((e = check_range(max_rows, 1, rows, "max_rows")) || (e = check_ptr(q, "q", 16)) || (e = check_ptr(out, "out", 16)) ||
        (e = check_ptr(row_starts, "row_starts", 4)))
        return e;
    const int64_t width = (int64_t)q_heads * v->head_dim;
    for (const int64_t st : {q_row_stride, out_row_stride})
        if (rows > 1 && (st < width || st % 8 || st > (int64_t(1) << 40)))
            return bad_value("q and out row strides must be multiples of 8 elements and at least q_heads * head_dim, got " + std::to_string(st));
    return MOA_SUCCESS;
}

}  // namespace
}  // namespace moa

using namespace moa;

extern "C" {

int moa_paged_cache_reserve(const moa_paged_cache* cache, const int32_t* new_tokens, void* stream) {
    PagedView v;
    int e;
    if ((e = cache_view(cache, 0, &v)) || (e = check_ptr(new_tokens, "new_tokens", 4))) return e;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    hipLaunchKernelGGL(paged_reserve_kernel, dim3(1), dim3(kPlanBlock), 0, static_cast<hipStream_t>(stream), v, new_tokens,
                       ctx->paged_list);
    return call_result(hipGetLastError(), "paged_cache_reserve launch");
}

int moa_paged_cache_append(const moa_paged_cache* cache, const uint16_t* k, int64_t k_row_stride, const uint16_t* v_rows,
                           int64_t v_row_stride, const int32_t* row_starts, int rows, int layer, void* stream) {
    PagedView v;
    int e;
    if ((e = cache_view(cache, layer, &v)) || (e = check_range(rows, 0, 1 << 20, "rows"))) return e;
    if (rows == 0) return MOA_SUCCESS;
    if ((e = check_ptr(k, "k", 16)) || (e = check_ptr(v_rows, "v", 16)) || (e = check_ptr(row_starts, "row_starts", 4))) return e;
    const int64_t width = (int64_t)v.kv_heads * v.head_dim;
    for (const int64_t st : {k_row_stride, v_row_stride})
        if (rows > 1 && (st < width || st % 8 || st > (int64_t(1) << 40)))
            return bad_value("k and v row strides must be multiples of 8 elements and at least kv_heads * head_dim, got " + std::to_string(st));
    DevCtx* ctx = call_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    auto* f = cache->element == MOA_PAGES_E4M3 ? paged_append_kernel<true> : paged_append_kernel<false>;
    hipLaunchKernelGGL(f, dim3((rows + 3) / 4), dim3(256), 0, static_cast<hipStream_t>(stream), v, k, k_row_stride, v_rows,
                       v_row_stride, row_starts, rows);
    return call_result(hipGetLastError(), "paged_cache_append launch");
}

int moa_paged_cache_fork(const moa_paged_cache* cache, const int32_t* parents, const int32_t* children, int count, void* stream) {
    PagedView v;
    int e;
    if ((e = cache_view(cache, 0, &v)) || (e = check_range(count, 0, kPagedMaxSequences, "count"))) return e;
    if (count == 0) return MOA_SUCCESS;
    if ((e = check_ptr(parents, "parents", 4)) || (e = check_ptr(children, "children", 4))) return e;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    int32_t *src = ctx->paged_list, *dst = src + kPagedMaxPages, *result = dst + kPagedMaxPages;
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(paged_fork_plan_kernel, dim3(1), dim3(kPlanBlock), 0, s, v, parents, children, count, src, dst, result);
    e = call_result(hipGetLastError(), "paged_cache_fork launch");
    if (e) return e;
    hipLaunchKernelGGL(paged_fork_kernel, dim3(copy_grid(copy_units(cache, count), ctx->cus)), dim3(kCopyBlock), 0, s, v, parents,
                       children, src, dst, result, elem_bytes(cache), dense_page(cache, cache->k_stride),
                       dense_page(cache, cache->v_stride));
    return call_result(hipGetLastError(), "paged_cache_fork launch");
}

int moa_paged_cache_free(const moa_paged_cache* cache, const int32_t* sequences, int count, void* stream) {
    PagedView v;
    int e;
    if ((e = cache_view(cache, 0, &v)) || (e = check_range(count, 0, 1 << 20, "count"))) return e;
    if (count == 0) return MOA_SUCCESS;
    if ((e = check_ptr(sequences, "sequences", 4))) return e;
    DevCtx* ctx = call_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    hipLaunchKernelGGL(paged_free_kernel, dim3(count < 4096 ? count : 4096), dim3(kCopyBlock), 0, static_cast<hipStream_t>(stream), v,
                       sequences, count);
    return call_result(hipGetLastError(), "paged_cache_free launch");
}

int moa_paged_cache_compact(const moa_paged_cache* cache, void* stream) {
    PagedView v;
    int e;
    if ((e = cache_view(cache, 0, &v))) return e;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    // at most half of the pages move: their sources and targets share the second list
    int32_t *place = ctx->paged_list, *src = place + kPagedMaxPages, *dst = src + kPagedMaxPages / 2, *result = src + kPagedMaxPages;
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(paged_compact_plan_kernel, dim3(1), dim3(kPlanBlock), 0, s, v, place, src, dst, result);
    e = call_result(hipGetLastError(), "paged_cache_compact launch");
    if (e) return e;
    const int64_t units = copy_units(cache, cache->pages / 2);
    hipLaunchKernelGGL(paged_compact_kernel, dim3(copy_grid(units < cache->sequences ? cache->sequences : units, ctx->cus)),
                       dim3(kCopyBlock), 0, s, v, place, src, dst, result, elem_bytes(cache), dense_page(cache, cache->k_stride),
                       dense_page(cache, cache->v_stride));
    return call_result(hipGetLastError(), "paged_cache_compact launch");
}

int moa_paged_attention(const uint16_t* q, int64_t q_row_stride, const moa_paged_cache* cache, const int32_t* row_starts,
                        uint16_t* out, int64_t out_row_stride, int rows, int q_heads, int layer, int window, float scale,
                        int max_rows, void* stream) {
    PagedView v;
    int e;
    if ((e = check_attention(q, q_row_stride, cache, row_starts, out, out_row_stride, rows, q_heads, layer, window, scale, max_rows, &v)))
        return e;
    if (rows == 0) return MOA_SUCCESS;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    const PagedAttentionCall a{q, out, q_row_stride, out_row_stride, row_starts, rows, q_heads, q_heads / v.kv_heads,
                               window, max_rows, scale * 1.4426950408889634f};
    return call_result(launch_paged_attention(v, a, static_cast<hipStream_t>(stream), ctx), "paged_attention launch");
}

int moa_paged_tree_attention(const uint16_t* q, int64_t q_row_stride, const moa_paged_cache* cache, const int32_t* row_starts,
                             const uint64_t* masks, int mask_words, uint16_t* out, int64_t out_row_stride, int rows, int q_heads,
                             int layer, int window, float scale, int max_rows, void* stream) {
    PagedView v;
    int e;
    if ((e = check_attention(q, q_row_stride, cache, row_starts, out, out_row_stride, rows, q_heads, layer, window, scale, max_rows, &v)) ||
        (e = check_range(mask_words, 1, kTreeMaxWords, "mask_words")))
        return e;
    if (rows == 0) return MOA_SUCCESS;
    if ((e = check_ptr(masks, "masks", 8)) || (e = check_range(max_rows, 1, 64 * mask_words, "max_rows"))) return e;
    if (window && window < max_rows)
        return bad_value("window must be 0 or at least max_rows, got " + std::to_string(window) + " and " + std::to_string(max_rows));
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    PagedTreeCall a;
    static_cast<PagedAttentionCall&>(a) = {q, out, q_row_stride, out_row_stride, row_starts, rows, q_heads, q_heads / v.kv_heads,
                                           window, max_rows, scale * 1.4426950408889634f};
    a.masks = masks, a.words = mask_words;
    return call_result(launch_paged_tree_attention(v, a, static_cast<hipStream_t>(stream), ctx), "paged_tree_attention launch");
}

int moa_paged_tree_commit(const moa_paged_cache* cache, const int32_t* row_starts, const uint64_t* masks, int mask_words,
                          const int32_t* leaves, int rows, void* stream) {
    PagedView v;
    int e;
    if ((e = cache_view(cache, 0, &v)) || (e = check_range(rows, 0, 1 << 20, "rows")) ||
        (e = check_range(mask_words, 1, kTreeMaxWords, "mask_words")))
        return e;
    if (rows == 0) return MOA_SUCCESS;
    if ((e = check_ptr(row_starts, "row_starts", 4)) || (e = check_ptr(masks, "masks", 8)) || (e = check_ptr(leaves, "leaves", 4)))
        return e;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    hipStream_t s = static_cast<hipStream_t>(stream);
    // a counter for each of a launch's sequences; of few sequences, as many workgroups as there are units, below a turn
    for (int first = 0; first < v.sequences; first += kSearchRows) {
        const int here = std::min(kSearchRows, v.sequences - first), most = std::min(commit_units(v, elem_bytes(cache)), (int)kRowTurn / 2);
        hipLaunchKernelGGL(paged_commit_kernel, dim3(std::max(1, std::min(most, 8 * ctx->cus / here)), here), dim3(kCopyBlock), 0, s, v, row_starts, masks,
                           mask_words, leaves, rows, first, ctx->search_tickets + (size_t)kSearchRows * kTicketStride, elem_bytes(cache));
        if ((e = call_result(hipGetLastError(), "paged_tree_commit launch"))) return e;
    }
    return MOA_SUCCESS;
}

int moa_paged_cache_reorder(const moa_paged_cache* cache, const int32_t* parents, int count, int beams, void* stream) {
    PagedView v;
    int e;
    if ((e = cache_view(cache, 0, &v)) || (e = check_range(count, 0, v.sequences, "count")) ||
        (e = check_range(beams, 1, kMaxBeams, "beams")))
        return e;
    if (count % beams) return bad_value("count must be a multiple of beams, got " + std::to_string(count) + " and " + std::to_string(beams));
    if (count == 0) return MOA_SUCCESS;
    if ((e = check_ptr(parents, "parents", 4))) return e;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    v.err = ctx->err;
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(paged_reorder_plan_kernel, dim3(1), dim3(kPlanBlock), 0, s, v, parents, count, beams, ctx->paged_list);
    if ((e = call_result(hipGetLastError(), "paged_cache_reorder launch"))) return e;
    // at least one sequence of a group keeps its pages
    const int64_t copies = copy_units(cache, count - count / beams), tables = (int64_t)(count / beams) * ((v.columns + kReorderColumns - 1) / kReorderColumns);
    hipLaunchKernelGGL(paged_reorder_kernel, dim3(copy_grid(std::max(copies, tables), ctx->cus)), dim3(kCopyBlock), 0, s, v, parents, count,
                       beams, ctx->paged_list, elem_bytes(cache));
    return call_result(hipGetLastError(), "paged_cache_reorder launch");
}

}  // extern "C"
