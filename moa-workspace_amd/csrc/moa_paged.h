// moa_paged.h -- the paged cache as its kernels see it: one layer's (or the first layer's) pages, the
// table, and the page arithmetic they share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moa_internal.h"
#include "moa_paged_plan.h"

namespace moa {

struct PagedView {
    uint8_t* k; uint8_t* v;               // the layer's pages
    const float* k_scale; const float* v_scale;  // the layer's [kv_heads], or nullptr (bf16)
    int32_t* table; int32_t* lens; int32_t* refs;
    int64_t k_layer, k_page, k_slot, k_head;     // strides in bytes
    int64_t v_layer, v_page, v_slot, v_head;
    int64_t table_stride;
    uint32_t slots, magic, shift;         // t / slots = t * magic >> shift, for t < 2^31
    int32_t layers, pages, kv_heads, head_dim, sequences, columns;
    bool near;                            // every offset within a layer's K, and V, is below 2^32 bytes
    bool alike;                           // K's and V's pages and slots have the same strides
    uint32_t* err;
};

// t / slots for 0 <= t < 2^31: with shift = 31 + ceil(log2 slots) and magic = floor(2^shift / slots) + 1 (at most
// 32 bits) the quotient is exact (Granlund and Montgomery's division by invariant integers).
__device__ __forceinline__ uint32_t page_of(const PagedView& c, uint32_t t) {
    return (uint32_t)((uint64_t)t * c.magic >> c.shift);
}

// Positions a sequence can have: at most 2^30.
__device__ __forceinline__ int paged_capacity(const PagedView& c) { return c.columns * (int)c.slots; }

// The sequence that row m belongs to by its row starts [sequences + 1]: the last one that starts at or before m
// (-1: none does), found by the whole wave, 64 probes a step.
__device__ __forceinline__ int sequence_of(const int32_t* starts, int sequences, int m) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = sequences + 1;  // the answer + 1 is the number of starts <= m
    while (n > 64) {
        const int step = (n + 63) / 64, at = lo + lane * step;
        const int last = at < lo + n ? starts[at] : 0x7fffffff;
        const int c = __popcll(__ballot(last <= m));
        if (c == 0) return -1;
        lo += (c - 1) * step;
        n = min(step, sequences + 1 - lo);
    }
    const int s = lane < n ? starts[lo + lane] : 0x7fffffff;
    return lo + __popcll(__ballot(s <= m)) - 1;
}

struct PagedAttentionCall {
    const uint16_t* q; uint16_t* out;
    int64_t q_row, out_row;               // strides in elements
    const int32_t* starts;
    int rows, q_heads, group, window, max_rows;
    float scale_log2;                     // scale * log2 e
};

// Rows that are nodes of trees: masks [rows][words], bit j % 64 of word j / 64 of a row: it sees node j of its sequence.
struct PagedTreeCall : PagedAttentionCall {
    const uint64_t* masks;
    int words;
};

hipError_t launch_paged_attention(const PagedView& c, const PagedAttentionCall& a, hipStream_t s, DevCtx* ctx);
hipError_t launch_paged_tree_attention(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx);
// The kernels of few and of many rows a sequence, for trees.
hipError_t launch_paged_tree_rows(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx);

}  // namespace moa
