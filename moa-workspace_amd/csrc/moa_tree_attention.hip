// moa_tree_attention.hip -- attention of drafted trees over the paged cache (include/moa_paged.h) for sequences of a few dozen rows.
//
// Every row of a tree sees the positions before it, so one pass over K and V serves all rows of a sequence: up to 64 or 128 of them in a
// workgroup, 16 for each of its waves. K and V go through LDS, in a ring of tiles of 16 KB: the matrix cores and LDS have a third of the
// time that memory takes, so what counts is that loads never pause.
#include <algorithm>

#include "moa_tree_rows.h"

namespace moa {
namespace {

constexpr int kTreeRows = 64;  // of a tile up to 256 dims

// The units of kTokenUnit positions of all sequences' tiles, a sequence's tiles behind each other, are one row of U, dealt out evenly: group
// w of `groups` takes units [w q, (w + 1) q), q = ceil(U / groups), crossing from tile to tile. A part that is not its whole tile leaves a
// record: number 2 w where it begins inside its tile, 2 w + 1 where it begins it, so split j of a tile that begins in group w0 is
// record 2 (w0 + j) + (j == 0).
struct TreeWalk {
    int64_t units, q;  // U, q
    int base;          // the 64 sequences looked at
    int64_t before;    // units before them
    Seq last;          // the last 64 sequences' lanes, the only ones of most calls
};

// A split tile, for the merge: its sequence's rows, its number there, its parts. A group begins one at most: its last.
struct TreeSplit { int row0, n, tile, parts; };

// Inclusive sums of numbers below 2^50: the low 20 bits and the others apart.
__device__ __forceinline__ int64_t scan_sum64(int64_t x) { return ((int64_t)scan_sum((int)(x >> 20)) << 20) + scan_sum((int)(x & 0xfffff)); }
__device__ __forceinline__ int64_t lane64(int64_t v, int l) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, l));
}
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {  // of numbers that are not negative; real calls' fit 32 bits
    return (a | b) >> 31 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

__device__ __forceinline__ int tree_tiles(const PagedTreeCall& a, const Seq& q) { return (q.n * a.group + kTreeRows - 1) / kTreeRows; }

__device__ TreeWalk tree_walk(const PagedView& c, const PagedTreeCall& a, int groups, int align) {
    TreeWalk w = {0, 1, 0, 0, {0, 0, 0}};
    bool bad = false;
    for (int base = 0; base < c.sequences; base += 64) {
        w.last = seq_of<true>(c, a, base + (threadIdx.x & 63), true, &bad);
        w.units += (int64_t)tree_tiles(a, w.last) * token_units(a, w.last, align);
    }
    raise_bad(c, bad);
    w.units = lane64(scan_sum64(w.units), 63);
    w.q = quotient(w.units + groups - 1, groups);
    w.q = w.q ? w.q : 1;
    return w;
}

// The tile that unit u (not before an earlier call's) belongs to, its units and the first of them. u < w.units.
__device__ void tree_at(const PagedView& c, const PagedTreeCall& a, TreeWalk& w, int align, int64_t u, Piece* out, int* units, int64_t* first) {
    const int lane = threadIdx.x & 63;
    bool bad = false;
    for (;; w.base += 64) {
        Seq q = w.last;
        if (c.sequences > 64) q = seq_of<true>(c, a, w.base + lane, true, &bad);
        const int n = token_units(a, q, align);
        const int64_t all = (int64_t)tree_tiles(a, q) * n, x = scan_sum64(all), end = lane64(x, 63);
        if (w.base + 64 >= c.sequences || u - w.before < end) {
            const int l = __builtin_ctzll(__ballot(x > u - w.before) | 1ull << 63);
            auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            const int64_t begin = w.before + lane64(x - all, l);
            *units = get(n);
            const int tile = (int)quotient(u - begin, max(*units, 1));
            *out = {w.base + l, get(q.row0), get(q.n), get(q.len), tile, 0, 1, 0, 0};
            *first = begin + (int64_t)tile * *units;
            return;
        }
        w.before += end;
    }
}

template <int D, bool E4M3>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void paged_tree_kernel(PagedView c, PagedTreeCall a, float* part, TreeSplit* split) {
    using T = TreeShape<D, E4M3>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::kLds];
    const int groups = gridDim.x / c.kv_heads, kvh = blockIdx.x % c.kv_heads, group = blockIdx.x / c.kv_heads;
    TreeWalk walk = tree_walk(c, a, groups, T::kTile);
    const int64_t end = min(walk.units, (group + 1) * walk.q);
    TreeSplit begun = {0, 0, 0, 0};
    for (int64_t unit = group * walk.q; unit < end;) {
        Piece t;
        int units;
        int64_t first;
        tree_at(c, a, walk, T::kTile, unit, &t, &units, &first);
        const int off = (int)(unit - first), take = (int)min((int64_t)(units - off), end - unit);
        const bool whole = off == 0 && take == units;
        unit += take;
        if (off == 0 && !whole) begun = {t.row0, t.n, t.tile, (int)(quotient(first + units - 1, walk.q) - group) + 1};  // at most once
        const int lo = token_first(a, Seq{t.row0, t.n, t.len}, T::kTile) + off * kTokenUnit;
        const int hi = (int)min((int64_t)lo + (int64_t)take * kTokenUnit, (int64_t)t.len);
        float* rec = whole ? nullptr : part + ((int64_t)kvh * 2 * groups + 2 * group + (off == 0)) * record_floats(T::kRows, D);
        tree_rows<D, E4M3>(c, a, t, kvh, lo, hi, rec, lds);
    }
    if (threadIdx.x == 0) split[kvh * groups + group] = begun;
}

// Rows of split tiles, eight in a workgroup, two for each wave.
constexpr int kTreeMergeRows = 8;

template <int D, bool E4M3>
__global__ __launch_bounds__(256) void paged_tree_merge_kernel(PagedView c, PagedTreeCall a, int groups, const float* part, const TreeSplit* split) {
    const int kvh = blockIdx.x % c.kv_heads, u = blockIdx.x / c.kv_heads, group = u / (kTreeRows / kTreeMergeRows);
    const TreeSplit s = split[kvh * groups + group];
    const int64_t size = record_floats(kTreeRows, D);
    const float* base = part + ((int64_t)kvh * 2 * groups + 2 * group) * size;
    auto rec = [&](int j) { return base + (2 * j + (j == 0)) * size; };
    const Piece t = {0, s.row0, s.n, 0, s.tile, 0, s.parts, 0, 0};
    for (int i = threadIdx.x >> 6; i < kTreeMergeRows; i += 4) {
        const int r = u % (kTreeRows / kTreeMergeRows) * kTreeMergeRows + i, row = s.tile * kTreeRows + r;
        if (s.parts > 1 && row < s.n * a.group) merge_row<D, E4M3>(c, a, t, kvh, rec, kTreeRows, r, row);
    }
}

template <int D, bool E4M3>
hipError_t launch_tree(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx) {
    const int heads = c.kv_heads;
    const int64_t capacity = (int64_t)c.columns * c.slots, sequences = std::min(c.sequences, a.rows);
    const int64_t units = (a.window ? std::min<int64_t>(capacity, (int64_t)a.window + a.max_rows + kTokenUnit) : capacity) / kTokenUnit + 1;
    const int64_t tiles = (int64_t)a.rows * a.group / kTreeRows + sequences;
    const int64_t most = (int64_t)kPagedChunkFloats / record_floats(kTreeRows, D) / heads / 2;
    const int groups = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>((int64_t)ctx->cus * 2 / heads, tiles * units), most));
    TreeSplit* split = reinterpret_cast<TreeSplit*>(ctx->paged_tokens);
    hipLaunchKernelGGL((paged_tree_kernel<D, E4M3>), dim3((uint32_t)(groups * heads)), dim3(256), 0, s, c, a, ctx->paged_chunks, split);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || groups == 1) return e;
    hipLaunchKernelGGL((paged_tree_merge_kernel<D, E4M3>), dim3((uint32_t)(groups * (kTreeRows / kTreeMergeRows) * heads)), dim3(256), 0, s, c, a, groups,
                       ctx->paged_chunks, split);
    return hipGetLastError();
}

template <int D>
hipError_t launch_type(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx) {
    return c.k_scale ? launch_tree<D, true>(c, a, s, ctx) : launch_tree<D, false>(c, a, s, ctx);
}

}  // namespace

hipError_t launch_paged_tree_attention(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx) {
    const int rows = a.max_rows * a.group;
    if (rows <= kTokenRows || rows > kTreeMaxRows || c.head_dim > 256) return launch_paged_tree_rows(c, a, s, ctx);
    switch (c.head_dim) {
        case 64: return launch_type<64>(c, a, s, ctx);
        case 128: return launch_type<128>(c, a, s, ctx);
        default: return launch_type<256>(c, a, s, ctx);
    }
}

}  // namespace moa
