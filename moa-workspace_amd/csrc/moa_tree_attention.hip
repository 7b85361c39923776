// moa_tree_attention.hip -- attention of drafted trees over the paged cache (include/moa_paged.h) for sequences of a few dozen rows.
//
// Every row of a tree sees the positions before it, so one pass over K and V serves a tile of 64 rows of a sequence, 16 for each of a
// workgroup's waves, and two tiles the 65 to 128 rows that still come here. K and V go through LDS (moa_tree_rows.h says how). The positions are dealt
// out evenly over as many workgroups as the device holds, and the rows of tiles that were split so are joined by a second launch.
//
// Measured, 40 trees of 9 to 33 nodes with 2 x 256 dims a KV head, bf16: 318 MB of K and V in 72 us, 4.4 TB/s, and 7 us of the merge. 32 trees of
// 5 to 16 nodes with 4 x 128 dims over E4M3 pages: 265 MB in 79 us and 10; loads, widening and the stores to LDS alone took 50 of 85, the products
// and the softmax, of two to four waves behind one barrier a tile, the rest. Dealing by (KV head, positions) in the other order, other
// places of the row groups among the waves, and twice the workgroups on a CU (tiles of 32 positions) changed nothing or were slower.
#include <algorithm>

#include "moa_tree_rows.h"

namespace moa {
namespace {

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

// A split tile, for the merge: its sequence's rows, its number there, its parts and the group that begins it. A group is in two at
// most: the one that its first part goes on with, and the one that its last part begins.
struct TreeSplit { int row0, n, tile, parts, first, unused[3]; };

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
    TreeSplit begun = {0, 0, 0, 0, 0, {}}, inside = begun;
    for (int64_t unit = group * walk.q; unit < end;) {
        Piece t;
        int units;
        int64_t first;
        tree_at(c, a, walk, T::kTile, unit, &t, &units, &first);
        const int off = (int)(unit - first), take = (int)min((int64_t)(units - off), end - unit);
        const bool whole = off == 0 && take == units;
        unit += take;
        if (!whole) {
            const int w0 = (int)quotient(first, walk.q);
            (off == 0 ? begun : inside) = {t.row0, t.n, t.tile, (int)quotient(first + units - 1, walk.q) - w0 + 1, w0, {}};
        }
        const int lo = token_first(a, Seq{t.row0, t.n, t.len}, T::kTile) + off * kTokenUnit;
        const int hi = (int)min((int64_t)lo + (int64_t)take * kTokenUnit, (int64_t)t.len);
        float* rec = whole ? nullptr : part + ((int64_t)kvh * 2 * groups + 2 * group + (off == 0)) * record_floats(kTreeRows, D);
        tree_rows<D, E4M3>(c, a, t, kvh, lo, hi, rec, lds);
    }
    if (threadIdx.x == 0) split[2 * (kvh * groups + group)] = begun, split[2 * (kvh * groups + group) + 1] = inside;
}

// The rows of a split tile are dealt out to kTreeMergeBlocks workgroups for each of its parts. Few parts: a wave takes a row. More: the four
// waves take a row's records in turn, eight at once, and join what they have in LDS.
constexpr int kTreeMergeBlocks = 8;

template <int D, bool E4M3>
__device__ __forceinline__ void tree_merge(const PagedView& c, const PagedTreeCall& a, const TreeSplit& s, int kvh, const float* base, int block) {
    constexpr int kPer = D / 64;  // dims of a lane
    __shared__ float vs[4][D], ms[4], ls[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, blocks = kTreeMergeBlocks * s.parts, rows = min(kTreeRows, s.n * a.group - s.tile * kTreeRows);
    auto rec = [&](int j) { return base + (2 * j + (j == 0)) * record_floats(kTreeRows, D); };
    const Piece t = {0, s.row0, s.n, 0, s.tile, 0, s.parts, 0, 0};
    if (s.parts <= 4) {
        for (int r = block + wave * blocks; r < rows; r += 4 * blocks) merge_row<D, E4M3>(c, a, t, kvh, rec, kTreeRows, r, s.tile * kTreeRows + r);
        return;
    }
    for (int r = block; r < rows; r += blocks) {
        float m = -INFINITY, l = 0.0f, v[kPer] = {};
        bool bad = false;
        constexpr int K = 8;
        for (int j0 = wave; j0 < s.parts; j0 += 4 * K) {
            float x[K], y[K], w[K][kPer], most = m;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const float* at = rec(min(j0 + 4 * k, s.parts - 1));
                x[k] = j0 + 4 * k < s.parts ? at[r] : -INFINITY;
                y[k] = at[kTreeRows + r];
#pragma unroll
                for (int i = 0; i < kPer; ++i) w[k][i] = at[2 * kTreeRows + r * D + lane * kPer + i];
            }
#pragma unroll
            for (int k = 0; k < K; ++k) bad |= x[k] != x[k], most = fmaxf(most, x[k]);
            const float g = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - most);
            m = most, l *= g;
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] *= g;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (j0 + 4 * k >= s.parts) continue;
                // (a record of no weight counts too: sums that are NaN for a row's own values make the row NaN)
                const float f = x[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[k] - m);
                l = fmaf(f, y[k], l);
#pragma unroll
                for (int i = 0; i < kPer; ++i) v[i] = fmaf(f, w[k][i], v[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) vs[wave][lane * kPer + i] = v[i];
        if (lane == 0) ms[wave] = bad ? NAN : m, ls[wave] = l;
        __syncthreads();
        bad = false, m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) bad |= ms[w] != ms[w], m = fmaxf(m, ms[w]);
        if (!bad && (int)threadIdx.x < D) {
            float o = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = ms[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms[w] - m);
                l = fmaf(f, ls[w], l);
                o = fmaf(f, vs[w][threadIdx.x], o);
            }
            const int row = s.tile * kTreeRows + r, node = row / a.group;
            a.out[(int64_t)(s.row0 + node) * a.out_row + (kvh * a.group + row - node * a.group) * D + threadIdx.x] =
                (uint16_t)f2bf(l == 0.0f ? 0.0f : o * ((E4M3 ? c.v_scale[kvh] : 1.0f) / l));
        }
        __syncthreads();  // the next row's
    }
}

template <int D, bool E4M3>
__global__ __launch_bounds__(256) void paged_tree_merge_kernel(PagedView c, PagedTreeCall a, int groups, const float* part, const TreeSplit* split) {
    const int kvh = blockIdx.x % c.kv_heads, u = blockIdx.x / c.kv_heads, group = u / kTreeMergeBlocks;
    const float* records = part + (int64_t)kvh * 2 * groups * record_floats(kTreeRows, D);
    const TreeSplit mine[2] = {split[2 * (kvh * groups + group)], split[2 * (kvh * groups + group) + 1]};
    for (const TreeSplit& s : mine)
        if (s.parts) tree_merge<D, E4M3>(c, a, s, kvh, records + 2 * (int64_t)s.first * record_floats(kTreeRows, D), (group - s.first) * kTreeMergeBlocks + u % kTreeMergeBlocks);
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
    hipLaunchKernelGGL((paged_tree_merge_kernel<D, E4M3>), dim3((uint32_t)(groups * kTreeMergeBlocks * heads)), dim3(256), 0, s, c, a, groups,
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
