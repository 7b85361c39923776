// moa_paged_rows.h -- what the kernels of the paged attention share: the sequences that take part, the rows and what they see, one row's
// careful evaluation, and the merge of a row's records.
#pragma once

#include <type_traits>

#include "moa_device.h"
#include "moa_paged.h"

namespace moa {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kTokenRows = 16;   // rows of a token-kernel item
constexpr int kTokenUnit = 128;  // positions that its work is dealt out by: one or two steps of four waves

// Weights are 2^(x - reference), the reference at most this far below the row's largest x so far: the output is
// rescaled only when the maximum has grown by more.
constexpr float kSlack = 8.0f;

__device__ __forceinline__ bf16x8 as_bf16x8(const uint4& v) { return __builtin_bit_cast(bf16x8, v); }

// Two weights as two pairs of bf16, high parts and rests: what is lost is at most 2^-16 of a weight. (One part alone loses 2^-8,
// which is more than what is left where values nearly cancel; a third, for the last 8 bits of f32, takes the chunk kernel another 24 %
// and is below what the f32 rounding of the scores can move.)
constexpr int kParts = 2;
__device__ __forceinline__ void split_weights(float p0, float p1, uint32_t (&w)[kParts]) {
    w[0] = pk_bf16(p0, p1);
    w[1] = pk_bf16(p0 - __uint_as_float(w[0] << 16), p1 - __uint_as_float(w[0] & 0xffff0000u));
}

// Rows that are nodes of trees see the positions before the tree and the nodes of their masks, in any order: their call's type
// chooses the rules below at compile time.
template <class A>
constexpr bool kTree = std::is_same_v<A, PagedTreeCall>;

// ------------------------------------------------------------------------------------ who does what

// A sequence that takes part: its first row of the call, new rows and length. n = 0: it does not, or is bad.
struct Seq { int row0, n, len; };

// tokens: the token kernel's sequences, else the chunk kernel's; kAny: all of them.
template <bool kAny = false>
__device__ __forceinline__ Seq seq_of(const PagedView& c, const PagedAttentionCall& a, int s, bool tokens, bool* bad) {
    Seq q = {0, 0, 0};
    if (s >= c.sequences) return q;
    q.row0 = a.starts[s];
    const int end = a.starts[s + 1];
    q.len = c.lens[s];
    if (end == q.row0) return q;
    if (!rows_in_range(q.row0, end, a.rows, a.max_rows) || q.len < 0 || q.len > paged_capacity(c)) {
        *bad = true;
        return q;
    }
    const int n = end - q.row0;
    if (kAny || (n * a.group <= kTokenRows) == tokens) q.n = n;  // at most 2^20 * 128 rows
    return q;
}

__device__ __forceinline__ void raise_bad(const PagedView& c, bool bad) {
    if (__any(bad) && blockIdx.x == 0 && (threadIdx.x & 63) == 0) atomicOr(c.err, kErrPaged);
}

// Part of a sequence's rows and positions: what a workgroup works on.
struct Piece {
    int s, row0, n, len;        // its sequence
    int tile, split, splits;    // the tile of rows, and which part of its positions
    int record;                 // of the tile's first split
    int row;                    // the merge: first row of the block, in its sequence
};

// First position and units of a sequence's span: from a multiple of `align` on, at least one unit. (A tree's first node stands where
// the first token of consecutive ones does, and no node's window begins before its.)
__device__ __forceinline__ int token_first(const PagedAttentionCall& a, const Seq& q, int align) {
    const int p0 = q.len - q.n;
    return a.window && p0 >= a.window ? (p0 - a.window + 1) / align * align : 0;
}
__device__ __forceinline__ int token_units(const PagedAttentionCall& a, const Seq& q, int align) {
    return q.n ? max(1, (q.len - token_first(a, q, align) + kTokenUnit - 1) / kTokenUnit) : 0;
}

// Inclusive sum over the wave's lanes: four shifts within rows of 16, then the rows' last lanes (DPP: no LDS on the way).
__device__ __forceinline__ int scan_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(scan_sum(x), 63); }

// Records of split tiles: per tile and split bm maxima, bm sums, out [bm][dim], f32. A record whose keys include a page
// outside the pool has NaN maxima: its rows are not written.
__host__ __device__ inline int64_t record_floats(int bm, int dim) { return (int64_t)bm * (2 + dim); }

// Row r of a sequence: where it lies in the call, and the positions it sees (of a tree's, those before the tree).
struct Row {
    int64_t m;      // row of the call
    int h, lo, hi;  // query head; positions [lo, hi)
};

// Trees: bit k of the result says whether row m of the call sees position t0 + k as a node (t0 + 63 not before the tree).
__device__ __forceinline__ uint64_t node_bits(const PagedTreeCall& a, const Piece& t, int64_t m, int t0) {
    const uint64_t* w = a.masks + m * a.words;
    const int at = t0 - (t.len - t.n), left = t.n - at;  // the first position's node (may be negative); nodes from it on
    if (left <= 0) return 0;
    uint64_t bits;
    if (at < 0) {
        bits = w[0] << -at;
    } else {
        const int i = at >> 6, r = at & 63;  // at < n <= 64 words
        bits = w[i] >> r;
        if (r && i + 1 < a.words) bits |= w[i + 1] << (64 - r);
    }
    return left >= 64 ? bits : bits & ((1ull << left) - 1);
}

// A node's depth in its tree, itself included: the nodes it sees.
__device__ __forceinline__ int node_depth(const PagedTreeCall& a, const Piece& t, int64_t m) {
    int d = 0;
    for (int i = 0; i < a.words; ++i) {
        const int left = t.n - 64 * i;
        if (left > 0) d += __popcll(a.masks[m * a.words + i] & (left >= 64 ? ~0ull : (1ull << left) - 1));
    }
    return d;
}

template <class A>
__device__ __forceinline__ Row row_of(const A& a, const Piece& t, int kvh, int r) {
    Row x;
    const int i = r / a.group;
    x.m = t.row0 + i;
    x.h = kvh * a.group + (r - i * a.group);
    int p = t.len - t.n + i;
    x.hi = p + 1;
    if constexpr (kTree<A>) {
        const int depth = node_depth(a, t, x.m), base = t.len - t.n;
        p = base + depth - 1;
        x.hi = depth ? max(base, 0) : 0;
    }
    x.lo = a.window && p >= a.window ? p - a.window + 1 : 0;
    return x;
}

// One row by one wave over positions [lo, hi), nothing outside them used: 64 positions at a time, a lane each for the
// scores; then lane l holds dims l * dim / 64 .. and takes the weights in turn. The kernels fall back to it where a value that
// their rows do not all see is infinite or NaN (zero times that is NaN). Pages are in range here.
template <bool E4M3, class A>
__device__ void careful_row(const PagedView& c, const A& a, const Piece& piece, const Row& row, const uint16_t* q, int kvh, float factor, int lo, int hi,
                            float* mx_out, float* sum_out, float (&o)[8]) {
    const int lane = threadIdx.x & 63, d = c.head_dim, per = d / 64, s = piece.s;
    float mx = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.0f;
    for (int t0 = lo; t0 < hi; t0 += 64) {
        const int t = min(t0 + lane, hi - 1);
        const uint32_t i = page_of(c, t);
        const int slot = t - i * c.slots, page = c.table[s * c.table_stride + i];
        const uint8_t* kp = c.k + page * c.k_page + slot * c.k_slot + kvh * c.k_head;
        float x = 0.0f;
        for (int j = 0; j < d; j += 8) {
            float e[8], f[8];
            bf16x8_to_f32(ld16(q + j), f);
            if (E4M3) {
                const uint2 w = *reinterpret_cast<const uint2*>(kp + j);
                fp8x4_to_f32(w.x, e);
                fp8x4_to_f32(w.y, e + 4);
            } else {
                bf16x8_to_f32(ld16(kp + 2 * j), e);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) x = fmaf(e[k], f[k], x);
        }
        uint64_t seen = 0;  // trees: which of the 64 the row sees
        bool sees = t0 + lane < hi;
        if constexpr (kTree<A>) {
            sees = sees && (t < row.hi || (t0 + 63 >= piece.len - piece.n && (node_bits(a, piece, row.m, t0) >> lane & 1)));
            seen = __ballot(sees);
        }
        x = sees ? x * factor : -INFINITY;
        float mn = x;
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor(mn, w, kWave));
        mn = fmaxf(mn, mx);
        const float f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mn);
        const float w = sees ? __builtin_amdgcn_exp2f(x - mn) : 0.0f;
        mx = mn;
        sum = fmaf(sum, f, wave_sum(w));
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] *= f;
        for (int j = 0; j < min(64, hi - t0); ++j) {
            if (kTree<A> && !(seen >> j & 1)) continue;
            const float wj = __shfl(w, j, kWave);
            const uint8_t* vp = c.v + __shfl(page, j, kWave) * c.v_page + __shfl(slot, j, kWave) * c.v_slot + kvh * c.v_head;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < per)
                    o[k] = fmaf(wj, E4M3 ? e4m3_to_f32(vp[lane * per + k]) : bf2f(reinterpret_cast<const uint16_t*>(vp)[lane * per + k]), o[k]);
        }
    }
    *mx_out = mx;
    *sum_out = sum;
}

// The careful path for a piece's rows [r0, r0 + nr) over positions [lo, hi), waves taking rows in turn. q(r, row): where row
// r0 + r's query lies, not in `out` once that is written (out may be q).
template <bool E4M3, class Q, class A>
__device__ void careful_piece(const PagedView& c, const A& a, const Piece& t, int kvh, int r0, int nr, int lo, int hi, Q q,
                              float* rec, int bm) {
    const int lane = threadIdx.x & 63, per = c.head_dim / 64;
    for (int r = threadIdx.x >> 6; r < nr; r += blockDim.x >> 6) {
        const Row x = row_of(a, t, kvh, r0 + r);
        float o[8], mx, sum;
        careful_row<E4M3>(c, a, t, x, q(r, x), kvh, E4M3 ? c.k_scale[kvh] * a.scale_log2 : a.scale_log2,
                          max(lo, x.lo), kTree<A> ? hi : min(hi, x.hi), &mx, &sum, o);
        if (rec) {
            if (lane == 0) rec[r] = mx, rec[bm + r] = sum;
            for (int k = 0; k < per; ++k) rec[2 * bm + (int64_t)r * c.head_dim + lane * per + k] = o[k];
        } else {
            const float inv = sum == 0.0f ? 0.0f : (E4M3 ? c.v_scale[kvh] : 1.0f) / sum;
            for (int k = 0; k < per; ++k) a.out[x.m * a.out_row + x.h * c.head_dim + lane * per + k] = (uint16_t)f2bf(o[k] * inv);
        }
    }
}

template <int W>
struct Words { uint32_t w[W]; };

template <int W>
__device__ __forceinline__ Words<W> ld_words(const uint8_t* p) {
    Words<W> r;
    if constexpr (W == 4) {
        const uint4 v = ld16(p);
        r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
    } else if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r.w[0] = v.x, r.w[1] = v.y;
    } else {
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    return r;
}

__device__ __forceinline__ uint32_t bf16_pair_of_fp8(uint32_t two) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(two, 1.0f, false));
}

// 16-byte chunk c of LDS row r lies in chunk c ^ swizzle(r): sixteen rows' reads of one chunk, and four rows' reads of four
// chunks, then meet on no bank. Rows of 128 bytes (64 dims) pair up: two rows span the banks.
template <int D>
__host__ __device__ constexpr int chunk_swizzle(int r) {
    return D == 64 ? ((r >> 1 & 1) << 2 | (r >> 2 & 3)) : ((r & 3) << 2 | (r >> 2 & 3));
}

typedef __attribute__((address_space(3))) void lds_void;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 16 bytes per lane from global memory into LDS, lane l's at lds + 16 l. In asm, since the compiler would let no LDS read
// pass before all such loads are done; the kernels wait for them by count. (One wait state between the
// write of m0 and its use, five between a vector instruction's write of a scalar register and its use.)
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t lds) {
    __asm__ volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    __asm__ volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"(lds) : "memory");
}

// Row r of the tile (rec(j): the record of split j, bm rows each), row `row` of its sequence, by one wave.
template <int D, bool E4M3, class R, class A>
__device__ __forceinline__ void merge_row(const PagedView& c, const A& a, const Piece& t, int kvh, R rec, int bm, int r, int row) {
    constexpr int kPer = D / 64;  // dims of a lane
    const int lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.0f, v[kPer] = {};
    bool bad = false;
    // records j0 .. of which `most` at once; find: they are all there are
    auto take = [&](auto most, int j0, bool find) __attribute__((always_inline)) {
        constexpr int K = decltype(most)::value;
        float x[K], y[K], w[K][kPer];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float* at = rec(min(j0 + k, t.splits - 1));
            x[k] = at[r];
            y[k] = at[bm + r];
            const float* o = at + 2 * bm + r * D + lane * kPer;
#pragma unroll
            for (int i = 0; i < kPer; ++i) w[k][i] = o[i];
        }
        if (find) {
#pragma unroll
            for (int k = 0; k < K; ++k) bad |= x[k] != x[k], m = fmaxf(m, x[k]);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (j0 + k >= t.splits) continue;
            // (a record of no weight counts too: sums that are NaN for a row's own values make the row NaN)
            const float f = x[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[k] - m);
            l = fmaf(f, y[k], l);
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] = fmaf(f, w[k][i], v[i]);
        }
    };
    if (t.splits == 2) {
        take(std::integral_constant<int, 2>{}, 0, true);
    } else if (t.splits <= 4) {
        take(std::integral_constant<int, 4>{}, 0, true);
    } else {
        for (int j = lane; j < t.splits; j += 64) {
            const float x = rec(j)[r];
            bad |= x != x;
            m = fmaxf(m, x);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
        for (int j0 = 0; j0 < t.splits; j0 += 4) take(std::integral_constant<int, 4>{}, j0, false);
    }
    if (__any(bad)) return;
    const Row x = row_of(a, t, kvh, row);
    const float inv = l == 0.0f ? 0.0f : (E4M3 ? c.v_scale[kvh] : 1.0f) / l;
    uint16_t* to = a.out + x.m * a.out_row + x.h * D + lane * kPer;
    if constexpr (kPer == 1) {
        *to = (uint16_t)f2bf(v[0] * inv);
    } else {
#pragma unroll
        for (int k = 0; k < kPer; k += 2) reinterpret_cast<uint32_t*>(to)[k / 2] = pk_bf16(v[k] * inv, v[k + 1] * inv);
    }
}

}  // namespace
}  // namespace moa
