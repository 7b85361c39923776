// moa_paged_attention.hip -- attention of new rows over the paged cache (include/moa_paged.h).
//
// Row i of a sequence's n new rows stands at p = len - n + i and sees positions max(0, p - window + 1) .. p. With
// x_t = scale (q . k_t) it gives sum_t e^(x_t - m) v_t / sum_t e^(x_t - m), m the largest x_t, in one pass over the
// positions with a running m and sum (in base 2: x log2 e). E4M3 pages: k_t and v_t are codes times the head's scale;
// K's joins the factor of x_t, V's the last division.
//
// The query heads of a KV head are rows beside each other: row r of a sequence is token r / group, head r % group of
// the KV head, so one pass over K and V serves them all. Sequences with at most 16 such rows go to the token kernel,
// the others to the chunk kernel; each finds its work from the row starts and lengths on the device.
#include <algorithm>
#include <type_traits>

#include "moa_device.h"
#include "moa_paged.h"

namespace moa {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kTokenRows = 16;   // rows of a token-kernel item
constexpr int kTokenUnit = 128;  // positions that work is dealt out by: one or two steps of four waves
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

// ------------------------------------------------------------------------------------ who does what

// A sequence that takes part: its first row of the call, new rows and length. n = 0: it does not, or is bad.
struct Seq { int row0, n, len; };

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
    if ((n * a.group <= kTokenRows) == tokens) q.n = n;  // at most 2^20 * 128 rows
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

// Token rows. The positions of all sequences, in units of kTokenUnit, are one row of U units, dealt out evenly: group w of
// `groups` takes units [w q, (w + 1) q), q = ceil(U / groups), crossing from sequence to sequence. A part that is not its whole
// sequence leaves a record for the merge: number 2 w where it begins inside its sequence, 2 w + 1 where it begins it, so
// split j of a sequence that begins in group w0 is record 2 (w0 + j) + (j == 0).
struct TokenWalk {
    int64_t units, q;           // U, q
    int base;                   // the 64 sequences looked at
    int64_t before;             // units before them
};

// First position and units of a sequence's span: from a multiple of `align` on, at least one unit.
__device__ __forceinline__ int token_first(const PagedAttentionCall& a, const Seq& q, int align) {
    const int p0 = q.len - q.n;
    return a.window && p0 >= a.window ? (p0 - a.window + 1) / align * align : 0;
}
__device__ __forceinline__ int token_units(const PagedAttentionCall& a, const Seq& q, int align) {
    return q.n ? max(1, (q.len - token_first(a, q, align) + kTokenUnit - 1) / kTokenUnit) : 0;
}

__device__ TokenWalk token_walk(const PagedView& c, const PagedAttentionCall& a, int groups, int align) {
    TokenWalk w = {0, 1, 0, 0};
    bool bad = false;
#pragma unroll 4
    for (int base = 0; base < c.sequences; base += 64)
        w.units += token_units(a, seq_of(c, a, base + (threadIdx.x & 63), true, &bad), align);
    raise_bad(c, bad);
    if (c.sequences <= 64) {  // at most 64 * 2^23 units
        w.units = wave_total((int)w.units);
    } else {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) w.units += __shfl_xor((long long)w.units, o, kWave);
    }
    // (a 64-bit quotient costs a microsecond; real calls have far fewer units)
    w.q = w.units >> 31 ? (w.units + groups - 1) / groups : ((uint32_t)w.units + (uint32_t)groups - 1) / (uint32_t)groups;
    w.q = w.q ? w.q : 1;
    return w;
}

// The sequence that unit u (not before an earlier call's) belongs to, its units and the first of them. u < w.units.
__device__ void token_at(const PagedView& c, const PagedAttentionCall& a, TokenWalk& w, int align, int64_t u, Piece* out, int* units,
                         int64_t* first) {
    const int lane = threadIdx.x & 63;
    bool bad = false;
    for (;; w.base += 64) {
        const Seq q = seq_of(c, a, w.base + lane, true, &bad);
        const int n = token_units(a, q, align), x = scan_sum(n), all = __builtin_amdgcn_readlane(x, 63);
        if (w.base + 64 >= c.sequences || u - w.before < all) {
            const int l = __builtin_ctzll(__ballot(x > (int)(u - w.before)) | 1ull << 63);
            auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            *out = {w.base + l, get(q.row0), get(q.n), get(q.len), 0, 0, 1, 0, 0};
            *units = get(n);
            *first = w.before + get(x - n);
            return;
        }
        w.before += all;
    }
}

// Block `want` of the rows of the sequences that are split, for the merge: four rows, or one where the parts are many; record: the
// sequence's first. False: there are not that many.
constexpr int kMergeWaveSplits = 16;
__device__ __forceinline__ int token_block_rows(int splits) { return splits > kMergeWaveSplits ? 1 : 4; }
__device__ bool token_block(const PagedView& c, const PagedAttentionCall& a, const TokenWalk& w, int align, int want, Piece* out) {
    const int lane = threadIdx.x & 63;
    bool bad = false;
    int64_t before = 0;
    int blocks_before = 0;
    for (int base = 0; base < c.sequences; base += 64) {
        const Seq q = seq_of(c, a, base + lane, true, &bad);
        const int n = token_units(a, q, align), x = scan_sum(n);
        const int64_t first = before + x - n, last = first + max(n, 1) - 1;
        const int64_t w0 = w.units >> 31 ? first / w.q : (uint32_t)first / (uint32_t)w.q;
        const int64_t w1 = w.units >> 31 ? last / w.q : (uint32_t)last / (uint32_t)w.q;
        const int splits = n ? (int)(w1 - w0) + 1 : 0, rows = token_block_rows(splits);
        const int blocks = splits > 1 ? (q.n * a.group + rows - 1) / rows : 0, xb = scan_sum(blocks);
        const uint64_t hit = __ballot(blocks_before + xb > want);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            *out = {base + l, get(q.row0), get(q.n), get(q.len), 0, 0, get(splits), 2 * get((int)w0), (want - blocks_before - get(xb - blocks)) * get(rows)};
            return true;
        }
        before += __builtin_amdgcn_readlane(x, 63);
        blocks_before += __builtin_amdgcn_readlane(xb, 63);
    }
    return false;
}

// Chunks: a sequence of r = n * group rows has ceil(r / kChunkRows) tiles; U is the sum over all tiles of the positions they
// see, in units of kChunkUnit. A tile of more units than twice an even share, per = 2 U / items, but at least kChunkMinUnits, is
// split into ceil(units / per) parts, which leave records for the merge: all split tiles together at most 2 U / per <= items
// of them. (A part costs a write and a read of its rows: 35 tiles of 8 heads of 256, window 1024, took 193 us in three parts
// each and 167 whole.) The last tiles of a sequence, which see the most, come first.
constexpr int kChunkRows = 128;
constexpr int kChunkUnit = 64;
struct ChunkPlan {
    int items;        // per KV head: workgroups that the device holds; records
    int most;         // no call has more items than this
    int most_blocks;  // nor more blocks of rows to merge
};

// A walk over the sequences' pieces in ascending order, by one wave: items (merge_rows = 0), or blocks of merge_rows rows of the
// tiles that are split.
struct ChunkWalk {
    int per;                          // units of a part; 0: the call has no chunks
    int base, pieces, records;        // the 64 sequences looked at; pieces and records before them
};

// Tiles of a sequence, and the units that a tile's rows see: all, or the window and the tile's tokens.
__device__ __forceinline__ int chunk_tiles(const PagedAttentionCall& a, const Seq& q) { return (q.n * a.group + kChunkRows - 1) / kChunkRows; }
__device__ __forceinline__ int chunk_units(const PagedAttentionCall& a, const Seq& q) {
    const int span = min(q.n, (kChunkRows + a.group - 1) / a.group + 1);
    const int seen = a.window ? min(q.len, a.window + span - 1 + kChunkUnit) : q.len;
    return max(1, (seen + kChunkUnit - 1) / kChunkUnit);
}

// last: the last 64 sequences' lanes, the only ones of most calls.
__device__ ChunkWalk chunk_walk(const PagedView& c, const PagedAttentionCall& a, const ChunkPlan& p, Seq* last) {
    int tiles = 0;
    float units = 0.0f;
    bool bad = false;
    Seq q = {};
#pragma unroll 4
    for (int base = 0; base < c.sequences; base += 64) {
        q = seq_of(c, a, base + (threadIdx.x & 63), false, &bad);
        const int n = chunk_tiles(a, q);
        tiles = min(tiles + n, 1 << 24);
        units += (float)n * (float)chunk_units(a, q);
    }
    *last = q;
    tiles = wave_total(tiles);
    // More tiles than the call's rows can have: sequences whose rows overlap, by row starts that descend. None of them runs.
    bad |= tiles > p.most - p.items;
    raise_bad(c, bad);
    if (tiles == 0 || tiles > p.most - p.items) return {0, 0, 0, 0};
    return {__builtin_amdgcn_readfirstlane(chunk_part_units(wave_sum(units), p.items)), 0, 0, 0};  // the same in every wave
}

// Piece `want`, not before an earlier call's. False: there are not that many. have: the only 64 sequences' lanes, or nullptr.
__device__ __forceinline__ bool find_piece(const PagedView& c, const PagedAttentionCall& a, ChunkWalk& w, int merge_rows, int want, const Seq* have,
                                           Piece* out) {
    const int lane = threadIdx.x & 63;
    bool bad = false;
    if (w.per == 0) return false;
    for (; w.base < c.sequences; w.base += 64) {
        Seq q;
        if (have && c.sequences <= 64) q = *have;
        else q = seq_of(c, a, w.base + lane, false, &bad);
        const int tiles = chunk_tiles(a, q), splits = q.n ? (chunk_units(a, q) + w.per - 1) / w.per : 0, items = tiles * splits;
        const int records = splits > 1 ? items : 0, xr = scan_sum(records);
        const int pieces = !merge_rows ? items : (splits > 1 ? (q.n * a.group + merge_rows - 1) / merge_rows : 0), x = scan_sum(pieces);
        const uint64_t hit = __ballot(w.pieces + x > want);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            *out = {w.base + l, get(q.row0), get(q.n), get(q.len), 0, 0, get(splits), 0, 0};
            const int last = get(tiles) - 1, k = want - w.pieces - get(x - pieces);
            int j;  // the tile's place, the last tile first
            if (merge_rows) {
                out->row = k * merge_rows;
                out->tile = out->row / kChunkRows;
                j = last - out->tile;
            } else {
                j = k / out->splits;
                out->tile = last - j;
                out->split = k - j * out->splits;
            }
            out->record = w.records + get(xr - records) + j * out->splits;
            return true;
        }
        w.pieces += __builtin_amdgcn_readlane(x, 63);
        w.records += __builtin_amdgcn_readlane(xr, 63);
    }
    return false;
}

// Records of split tiles: per tile and split bm maxima, bm sums, out [bm][dim], f32. A record whose keys include a page
// outside the pool has NaN maxima: its rows are not written.
__host__ __device__ inline int64_t record_floats(int bm, int dim) { return (int64_t)bm * (2 + dim); }

// One row by one wave over positions [lo, hi), nothing outside them used: 64 positions at a time, a lane each for the
// scores; then lane l holds dims l * dim / 64 .. and takes the weights in turn. The kernels fall back to it where a value that
// their rows do not all see is infinite or NaN (zero times that is NaN). Pages are in range here.
template <bool E4M3>
__device__ void careful_row(const PagedView& c, const uint16_t* q, int s, int kvh, float factor, int lo, int hi, float* mx_out,
                            float* sum_out, float (&o)[8]) {
    const int lane = threadIdx.x & 63, d = c.head_dim, per = d / 64;
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
        x = t0 + lane < hi ? x * factor : -INFINITY;
        float mn = x;
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor(mn, w, kWave));
        mn = fmaxf(mn, mx);
        const float f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mn);
        const float w = t0 + lane < hi ? __builtin_amdgcn_exp2f(x - mn) : 0.0f;
        mx = mn;
        sum = fmaf(sum, f, wave_sum(w));
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] *= f;
        for (int j = 0; j < min(64, hi - t0); ++j) {
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

// Row r of a sequence: where it lies in the call, and the positions it sees.
struct Row {
    int64_t m;      // row of the call
    int h, lo, hi;  // query head; positions [lo, hi)
};
__device__ __forceinline__ Row row_of(const PagedAttentionCall& a, const Piece& t, int kvh, int r) {
    Row x;
    const int i = r / a.group, p = t.len - t.n + i;
    x.m = t.row0 + i;
    x.h = kvh * a.group + (r - i * a.group);
    x.hi = p + 1;
    x.lo = a.window && p >= a.window ? p - a.window + 1 : 0;
    return x;
}

// The positions [lo, hi) of a tile's split: what rows r0 .. r1 of its sequence see, from a multiple of `align` on, in even
// parts of whole units.
struct Span { int lo, hi; };
__device__ __forceinline__ Span span_of(const PagedAttentionCall& a, const Piece& t, int r0, int r1, int align) {
    constexpr int unit = kChunkUnit;
    const int p0 = t.len - t.n + r0 / a.group, p1 = t.len - t.n + r1 / a.group;
    const int lo = a.window && p0 >= a.window ? (p0 - a.window + 1) / align * align : 0, hi = max(p1 + 1, lo);
    const int units = (hi - lo + unit - 1) / unit, per = (units + t.splits - 1) / t.splits;
    const int64_t from = (int64_t)t.split * per * unit, to = from + (int64_t)per * unit;
    return {(int)min((int64_t)hi, lo + from), (int)min((int64_t)hi, lo + to)};
}

// The careful path for a piece's rows [r0, r0 + nr) over positions [lo, hi), waves taking rows in turn. q(r, row): where row
// r0 + r's query lies, not in `out` once that is written (out may be q).
template <bool E4M3, class Q>
__device__ void careful_piece(const PagedView& c, const PagedAttentionCall& a, const Piece& t, int kvh, int r0, int nr, int lo, int hi, Q q,
                              float* rec, int bm) {
    const int lane = threadIdx.x & 63, per = c.head_dim / 64;
    for (int r = threadIdx.x >> 6; r < nr; r += blockDim.x >> 6) {
        const Row x = row_of(a, t, kvh, r0 + r);
        float o[8], mx, sum;
        careful_row<E4M3>(c, q(r, x), t.s, kvh, E4M3 ? c.k_scale[kvh] * a.scale_log2 : a.scale_log2,
                          max(lo, x.lo), min(hi, x.hi), &mx, &sum, o);
        if (rec) {
            if (lane == 0) rec[r] = mx, rec[bm + r] = sum;
            for (int k = 0; k < per; ++k) rec[2 * bm + (int64_t)r * c.head_dim + lane * per + k] = o[k];
        } else {
            const float inv = sum == 0.0f ? 0.0f : (E4M3 ? c.v_scale[kvh] : 1.0f) / sum;
            for (int k = 0; k < per; ++k) a.out[x.m * a.out_row + x.h * c.head_dim + lane * per + k] = (uint16_t)f2bf(o[k] * inv);
        }
    }
}

// ------------------------------------------------------------------------------------ the token kernel

// Up to 16 rows of a sequence over a part of its positions: bound by the bytes of K and V, which go from memory to
// registers and never through LDS. Four waves take a tile of 16 or 32 positions each in turn. Scores are K times Q^T
// (16 x 16 x 32 MFMAs): lane (c = lane % 16, g = lane / 16) then holds, for row c, positions 4 g .. 4 g + 3 of each 16,
// which are just the positions it supplies as A of P times V when V's lanes take the same ones: P moves between no
// lanes. V's lane (c, g) loads kVD dims of each of its positions, and v_perm pairs two positions of a dim; MFMA (b, d)
// then covers dims 16 kVD b + kVD c + d of all c. P enters as two bf16 parts: tiles of 16 positions put both into one
// MFMA, beside the same V twice, tiles of 32 take two. This
// tile's V and the next tile's K are in flight during the arithmetic. (48 sequences of 900 to 32000 positions, 16 heads of 512
// over one: 1.8 GB in 312 us, 5.8 TB/s; 64 of 100 to 9000, 16 rows of 128 over each of 8 heads, E4M3: 0.63 GB in 146, 4.3.)
template <int D, bool E4M3>
struct TokenShape {
    static constexpr int kElem = E4M3 ? 1 : 2;
    static constexpr int kSub = D * kElem >= 512 ? 1 : 2;                       // 16 positions each: K and V of a tile in 128 registers
    static constexpr int kTile = 16 * kSub;
    static constexpr int kHeld = D == 512 ? 1 : 2;                              // workgroups on a CU: waves per SIMD
    static constexpr int kKLoads = D * kElem / 64;                              // 16-byte loads of a K row per lane
    static constexpr int kVD = (E4M3 ? 16 : 8) < D / 16 ? (E4M3 ? 16 : 8) : D / 16;  // dims per V load
    static constexpr int kVB = D / (16 * kVD);                                  // V loads of a row per lane
    static constexpr int kVWords = kVD * kElem / 4;
    static constexpr int kQStride = D + 8;                                      // LDS row of Q: 16 rows start on 16 bank groups
    static constexpr int kLds = 16 * kQStride * 2 + 4 * kTokenRows * D * 4 + 2 * 4 * kTokenRows * 4;
};

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

// A split sequence's last workgroup, found by a counter per (KV head, group that begins it: one split sequence at most), joins its
// records: they are written and read past the XCDs' caches (agent scope). A thread takes four dims of a row, so this is for
// few rows, and for few parts, which it reads one batch after the other: rows * dims up to kJoinElements, up to kJoinUnits units
// a sequence. One token of 8 x 2 heads of 256 over 700 positions: 11.8 us, 13.6 with a merge launch; 120 of them in a window of
// 1024: 158 and 166. Beyond: 4 tokens (8 rows) over 700 to 1500 positions 16.7 and 14.4, one sequence of 16 rows of 512 38.9 and
// 20.6, two tokens over 4000 to 5000 positions 27.7 and 24.4.
constexpr int kJoinUnits = 16;
static_assert(kJoinUnits < (int)kJoinTurn, "a sequence's parts are fewer than a turn of its counter");
constexpr int kJoinElements = 1024;

template <int D, bool E4M3>
__device__ __forceinline__ void join_records(const PagedView& c, const PagedAttentionCall& a, const Piece& t, int kvh, const float* base, int splits) {
    constexpr int kAhead = 8, kSize = kTokenRows * (2 + D) * 4;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, (uint32_t)(2 * splits * kSize), 0x00020000);
    const float vs = E4M3 ? c.v_scale[kvh] : 1.0f;
    const int r = threadIdx.x / (D / 4), d = 4 * (threadIdx.x - r * (D / 4));
    if (r >= t.n * a.group) return;
    float m = -INFINITY, l = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    bool bad = false;
    for (int j0 = 0; j0 < splits; j0 += kAhead) {
        float x[kAhead], y[kAhead], most = m;
        float4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int j = min(j0 + k, splits - 1), at = (2 * j + (j == 0)) * kSize;
            x[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, at + 4 * r, 0, 16 /* sc1 */));
            y[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, at + 4 * (kTokenRows + r), 0, 16));
            w[k] = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(rs, at + 4 * (2 * kTokenRows + r * D + d), 0, 16));
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) bad |= x[k] != x[k], most = fmaxf(most, x[k]);
        const float g = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - most);
        m = most;
        l *= g, v.x *= g, v.y *= g, v.z *= g, v.w *= g;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (j0 + k >= splits) continue;
            const float f = x[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[k] - m);
            l = fmaf(f, y[k], l);
            v.x = fmaf(f, w[k].x, v.x), v.y = fmaf(f, w[k].y, v.y);
            v.z = fmaf(f, w[k].z, v.z), v.w = fmaf(f, w[k].w, v.w);
        }
    }
    if (bad) return;
    const Row x = row_of(a, t, kvh, r);
    const float inv = l == 0.0f ? 0.0f : vs / l;
    *reinterpret_cast<uint2*>(a.out + x.m * a.out_row + x.h * D + d) = make_uint2(pk_bf16(v.x * inv, v.y * inv), pk_bf16(v.z * inv, v.w * inv));
}

// kJoin: the workgroups join their records (tickets [kv_heads][groups], multiples of kJoinTurn); else the merge kernel does.
template <int D, bool E4M3, bool kJoin = false>
__device__ __forceinline__ void token_part(const PagedView& c, const PagedAttentionCall& a, float* part, int kvh, int group, int groups,
                                           uint8_t* lds, uint32_t* tickets = nullptr) {
    using T = TokenShape<D, E4M3>;
    constexpr int NT = T::kSub;
    uint16_t* qs = reinterpret_cast<uint16_t*>(lds);                           // [16][kQStride]
    float* os = reinterpret_cast<float*>(lds + 16 * T::kQStride * 2);          // [4 waves][kTokenRows][D]
    float(*ms)[kTokenRows] = reinterpret_cast<float(*)[kTokenRows]>(os + 4 * kTokenRows * D);
    float(*ls)[kTokenRows] = ms + 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const float factor = E4M3 ? c.k_scale[kvh] * a.scale_log2 : a.scale_log2;
    TokenWalk walk = token_walk(c, a, groups, T::kTile);
    const int64_t end = min(walk.units, (group + 1) * walk.q);
    for (int64_t unit = group * walk.q; unit < end;) {
        Piece t;
        int units;
        int64_t first;
        token_at(c, a, walk, T::kTile, unit, &t, &units, &first);
        const int off = (int)(unit - first), take = (int)min((int64_t)(units - off), end - unit);
        const bool whole = off == 0 && take == units;
        unit += take;
        const int nr = t.n * a.group, from = token_first(a, Seq{t.row0, t.n, t.len}, T::kTile);
        const int lo = from + off * kTokenUnit, hi = (int)min((int64_t)lo + (int64_t)take * kTokenUnit, (int64_t)t.len);
        __syncthreads();  // the part before has been written out
        for (int i = threadIdx.x; i < 16 * D / 8; i += 256) {
            const int r = i / (D / 8), j = i - r * (D / 8);
            const Row x = row_of(a, t, kvh, min(r, nr - 1));
            *reinterpret_cast<uint4*>(qs + r * T::kQStride + 8 * j) = ld16(a.q + x.m * a.q_row + x.h * D + 8 * j);
        }
        const Row mine = row_of(a, t, kvh, min(l16, nr - 1));
        const int see_lo = l16 < nr ? mine.lo : 0, see_hi = l16 < nr ? mine.hi : 0;
        __syncthreads();

        f32x4 o[T::kVB][T::kVD];
#pragma unroll
        for (int b = 0; b < T::kVB; ++b)
#pragma unroll
            for (int d = 0; d < T::kVD; ++d) o[b][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float m_run = -INFINITY, m_ref = -INFINITY, l_run = 0.0f;
        bool bad = false;

        const int32_t* table = c.table + t.s * c.table_stride;
        // lane l looks after position t0 + l % kTile: its page (the next tile's is asked for a tile ahead)
        auto page_at = [&](int t0) { return t0 < hi ? table[page_of(c, min(t0 + lane % T::kTile, hi - 1))] : 0; };
        uint4 kf[NT][T::kKLoads];
        Words<T::kVWords> vf[T::kVB][4 * NT];
        int64_t koff = 0, voff = 0;
        auto place = [&](int page, int t0) {  // offsets of the lane's position; a bad page becomes page 0, and is remembered
            if (t0 >= hi) return;
            const int p = min(t0 + lane % T::kTile, hi - 1);
            const bool in = page >= 0 && page < c.pages;
            bad |= !in;
            page = in ? page : 0;
            const uint32_t slot = p - page_of(c, p) * c.slots;
            koff = page * c.k_page + slot * c.k_slot;
            voff = page * c.v_page + slot * c.v_slot;
        };
        const uint8_t* kbase = c.k + kvh * c.k_head + 16 * g;
        const uint8_t* vbase = c.v + kvh * c.v_head + l16 * T::kVD * T::kElem;
        auto load_k = [&] {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint8_t* p = kbase + __shfl(koff, 16 * i + l16, kWave);
#pragma unroll
                for (int j = 0; j < T::kKLoads; ++j) kf[i][j] = ld16(p + 64 * j);
            }
        };
        auto load_v = [&] {
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) {
                const uint8_t* p = vbase + __shfl(voff, 16 * (i >> 2) + 4 * g + (i & 3), kWave);
#pragma unroll
                for (int b = 0; b < T::kVB; ++b) vf[b][i] = ld_words<T::kVWords>(p + 16 * T::kVD * T::kElem * b);
            }
        };

        int t0 = lo + wave * T::kTile;
        constexpr int kStep = 4 * T::kTile;
        int page = page_at(t0), page1 = page_at(t0 + kStep);
        place(page, t0);
        if (t0 < hi) load_k();
        for (; t0 < hi; t0 += kStep) {
            load_v();
            if constexpr (D == 512) __asm__ volatile("" ::: "memory");  // Q is read from LDS again: no registers for it
            f32x4 sc[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) sc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            // Q's dims follow the order K's 16-byte loads have: bf16 dims 32 j + 8 g, E4M3 dims 64 j + 16 g, two steps a load
#pragma unroll
            for (int j = 0; j < T::kKLoads; ++j) {
                if constexpr (E4M3) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bf16x8 qf = as_bf16x8(ld16(qs + l16 * T::kQStride + 64 * j + 16 * g + 8 * h));
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            const uint32_t w0 = h ? kf[i][j].z : kf[i][j].x, w1 = h ? kf[i][j].w : kf[i][j].y;
                            const uint4 kb = make_uint4(bf16_pair_of_fp8(w0), bf16_pair_of_fp8(w0 >> 16), bf16_pair_of_fp8(w1),
                                                        bf16_pair_of_fp8(w1 >> 16));
                            sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kb), qf, sc[i], 0, 0, 0);
                        }
                    }
                } else {
                    const bf16x8 qf = as_bf16x8(ld16(qs + l16 * T::kQStride + 32 * j + 8 * g));
#pragma unroll
                    for (int i = 0; i < NT; ++i) sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kf[i][j]), qf, sc[i], 0, 0, 0);
                }
            }
            // the next tile's K
            page = page1;
            page1 = page_at(t0 + 2 * kStep);
            place(page, t0 + kStep);
            if (t0 + kStep < hi) load_k();

            // weights of row l16 at positions t0 + 16 i + 4 g + e
            float x[NT][4], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int p = t0 + 16 * i + 4 * g + e;
                    x[i][e] = p >= see_lo && p < see_hi ? sc[i][e] * factor : -INFINITY;
                    mx = fmaxf(mx, x[i][e]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            m_run = fmaxf(m_run, mx);
            float scale = 1.0f;
            if (m_run > m_ref + kSlack) {
                scale = m_ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_ref - m_run);  // -inf: sum and out are zero
                m_ref = m_run;
            }
            if (__any(scale != 1.0f)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float f = __shfl(scale, 4 * g + e, kWave);
#pragma unroll
                    for (int b = 0; b < T::kVB; ++b)
#pragma unroll
                        for (int d = 0; d < T::kVD; ++d) o[b][d][e] *= f;
                }
            }
            const float mu = m_ref == -INFINITY ? 0.0f : m_ref;
            float sum = 0.0f;
            uint32_t pw[2 * NT][kParts];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(x[i][e] - mu), p1 = __builtin_amdgcn_exp2f(x[i][e + 1] - mu);
                    sum += p0 + p1;
                    split_weights(p0, p1, pw[2 * i + e / 2]);
                }
            l_run = fmaf(l_run, scale, sum);
#pragma unroll
            for (int b = 0; b < T::kVB; ++b)
#pragma unroll
                for (int d = 0; d < T::kVD; ++d) {
                    uint32_t w[2 * NT];
#pragma unroll
                    for (int i = 0; i < 2 * NT; ++i) {
                        if constexpr (E4M3)
                            w[i] = bf16_pair_of_fp8(__builtin_amdgcn_perm(vf[b][2 * i + 1].w[d / 4], vf[b][2 * i].w[d / 4],
                                                                          0x0c0c0000u | (4 + d % 4) << 8 | d % 4));
                        else
                            w[i] = __builtin_amdgcn_perm(vf[b][2 * i + 1].w[d / 2], vf[b][2 * i].w[d / 2], d & 1 ? 0x07060302u : 0x05040100u);
                    }
                    if constexpr (NT == 1) {
                        o[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(make_uint4(pw[0][0], pw[1][0], pw[0][1], pw[1][1])),
                                                                          as_bf16x8(make_uint4(w[0], w[1], w[0], w[1])), o[b][d], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int p = 0; p < kParts; ++p)
                            o[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(make_uint4(pw[0][p], pw[1][p], pw[2][p], pw[3][p])),
                                                                              as_bf16x8(make_uint4(w[0], w[1], w[2], w[3])), o[b][d], 0, 0, 0);
                    }
                }
        }

        // the four waves' states into one
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
        if (g == 0) ms[wave][l16] = m_ref, ls[wave][l16] = l_run;
#pragma unroll
        for (int b = 0; b < T::kVB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < T::kVD; d += 4)
                    *reinterpret_cast<float4*>(os + ((wave * kTokenRows + 4 * g + e) * D + 16 * T::kVD * b + T::kVD * l16 + d)) =
                        make_float4(o[b][d][e], o[b][d + 1][e], o[b][d + 2][e], o[b][d + 3][e]);
        bad = __syncthreads_or(bad);
        float* rec = whole ? nullptr : part + ((int64_t)kvh * 2 * groups + 2 * group + (off == 0)) * record_floats(kTokenRows, D);
        bool odd = false;
        const float vs = E4M3 ? c.v_scale[kvh] : 1.0f;
        for (int i = threadIdx.x; i < nr * (D / 4); i += 256) {
            const int r = i / (D / 4), d = 4 * (i - r * (D / 4));
            const float m = fmaxf(fmaxf(ms[0][r], ms[1][r]), fmaxf(ms[2][r], ms[3][r]));
            float l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = ms[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms[w][r] - m);
                const float4 y = *reinterpret_cast<const float4*>(os + (w * kTokenRows + r) * D + d);
                l = fmaf(f, ls[w][r], l);
                v[0] = fmaf(f, y.x, v[0]), v[1] = fmaf(f, y.y, v[1]), v[2] = fmaf(f, y.z, v[2]), v[3] = fmaf(f, y.w, v[3]);
            }
            odd |= !(fabsf(v[0]) + fabsf(v[1]) + fabsf(v[2]) + fabsf(v[3]) < INFINITY);
            if (rec && kJoin) {
                const __amdgpu_buffer_rsrc_t rs =
                    __builtin_amdgcn_make_buffer_rsrc(rec, 0, (uint32_t)(kTokenRows * (2 + D) * 4), 0x00020000);
                const float most = bad ? NAN : m;
                if (d == 0) {
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, most), rs, 4 * r, 0, 16 /* sc1 */);
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, l), rs, 4 * (kTokenRows + r), 0, 16);
                }
                typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
                const u32x4 w = {__builtin_bit_cast(uint32_t, v[0]), __builtin_bit_cast(uint32_t, v[1]), __builtin_bit_cast(uint32_t, v[2]),
                                 __builtin_bit_cast(uint32_t, v[3])};
                __builtin_amdgcn_raw_buffer_store_b128(w, rs, 4 * (2 * kTokenRows + r * D + d), 0, 16);
            } else if (rec) {
                if (d == 0) rec[r] = bad ? NAN : m, rec[kTokenRows + r] = l;
                *reinterpret_cast<float4*>(rec + 2 * kTokenRows + r * D + d) = make_float4(v[0], v[1], v[2], v[3]);
            } else if (!bad) {
                const Row x = row_of(a, t, kvh, r);
                const float inv = l == 0.0f ? 0.0f : vs / l;
                *reinterpret_cast<uint2*>(a.out + x.m * a.out_row + x.h * D + d) =
                    make_uint2(pk_bf16(v[0] * inv, v[1] * inv), pk_bf16(v[2] * inv, v[3] * inv));
            }
        }
        odd = __syncthreads_or(odd);
        if (bad && threadIdx.x == 0) atomicOr(c.err, kErrPaged);
        if (odd && !bad) careful_piece<E4M3>(c, a, t, kvh, 0, nr, lo, hi, [&](int r, const Row&) { return qs + r * T::kQStride; }, rec, kTokenRows);
        if constexpr (kJoin) {
            if (rec) {
                if (odd && !bad) __threadfence();  // the careful path's stores stop at the XCD's cache
                __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                const int w0 = (int)((uint32_t)first / (uint32_t)walk.q), w1 = (int)((uint32_t)(first + units - 1) / (uint32_t)walk.q);
                uint32_t* flag = reinterpret_cast<uint32_t*>(ms);
                if (threadIdx.x == 0) {
                    uint32_t* ticket = tickets + kvh * groups + w0;
                    const uint32_t share = join_share(off == 0, w1 - w0 + 1);
                    *flag = join_last(__hip_atomic_fetch_add(ticket, share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), share);
                }
                __syncthreads();
                if (*flag) join_records<D, E4M3>(c, a, t, kvh, part + ((int64_t)kvh * 2 * groups + 2 * w0) * record_floats(kTokenRows, D), w1 - w0 + 1);
            }
        }
    }
}

template <int D, bool E4M3, bool kJoin>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(TokenShape<D, E4M3>::kHeld))) void paged_token_kernel(
    PagedView c, PagedAttentionCall a, float* part, uint32_t* tickets) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[TokenShape<D, E4M3>::kLds];
    const int groups = gridDim.x / c.kv_heads;
    int kvh = blockIdx.x % c.kv_heads, group = blockIdx.x / c.kv_heads;
    // Rows of half a cache line (64 codes): the heads of a position to one of the 8 XCDs, which then fetches the line once (64
    // sequences of 8 heads: 91 us, 117 with a head per XCD; whole lines are 1-4 % faster with a head per XCD).
    if (D * TokenShape<D, E4M3>::kElem < 128 && groups % 8 == 0) {
        kvh = blockIdx.x / 8 % c.kv_heads;
        group = blockIdx.x % 8 * (groups / 8) + blockIdx.x / 8 / c.kv_heads;
    }
    token_part<D, E4M3, kJoin>(c, a, part, kvh, group, groups, lds, tickets);
}

// ------------------------------------------------------------------------------------ the chunk kernel

// 128 rows of a sequence (32 per wave) over the positions they see: bound by the matrix cores and LDS. K and V tiles
// of kTile positions go through LDS, two buffers, the next tile loading while this one is used (bf16: loads straight into
// LDS; E4M3: through registers, widened to bf16 once for all waves). Scores are K times Q^T (32 x 32 x 16 MFMAs):
// lane (c = lane % 32, hf = lane / 32) holds, for row c, positions 8 (e / 4) + 4 hf + e % 4 of 32, and 8 of them in a
// row are what it supplies as B of V^T times P^T when V's transposing LDS reads fetch the same positions: P moves
// between no lanes, and a row's maximum, sum and rescaling stay in its lane. P enters as two bf16 parts, which share V's
// fragments, and up to 256 dims 16 positions are weighed beside the products of the 16 before them. (Four prompts of 1100 to 4100
// tokens, 32 heads of 128 over 8: 298 to 310 us from card to card, 0.59 PFLOP/s of the formula's work; 318 with all weights first,
// 250 with one part. The same over E4M3 pages: 294.)
// 512 dims: a row's Q and out do not fit beside each other in a wave's registers, so two waves share 32 rows, each with
// half of the dims: they add the halves of the scores through LDS, and each weighs half of the positions for both (1000 rows of
// 16 heads over 15800 positions: 810 to 860 us from card to card, 677 with one part; over E4M3 pages 1020).
template <int D, bool E4M3>
struct ChunkShape {
    static constexpr int kTile = D >= 256 ? 32 : 64;
    static constexpr int kSub = kTile / 32;
    static constexpr int kPair = D == 512 ? 2 : 1;              // waves that share 32 rows
    static constexpr int kThreads = 256 * kPair;
    static constexpr int kHeld = D == 512 ? 1 : 2;              // workgroups on a CU: two waves per SIMD
    static constexpr int kRowBytes = 2 * D;                     // LDS row of a position
    static constexpr int kRowsPerLoad = 1024 / kRowBytes;       // positions a wave's load into LDS covers
    static constexpr int kWaveRows = kTile / (4 * kPair);       // positions of a tile that a wave loads
    static constexpr int kLoads = kWaveRows / kRowsPerLoad;     // loads of K (and of V) per wave and tile
    static constexpr int kCodeLoads = kTile * D / 16 / kThreads;     // E4M3: 16-byte loads of K (and V) per thread and tile
    static constexpr int kGroup = 64 / kWaveRows;               // tiles whose positions a wave's lanes look up at once
    static constexpr int kTileBytes = kTile * kRowBytes;
    static constexpr int kLds = 4 * kTileBytes + (kPair == 2 ? 8 * 4 * 64 * 16 : 256);
};

// 16-byte chunk c of LDS row r lies in chunk c ^ swizzle(r): sixteen rows' reads of one chunk, and four rows' reads of four
// chunks, then meet on no bank. Rows of 128 bytes (64 dims) pair up: two rows span the banks.
template <int D>
__host__ __device__ constexpr int chunk_swizzle(int r) {
    return D == 64 ? ((r >> 1 & 1) << 2 | (r >> 2 & 3)) : ((r & 3) << 2 | (r >> 2 & 3));
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 16 bytes per lane from global memory into LDS, lane l's at lds + 16 l. In asm, since the compiler would let no LDS read
// pass before all such loads are done; `ready` waits for them. (One wait state between the
// write of m0 and its use, five between a vector instruction's write of a scalar register and its use.)
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t lds) {
    __asm__ volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    __asm__ volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"(lds) : "memory");
}

// v, opaque to the compiler: what is computed from it in a loop is not kept in registers across the loop.
__device__ __forceinline__ int in_loop(int v) {
    __asm__ volatile("" : "+v"(v));
    return v;
}
// The lane, computed where it is used: registers that the chunk kernel's loop reloaded from scratch memory would wait for every
// load into LDS before them (512 dims, 1000 rows over 15800 positions: three such reloads a tile cost 24 us). What the chunk kernels
// still spill (32 and 46 registers at 256 dims, bf16 and E4M3, 24 and 52 at 512) lies outside that loop, but for one reload a tile before
// each of the products at 256 dims and, with E4M3 pages, for five at 256 dims and three at 512; seen positions computed in the loop instead
// of held took one away: 148 us for 152 there, 1 % more elsewhere, and were left out.
__device__ __forceinline__ int lane_here() {
    int v;
    __asm__ volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(v));
    return v;
}

// Items first, first + stride, ... of KV head kvh. lds: T::kLds bytes at a multiple of 1024.
template <int D, bool E4M3>
__device__ __forceinline__ void chunk_part(const PagedView& c, const PagedAttentionCall& a, const ChunkPlan& plan, float* part, int kvh, int first,
                                           int stride, uint8_t* lds_base) {
    using T = ChunkShape<D, E4M3>;
    constexpr int kTile = T::kTile, kPair = T::kPair, kWaves = 4 * kPair, kMine = D / kPair;  // dims of a wave
    constexpr int kSteps = kMine / 16, kDims = kMine / 32;
    constexpr int kTileBytes = T::kTileBytes;
    uint8_t* tiles = lds_base;                                            // two buffers of K and V
    float4* xs = reinterpret_cast<float4*>(lds_base + 4 * kTileBytes);    // pairs: the other wave's half of the scores; flags of the waves
    auto any_wave = [&](bool x, bool y) {  // bit 0: x holds in some thread of the workgroup, bit 1: y does
        uint32_t* f = reinterpret_cast<uint32_t*>(xs);
        __syncthreads();
        const uint32_t mine = (__any(x) ? 1u : 0u) | (__any(y) ? 2u : 0u);
        if ((threadIdx.x & 63) == 0) f[threadIdx.x >> 6] = mine;
        __syncthreads();
        uint32_t r = 0;
        for (int w = 0; w < kWaves; ++w) r |= f[w];
        return r;
    };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, hf = lane >> 5;
    const int rg = wave & 3, half = wave >> 2;  // rows 32 rg .., dims half * kMine ..
    // x = factor (q . k): a negative factor's sign goes to q, so that the largest product is the largest x; and a factor of
    // zero stays above it, so that a product of -inf (a position that a row does not see) stays -inf (a NaN stays one)
    const float signed_factor = E4M3 ? c.k_scale[kvh] * a.scale_log2 : a.scale_log2;
    const float factor = fabsf(signed_factor) < 1.2e-38f ? 1.2e-38f : fabsf(signed_factor);
    const uint32_t flip = signed_factor < 0.0f ? 0x80008000u : 0u;
    // LDS byte addresses of a lane: K rows lane % 32, chunk 2 s + lane / 32; V's transposing reads, dim tile 0
    auto k_address = [&] {
        const int ln = lane_here(), r = ln & 31;
        return r * T::kRowBytes + ((ln >> 5) ^ chunk_swizzle<D>(r)) * 16;
    };
    auto v_address = [&] {
        const int ln = lane_here(), r = 4 * (ln >> 5) + (ln >> 2 & 3);
        return r * T::kRowBytes + ((2 * (ln >> 4 & 1) + (ln >> 1 & 1)) ^ chunk_swizzle<D>(r)) * 16 + (ln & 1) * 8;
    };
    Seq seqs;
    ChunkWalk walk = chunk_walk(c, a, plan, &seqs);
    Piece t;
    auto run = [&]() __attribute__((always_inline)) {
        const int r0 = t.tile * kChunkRows, nr = (int)min((int64_t)kChunkRows, (int64_t)t.n * a.group - r0);
        const Span span = span_of(a, t, r0, r0 + nr - 1, kTile);
        const int lo = span.lo, hi = span.hi;
        const int wrow = 32 * rg + l32;  // the lane's row of the tile
        const Row mine = row_of(a, t, kvh, r0 + min(wrow, nr - 1));
        const int see_lo = wrow < nr ? mine.lo : 0, see_hi = wrow < nr ? mine.hi : 0;
        // positions that all of the wave's rows see, and that any does
        int all_lo = mine.lo, all_hi = mine.hi, any_lo = mine.lo, any_hi = mine.hi;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            all_lo = max(all_lo, __shfl_xor(all_lo, o)), all_hi = min(all_hi, __shfl_xor(all_hi, o));
            any_lo = min(any_lo, __shfl_xor(any_lo, o)), any_hi = max(any_hi, __shfl_xor(any_hi, o));
        }
        all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
        any_lo = __builtin_amdgcn_readfirstlane(any_lo), any_hi = __builtin_amdgcn_readfirstlane(any_hi);
        if (32 * rg >= nr) any_hi = 0;  // no rows

        uint4 qf[kSteps];
        {
            const uint16_t* qp = a.q + mine.m * a.q_row + mine.h * D + half * kMine + 8 * hf;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                qf[s] = ld16(qp + 16 * s);
                qf[s] = make_uint4(qf[s].x ^ flip, qf[s].y ^ flip, qf[s].z ^ flip, qf[s].w ^ flip);
            }
        }
        f32x16 o[kDims];
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
        float m_run = -INFINITY, m_ref = -INFINITY, l_run = 0.0f;
        bool bad = false;

        const int32_t* table = c.table + t.s * c.table_stride;
        const uint8_t *kbase = c.k + kvh * c.k_head, *vbase = c.v + kvh * c.v_head;
        // Lane l looks after position l % kWaveRows of the wave's part of tile l / kWaveRows, kGroup tiles at once; the next
        // group's pages are asked for a group ahead.
        const int own = lane / T::kWaveRows * kTile + wave * T::kWaveRows + lane % T::kWaveRows;
        auto page_at = [&](int t0) { return t0 < hi ? table[page_of(c, min(t0 + own, hi - 1))] : 0; };
        int64_t koff = 0, voff = 0;
        auto place = [&](int page, int t0) {
            const int p = min(t0 + own, hi - 1);
            const bool in = page >= 0 && page < c.pages;
            bad |= !in;
            page = in ? page : 0;
            const uint32_t slot = p - page_of(c, p) * c.slots;
            koff = page * c.k_page + slot * c.k_slot;
            voff = page * c.v_page + slot * c.v_slot;
        };
        // bf16: the wave's part of tile `ti` of the group, straight into LDS
        auto load_tile = [&](uint32_t tile, int ti) __attribute__((always_inline)) {
            constexpr int kLanes = 64 / T::kRowsPerLoad;  // lanes of a row
            const int ln = lane_here(), from = ti * T::kWaveRows + ln / kLanes;
#pragma unroll
            for (int i = 0; i < T::kLoads; ++i) {
                const int row = wave * T::kWaveRows + i * T::kRowsPerLoad;
                const int at = ((ln % kLanes) ^ chunk_swizzle<D>(row + ln / kLanes)) * 16, src = from + i * T::kRowsPerLoad;
                const uint32_t kd = tile + row * T::kRowBytes, vd = kd + kTileBytes;
                if (c.near) {
                    const uint32_t ko = (uint32_t)__shfl((int)koff, src, kWave);
                    const uint32_t vo = c.alike ? ko : (uint32_t)__shfl((int)voff, src, kWave);
                    load_to_lds(kbase, ko + at, kd);
                    load_to_lds(vbase, vo + at, vd);
                } else {
                    load_to_lds(kbase + __shfl(koff, src, kWave) + at, kd);
                    load_to_lds(vbase + __shfl(voff, src, kWave) + at, vd);
                }
            }
        };
        // E4M3: the same positions' codes into registers, 16 a load, and from there into LDS as bf16
        constexpr int kCodeLanes = D / 16;
        uint4 kc[T::kCodeLoads], vc[T::kCodeLoads];
        auto load_codes = [&](int ti) __attribute__((always_inline)) {
            const int ln = lane_here();
#pragma unroll
            for (int j = 0; j < T::kCodeLoads; ++j) {
                const int src = ti * T::kWaveRows + j * (64 / kCodeLanes) + ln / kCodeLanes, at = ln % kCodeLanes * 16;
                kc[j] = ld16(kbase + __shfl(koff, src, kWave) + at);
                vc[j] = ld16(vbase + __shfl(voff, src, kWave) + at);
            }
        };
        auto store_codes = [&](uint8_t* kd) __attribute__((always_inline)) {
            auto put = [&](uint8_t* d, const uint4& w, int row, int col) {
                const uint4 lo8 = make_uint4(bf16_pair_of_fp8(w.x), bf16_pair_of_fp8(w.x >> 16), bf16_pair_of_fp8(w.y), bf16_pair_of_fp8(w.y >> 16));
                const uint4 hi8 = make_uint4(bf16_pair_of_fp8(w.z), bf16_pair_of_fp8(w.z >> 16), bf16_pair_of_fp8(w.w), bf16_pair_of_fp8(w.w >> 16));
                *reinterpret_cast<uint4*>(d + row * T::kRowBytes + ((2 * col) ^ chunk_swizzle<D>(row)) * 16) = lo8;
                *reinterpret_cast<uint4*>(d + row * T::kRowBytes + ((2 * col + 1) ^ chunk_swizzle<D>(row)) * 16) = hi8;
            };
            const int ln = lane_here();
#pragma unroll
            for (int j = 0; j < T::kCodeLoads; ++j) {
                const int row = wave * T::kWaveRows + j * (64 / kCodeLanes) + ln / kCodeLanes, col = ln % kCodeLanes;
                put(kd, kc[j], row, col);
                put(kd + kTileBytes, vc[j], row, col);
            }
        };

        // pairs: what the waves of the workgroup wrote for each other is there; loads into LDS stay in flight
        auto exchanged = [] {
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __asm__ volatile("" ::: "memory");
        };
        auto compute = [&](uint32_t tile, int t0) __attribute__((always_inline)) {  // tile: the buffer's place in `tiles`
            const bool sees = t0 < any_hi && t0 + kTile > any_lo;
            if (kPair == 1 && !sees) return;
            f32x16 sc[T::kSub];
#pragma unroll
            for (int b = 0; b < T::kSub; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[b][e] = 0.0f;
            // fragments are read kAhead steps before their MFMAs, and no further: the registers belong to Q and out
            {
                constexpr int kAhead = T::kSub == 2 ? 2 : 3;
                const uint8_t* kt = tiles + tile + half * kMine * 2;
                const int kx = k_address() ^ (kPair == 2 ? half * 16 * T::kRowBytes : 0);  // pairs: own positions first
                bf16x8 kf[kAhead][T::kSub];
                auto read_k = [&](int s) __attribute__((always_inline)) {
#pragma unroll
                    for (int b = 0; b < T::kSub; ++b)
                        kf[s % kAhead][b] = *reinterpret_cast<const bf16x8*>(kt + (kx ^ (32 * (s & 7))) + 256 * (s >> 3) + b * 32 * T::kRowBytes);
                };
#pragma unroll
                for (int s = 0; s < kAhead; ++s) read_k(s);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                    for (int b = 0; b < T::kSub; ++b)
                        sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s % kAhead][b], as_bf16x8(qf[s]), sc[b], 0, 0, 0);
                    if (s + kAhead < kSteps) read_k(s + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            uint32_t pw[T::kSub][8][kParts];
            if constexpr (kPair == 1) {
                if (t0 < all_lo || t0 + kTile > all_hi) {  // some row does not see all of it
                    const int from = in_loop(see_lo - t0 - 4 * hf), to = in_loop(see_hi - t0 - 4 * hf);
#pragma unroll
                    for (int b = 0; b < T::kSub; ++b)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int p = 32 * b + 8 * (e >> 2) + (e & 3);
                            sc[b][e] = p >= from && p < to ? sc[b][e] : -INFINITY;
                        }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < T::kSub; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[b][e]);
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                m_run = fmaxf(m_run, mx * factor);
                float scale = 1.0f;
                if (m_run > m_ref + kSlack) {
                    scale = m_ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_ref - m_run);
                    m_ref = m_run;
                }
                if (__any(scale != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < kDims; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[d][e] *= scale;
                }
                l_run *= scale;
            } else {
                // The positions of 16 a wave: the other's half of their scores comes through LDS, and the weights go back. A
                // wave's weights stand against its own reference, a whole number, so that they move to the larger of the
                // two exactly.
                const int ln = lane_here();
                // `mine`: own scores, later the other's weights and reference; `theirs`: the reverse
                float4 *mine = xs + wave * 256 + ln, *theirs = xs + (wave ^ 4) * 256 + ln;
                mine[0] = make_float4(sc[0][8], sc[0][9], sc[0][10], sc[0][11]);
                mine[64] = make_float4(sc[0][12], sc[0][13], sc[0][14], sc[0][15]);
                exchanged();
                if (!sees) {
                    exchanged();
                    return;
                }
                const float4 y0 = theirs[0], y1 = theirs[64];
                float x[8] = {sc[0][0] + y0.x, sc[0][1] + y0.y, sc[0][2] + y0.z, sc[0][3] + y0.w,
                              sc[0][4] + y1.x, sc[0][5] + y1.y, sc[0][6] + y1.z, sc[0][7] + y1.w};
                if (t0 < all_lo || t0 + kTile > all_hi) {  // some row does not see all of it
                    const int from = in_loop(see_lo - t0 - 4 * hf - 16 * half), to = in_loop(see_hi - t0 - 4 * hf - 16 * half);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int p = 8 * (e >> 2) + (e & 3);
                        x[e] = p >= from && p < to ? x[e] : -INFINITY;
                    }
                }
                float mx = x[0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
                mx = fmaxf(mx, __shfl_xor(mx, 32)) * factor;
                const float r = mx > m_ref + kSlack ? ceilf(mx) : m_ref, mu = r == -INFINITY ? 0.0f : r;
                uint32_t own[4][kParts];
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    split_weights(__builtin_amdgcn_exp2f(fmaf(x[e], factor, -mu)), __builtin_amdgcn_exp2f(fmaf(x[e + 1], factor, -mu)), own[e / 2]);
#pragma unroll
                for (int i = 0; i < kParts; ++i) reinterpret_cast<uint4*>(theirs)[64 * i] = make_uint4(own[0][i], own[1][i], own[2][i], own[3][i]);
                *reinterpret_cast<float*>(theirs + 192) = r;
                exchanged();
                const float s = *reinterpret_cast<const float*>(mine + 192), most = fmaxf(r, s);
#pragma unroll
                for (int i = 0; i < kParts; ++i) {
                    const uint4 w = reinterpret_cast<const uint4*>(mine)[64 * i];
                    const uint32_t other[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        pw[0][j][i] = half ? other[j] : own[j][i];
                        pw[0][4 + j][i] = half ? own[j][i] : other[j];
                    }
                }
                const float scale = most == m_ref || m_ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_ref - most);
                const bool moved = __any(most != m_ref);
                m_ref = most;
                if (__any(scale != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < kDims; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[d][e] *= scale;
                }
                if (moved) {
                    const float f = r == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(r - most), g = s == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s - most);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float h = (j < 4) == (half == 0) ? f : g;
#pragma unroll
                        for (int i = 0; i < kParts; ++i)
                            pw[0][j][i] = pk_bf16(bf2f(pw[0][j][i] & 0xffffu) * h, bf2f(pw[0][j][i] >> 16) * h);
                    }
                }
                const bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < kParts; ++i) sum = dot2_bf16(pw[0][j][i], ones, sum);
                l_run = fmaf(l_run, scale, sum);
            }
            {
                // step n: 16 positions n / kDims, dim tile n % kDims (the next 16 positions weighed beside it: see above). V is read kAhead
                // steps ahead: four took 256 dims (mixed chunks and tokens) 172 us and 512 dims 886, three 152 and 810 (registers).
                constexpr int kAhead = T::kSub == 2 ? 4 : 3, kUnits = 2 * T::kSub, kN = kUnits * kDims;
                const float mu = m_ref == -INFINITY ? 0.0f : m_ref;
                float sum = 0.0f;  // (pairs of waves have added theirs)
                auto weigh = [&](int u, int j) __attribute__((always_inline)) {  // pair j of 4
                    const int b = u / 2, e = 8 * (u & 1) + 2 * j;
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[b][e], factor, -mu)), p1 = __builtin_amdgcn_exp2f(fmaf(sc[b][e + 1], factor, -mu));
                    split_weights(p0, p1, pw[b][e / 2]);
                    sum += p0 + p1;
                };
                uint8_t* vt = tiles + tile + kTileBytes + half * kMine * 2;
                const int vx = v_address();
                s16x4 vr[kAhead][2];
                auto read_v = [&](int n) __attribute__((always_inline)) {
                    const int d = n % kDims, u = n / kDims;
#pragma unroll
                    for (int i = 0; i < 2; ++i)  // positions 8 i + 4 hf ..; an odd i's swizzle differs in bit 1 of the chunk
                        vr[n % kAhead][i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s16x4*)(vt + (vx ^ (64 * (d & 3) + 32 * i)) + 256 * (d >> 2) + (16 * u + 8 * i) * T::kRowBytes));
                };
#pragma unroll
                for (int n = 0; n < kAhead; ++n) read_v(n);
                if constexpr (kPair == 1) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) weigh(0, j);
                }
#pragma unroll
                for (int n = 0; n < kN; ++n) {
                    const int d = n % kDims, u = n / kDims, b = u / 2, i = u & 1;
                    const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(vr[n % kAhead][0], vr[n % kAhead][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            vf, as_bf16x8(make_uint4(pw[b][4 * i][p], pw[b][4 * i + 1][p], pw[b][4 * i + 2][p], pw[b][4 * i + 3][p])), o[d], 0, 0, 0);
                    if (n + kAhead < kN) read_v(n + kAhead);
                    if constexpr (kPair == 1) {
                        if (u + 1 < kUnits) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (j * kDims / 4 == d) weigh(u + 1, j);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                l_run += sum;
            }
        };
        // this wave's loads into LDS are done, and then everybody's; and everybody has read the other buffer
        auto ready = [&] {
            __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __asm__ volatile("" ::: "memory");
        };

        __syncthreads();  // the item before has read its last tile
        const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)tiles;
        constexpr int kGroupStep = T::kGroup * kTile;
        int page = 0, ti = 0;  // the next group's pages; the tile's place in its group
        if (lo < hi) {
            place(page_at(lo), lo);
            page = page_at(lo + kGroupStep);
            if constexpr (E4M3) {
                load_codes(0);
                store_codes(tiles);
            } else {
                load_tile(lds, 0);
            }
        }
        uint32_t at = 0;  // the buffer in use
        for (int t0 = lo; t0 < hi; t0 += kTile) {
            ready();
            const uint32_t next = at ^ (2 * kTileBytes);
            const bool more = t0 + kTile < hi;
            if (more) {
                if (++ti == T::kGroup) {
                    ti = 0;
                    place(page, t0 + kTile);
                    page = page_at(t0 + kTile + kGroupStep);
                }
                if constexpr (E4M3) load_codes(ti);
                else load_tile(lds + next, ti);
            }
            compute(at, t0);
            if (E4M3 && more) store_codes(tiles + next);
            at = next;
        }

        l_run += __shfl_xor(l_run, 32);
        float most = 0.0f;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) most += fabsf(o[d][e]);
        const uint32_t flags = any_wave(bad, wrow < nr && !(most < INFINITY));
        bad = flags & 1;
        const bool odd = flags & 2;  // the careful path writes, and reads q, which may be out
        float* rec = t.splits > 1 ? part + ((int64_t)kvh * plan.items + t.record + t.split) * record_floats(kChunkRows, D) : nullptr;
        const float inv = l_run == 0.0f ? 0.0f : (E4M3 ? c.v_scale[kvh] : 1.0f) / l_run;
        if (wrow < nr && (bad || !odd)) {
            const int first = half * kMine + 4 * hf;  // of the lane's dims: first + 32 d + 2 e .. + 3
            if (rec) {
                float* to = rec + 2 * kChunkRows + wrow * D + first;
#pragma unroll
                for (int d = 0; d < kDims; ++d)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4*>(to + 32 * d + 2 * e) = make_float4(o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]);
            } else if (!bad) {
                uint16_t* to = a.out + mine.m * a.out_row + mine.h * D + first;
#pragma unroll
                for (int d = 0; d < kDims; ++d)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<uint2*>(to + 32 * d + 2 * e) =
                            make_uint2(pk_bf16(o[d][e] * inv, o[d][e + 1] * inv), pk_bf16(o[d][e + 2] * inv, o[d][e + 3] * inv));
            }
            if (rec && hf == 0 && half == 0) rec[wrow] = bad ? NAN : m_ref, rec[kChunkRows + wrow] = l_run;
        }
        if (bad && threadIdx.x == 0) atomicOr(c.err, kErrPaged);
        if (odd && !bad) careful_piece<E4M3>(c, a, t, kvh, r0, nr, lo, hi, [&](int, const Row& x) { return a.q + x.m * a.q_row + x.h * D; }, rec, kChunkRows);
    };
    // Few workgroups have a second item: the first takes the sequences that the walk has read (four prompts of 32 heads of 128,
    // five items in turn on a place: 3 us less than with them read again; 512 dims: 8 us more, for want of registers).
    int item = first;
    if constexpr (kPair == 1) {
        if (item >= plan.most || !find_piece(c, a, walk, 0, item, &seqs, &t)) return;
        do {
            run();
            item += stride;
        } while (item < plan.most && find_piece(c, a, walk, 0, item, nullptr, &t));
    } else {
        for (; item < plan.most && find_piece(c, a, walk, 0, item, nullptr, &t); item += stride) run();
    }
}

// Chunks, and up to 256 dims the token rows beside them: a workgroup of either kind fits a CU next to one of the other, the
// one bound by memory, the other by arithmetic. `stripe` groups in a row (a KV head's share of one workgroup per CU) are
// chunks', the next tokens', until the token groups are used up. (30 single tokens and 5 chunks of 8 heads of 256, window 1024:
// 152 us, with weights of one part 118; in two launches 32 us more.)
template <int D, bool E4M3>
__global__ __launch_bounds__((ChunkShape<D, E4M3>::kThreads)) __attribute__((amdgpu_waves_per_eu(2))) void paged_chunk_kernel(
    PagedView c, PagedAttentionCall a, ChunkPlan plan, int token_groups, int stripe, float* token_records, float* chunk_records) {
    using T = ChunkShape<D, E4M3>;
    constexpr int kLds = T::kPair == 1 && TokenShape<D, E4M3>::kLds > T::kLds ? TokenShape<D, E4M3>::kLds : T::kLds;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    const int kvh = blockIdx.x % c.kv_heads, g = blockIdx.x / c.kv_heads, groups = gridDim.x / c.kv_heads;
    int tokens_before = 0;
    if constexpr (T::kPair == 1) {
        const int row = g / stripe, at = g - row * stripe, tokens = row / 2 * stripe + (row & 1 ? at : 0);
        if ((row & 1) && tokens < token_groups) {
            token_part<D, E4M3>(c, a, token_records, kvh, tokens, token_groups, lds);
            return;
        }
        tokens_before = min(tokens, token_groups);
    }
    chunk_part<D, E4M3>(c, a, plan, chunk_records, kvh, g - tokens_before, groups - (T::kPair == 1 ? token_groups : 0), lds);
}

// ------------------------------------------------------------------------------------------- the merge

// Rows of split tiles, both kernels' in one launch. A workgroup takes a block of rows of a tile and finds it once. Few
// splits: a wave per row, its lanes across the dims. More (long sequences of few rows): the workgroup takes 128 dims of a
// row, its threads in groups that take the records in turn. Bound by its chain of round trips where the records are few, so maxima,
// sums and outputs are asked for at once. (250 records of 128 rows of 512: 15.8 us, 19.5 with the maxima first; 64 times 16 rows of
// 8 heads of 128: 8.4 and 10.6.)
constexpr int kMergeDims = 128;
constexpr int kMergeChunkRows = 8;

// Row r of the tile (rec(j): the record of split j, bm rows each), row `row` of its sequence, by one wave.
template <int D, bool E4M3, class R>
__device__ __forceinline__ void merge_row(const PagedView& c, const PagedAttentionCall& a, const Piece& t, int kvh, R rec, int bm, int r, int row) {
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

template <int D, bool E4M3>
__device__ void merge_tokens(const PagedView& c, const PagedAttentionCall& a, int groups, int blocks, const float* part, int kvh,
                             int first, int stride) {
    constexpr int DB = D < kMergeDims ? D : kMergeDims, kBlocks = D / DB, kCols = DB / 4, kGroups = 256 / kCols, kAhead = 4;
    __shared__ float4 ov[kGroups][kCols];
    __shared__ float om[kGroups], ol[kGroups];
    const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
    constexpr int kAlign = TokenShape<D, E4M3>::kTile;
    const int64_t size = record_floats(kTokenRows, D);
    const TokenWalk walk = token_walk(c, a, groups, kAlign);
    Piece t;
    // the dims of a block are dealt out too where its records are many
    for (int u = first; u < blocks * kBlocks && token_block(c, a, walk, kAlign, u / kBlocks, &t); u += stride) {
        const float* base = part + ((int64_t)kvh * 2 * groups + t.record) * size;
        auto rec = [&](int j) { return base + (2 * j + (j == 0)) * size; };
        if (t.splits <= kMergeWaveSplits) {
            const int r = t.row + (threadIdx.x >> 6);
            if (u % kBlocks == 0 && r < t.n * a.group) merge_row<D, E4M3>(c, a, t, kvh, rec, kTokenRows, r, r);
            continue;
        }
        const int r = t.row, d = u % kBlocks * DB + 4 * col, at = 2 * kTokenRows + r * D + d;
        // this group's records, with a running maximum (rescaled at most 512 / kGroups / kAhead times)
        float m = -INFINITY, l = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        bool bad = false;
        for (int j0 = grp; j0 < t.splits; j0 += kGroups * kAhead) {
            float x[kAhead], y[kAhead], most = m;
            float4 w[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const float* from = rec(min(j0 + k * kGroups, t.splits - 1));
                x[k] = from[r];
                y[k] = from[kTokenRows + r];
                w[k] = *reinterpret_cast<const float4*>(from + at);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) bad |= x[k] != x[k], most = fmaxf(most, x[k]);
            const float g = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - most);
            m = most;
            l *= g, v.x *= g, v.y *= g, v.z *= g, v.w *= g;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (j0 + k * kGroups >= t.splits) continue;
                const float f = x[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[k] - m);
                l = fmaf(f, y[k], l);
                v.x = fmaf(f, w[k].x, v.x), v.y = fmaf(f, w[k].y, v.y);
                v.z = fmaf(f, w[k].z, v.z), v.w = fmaf(f, w[k].w, v.w);
            }
        }
        ov[grp][col] = v;
        if (col == 0) om[grp] = bad ? NAN : m, ol[grp] = l;
        __syncthreads();
        if (grp == 0) {
            m = -INFINITY, l = 0.0f, v = make_float4(0.0f, 0.0f, 0.0f, 0.0f), bad = false;
#pragma unroll
            for (int k = 0; k < kGroups; ++k) bad |= om[k] != om[k], m = fmaxf(m, om[k]);
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const float f = om[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(om[k] - m);
                const float4 y = ov[k][col];
                l = fmaf(f, ol[k], l);
                v.x = fmaf(f, y.x, v.x), v.y = fmaf(f, y.y, v.y), v.z = fmaf(f, y.z, v.z), v.w = fmaf(f, y.w, v.w);
            }
            if (!bad) {
                const Row x = row_of(a, t, kvh, r);
                const float inv = l == 0.0f ? 0.0f : (E4M3 ? c.v_scale[kvh] : 1.0f) / l;
                *reinterpret_cast<uint2*>(a.out + x.m * a.out_row + x.h * D + d) =
                    make_uint2(pk_bf16(v.x * inv, v.y * inv), pk_bf16(v.z * inv, v.w * inv));
            }
        }
        __syncthreads();
    }
}

template <int D, bool E4M3>
__device__ void merge_chunks(const PagedView& c, const PagedAttentionCall& a, const ChunkPlan& plan, const float* part, int kvh, int first,
                             int stride) {
    Seq seqs;
    ChunkWalk walk = chunk_walk(c, a, plan, &seqs);
    Piece t;
    for (int u = first; u < plan.most_blocks && find_piece(c, a, walk, kMergeChunkRows, u, &seqs, &t); u += stride) {
        const float* base = part + ((int64_t)kvh * plan.items + t.record) * record_floats(kChunkRows, D);
        auto rec = [&](int j) { return base + j * record_floats(kChunkRows, D); };
        const int rows = min(kMergeChunkRows, t.n * a.group - t.row);
        for (int i = threadIdx.x >> 6; i < rows; i += 4)
            merge_row<D, E4M3>(c, a, t, kvh, rec, kChunkRows, t.row - t.tile * kChunkRows + i, t.row + i);
    }
}

// The first token_wgs workgroups of a KV head merge tokens (dealt out to token_groups groups, at most token_blocks blocks),
// the others chunks.
template <int D, bool E4M3>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedView c, PagedAttentionCall a, int token_groups, int token_blocks, int token_wgs,
                                                          ChunkPlan chunks, const float* token_part, const float* chunk_part) {
    const int kvh = blockIdx.x % c.kv_heads, g = blockIdx.x / c.kv_heads, wgs = gridDim.x / c.kv_heads;
    if (g < token_wgs) merge_tokens<D, E4M3>(c, a, token_groups, token_blocks, token_part, kvh, g, token_wgs);
    else merge_chunks<D, E4M3>(c, a, chunks, chunk_part, kvh, g - token_wgs, wgs - token_wgs);
}

int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

template <int D, bool E4M3>
hipError_t launch(const PagedView& c, const PagedAttentionCall& a, hipStream_t s, DevCtx* ctx) {
    using T = TokenShape<D, E4M3>;
    const int heads = c.kv_heads;
    const bool chunks_too = (int64_t)a.max_rows * a.group > kTokenRows;
    const int64_t capacity = (int64_t)c.columns * c.slots;
    const int64_t sequences = std::min(c.sequences, a.rows);  // with rows
    // Tokens: a group per workgroup that the device holds (beside chunks in one launch: per CU), units permitting, so that all
    // end together.
    const bool one_launch = chunks_too && ChunkShape<D, E4M3>::kPair == 1;
    const int64_t units = (a.window ? std::min<int64_t>(capacity, (int64_t)a.window + a.max_rows + kTokenUnit) : capacity) / kTokenUnit + 1;
    const int groups = (int)clamp64(std::min<int64_t>((int64_t)ctx->cus * (one_launch ? 1 : T::kHeld) / heads, sequences * units), 1,
                                    (int64_t)kPagedTokenFloats / record_floats(kTokenRows, D) / heads / 2);
    hipError_t e = hipSuccess;
    const bool join = !chunks_too && units <= kJoinUnits && (int64_t)a.max_rows * a.group * D <= kJoinElements && (int64_t)groups * heads <= kPagedTickets;
    if (join) {
        hipLaunchKernelGGL((paged_token_kernel<D, E4M3, true>), dim3((uint32_t)(groups * heads)), dim3(256), 0, s, c, a, ctx->paged_tokens,
                           ctx->paged_tickets);
        return hipGetLastError();
    }
    if (!one_launch) {
        hipLaunchKernelGGL((paged_token_kernel<D, E4M3, false>), dim3((uint32_t)(groups * heads)), dim3(256), 0, s, c, a, ctx->paged_tokens,
                           ctx->paged_tickets);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    // blocks of rows of split sequences, at most; each has another group's part
    int64_t token_blocks = groups > 1 ? std::min<int64_t>((int64_t)a.rows * a.group, (int64_t)groups * kTokenRows) : 0;
    const int64_t token_wgs = std::min<int64_t>(token_blocks * std::max(1, D / kMergeDims), std::max(1, (chunks_too ? 512 : 2048) / heads));
    int64_t chunk_wgs = 0;
    ChunkPlan chunks{};
    if (chunks_too) {
        const int64_t records = (int64_t)kPagedChunkFloats / record_floats(kChunkRows, D) / heads;
        const int64_t tiles = (int64_t)a.rows * a.group / kChunkRows + sequences;
        chunks.items = (int)clamp64((int64_t)ctx->cus * ChunkShape<D, E4M3>::kHeld / heads, 1, records);
        chunks.most = (int)(tiles + chunks.items);
        // a split tile has two records at least
        chunks.most_blocks = chunks.items / 2 * (kChunkRows / kMergeChunkRows);
        const int64_t grid = std::min<int64_t>(chunks.most, std::max(1, 65536 / heads)) + (one_launch ? groups : 0);
        hipLaunchKernelGGL((paged_chunk_kernel<D, E4M3>), dim3((uint32_t)(grid * heads)), dim3(ChunkShape<D, E4M3>::kThreads), 0, s, c, a, chunks,
                           groups, std::max(1, ctx->cus / heads), ctx->paged_tokens, ctx->paged_chunks);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
        chunk_wgs = std::min<int64_t>(chunks.most_blocks, std::max(1, 2048 / heads));
    }
    if (token_wgs + chunk_wgs == 0) return e;
    hipLaunchKernelGGL((paged_merge_kernel<D, E4M3>), dim3((uint32_t)((token_wgs + chunk_wgs) * heads)), dim3(256), 0, s, c, a, groups,
                       (int)token_blocks, (int)token_wgs, chunks, ctx->paged_tokens, ctx->paged_chunks);
    return hipGetLastError();
}

template <int D>
hipError_t launch_type(const PagedView& c, const PagedAttentionCall& a, hipStream_t s, DevCtx* ctx) {
    return c.k_scale ? launch<D, true>(c, a, s, ctx) : launch<D, false>(c, a, s, ctx);
}

}  // namespace

hipError_t launch_paged_attention(const PagedView& c, const PagedAttentionCall& a, hipStream_t s, DevCtx* ctx) {
    switch (c.head_dim) {
        case 64: return launch_type<64>(c, a, s, ctx);
        case 128: return launch_type<128>(c, a, s, ctx);
        case 256: return launch_type<256>(c, a, s, ctx);
        default: return launch_type<512>(c, a, s, ctx);
    }
}

}  // namespace moa
