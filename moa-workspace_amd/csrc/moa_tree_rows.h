// moa_tree_rows.h -- the rows of a tile of a drafted tree over a part of their positions, for the kernels that deal the parts out.
#pragma once

#include "moa_paged_rows.h"

namespace moa {
namespace {

constexpr int kTreeRows = 64;      // of a tile: 16 for each of four waves

// Rows of a sequence that come here, up to 256 dims: from 17 on, since the token kernel reads K and V without LDS for all 16 that one MFMA takes
// (one sequence of 12000 positions, 16 rows of 256 dims: 22 us there, 51 here), to two tiles, as many rows as the chunk kernel shares a tile of
// K and V among. Against that kernel, 16 sequences of 1000 to 9000 positions, us here / there at 24, 64, 100 and 128 rows: 256 dims bf16
// 145 / 207, 200 / 261, 225 / 240, 266 / 266; 256 dims E4M3 105 / 185, 154 / 247, 171 / 213, 262 / 260; 128 dims bf16 81 / 89, 95 / 100, 146 / 134,
// 164 / 167; 128 dims E4M3 61 / 77, 79 / 98, 121 / 128, 160 / 157. One sequence of 4000 positions, 100 rows: 27 / 46 (256 dims), 22 / 27 (128).
// Rows of 512 dims took 590 us here and 376 there (12 sequences of up to 16000 positions): half the registers of a wave hold its output.
// One bound for all types and dims, though 128 dims bf16 change sides between 64 and 100 rows (9 % at 100) and E4M3 at 128 (2 %). It is compared
// with the call's max_rows: a batch with one larger tree goes to the chunk kernel whole.
constexpr int kTreeMaxRows = 128;

template <int D, bool E4M3>
struct TreeShape {
    // Positions of a tile: 16 KB of K and V as bf16, 32 KB of 256 dims; and of E4M3 of 128 dims, where only two tiles are in LDS and more of
    // the work lies between barriers then (32 trees, 265 MB: 87 us, 94 with 32 positions).
    static constexpr int kTile = D == 64 || (D == 128 && E4M3) ? 64 : 32;
    static constexpr int kSub = kTile / 16;
    static constexpr int kRowBytes = 2 * D;                  // LDS row of a position
    static constexpr int kStage = 2 * kTile * kRowBytes;
    // Two workgroups share a CU's 160 KB. bf16: the tile in use and those on their way, five of 16 KB up to 128 dims, two of 32 KB at 256.
    // E4M3: two tiles as bf16, and kAhead tiles of codes on their way in registers, 32 of them (at 256 dims 18 registers spill, 44 bytes a lane).
    static constexpr int kStages = E4M3 ? 2 : 80 * 1024 / kStage;
    static constexpr int kLds = kStages * kStage;
    static constexpr int kAhead = D == 64 ? 4 : 2;
    static constexpr int kWaveRows = kTile / 4;              // positions of a tile that a wave loads
    static constexpr int kRowsPerLoad = 1024 / kRowBytes;    // positions that a load of 16 bytes a lane covers
    static constexpr int kLoads = kWaveRows / kRowsPerLoad;  // of K, and of V, per wave and tile
    static constexpr int kCodeLoads = kTile * D / 16 / 256;  // E4M3: the same per thread
    static constexpr int kGroup = 64 / kWaveRows;            // tiles whose positions a wave's lanes look up at once
};

// 16-byte chunk c of LDS row r lies in chunk c ^ swizzle(r). What has to fall on all banks: K's reads, which take one chunk of four quads of rows
// beside each other, the quads of lanes l and l + 16 from different ones (any four different low bits do, where the lane's step leaves them alone);
// V's, two chunks of eight rows (bit 1 differs between quads 0 and 1, and 2 and 3); and the writes of widened codes, every other chunk of a
// row and of the row four behind (bit 0 differs there). Rows of 128 bytes (64 dims) pair up: two rows span the banks.
template <int D>
__host__ __device__ constexpr int tree_swizzle(int r) {
    const int quad = (r >> 2 & 1) * 3 ^ (r >> 3 & 1);
    return D == 64 ? (r >> 1 & 1) << 2 | quad : (r & 3) << 2 | quad;
}
// The chunk of a row that lane group g multiplies in step s. (Any order of the dims will do that Q has too.)
template <int D>
__host__ __device__ constexpr int tree_chunk(int s, int g) {
    return D == 64 ? 4 * (g & 1) + (g >> 1) + 2 * s : 16 * (s >> 2) + 4 * g + (s & 3);
}

// The largest of a row's values, over the four lanes that hold it: 16 and 32 lanes apart, in vector registers.
__device__ __forceinline__ float rows_max(float x) {
    auto pair = [](auto y) { return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1])); };
    x = pair(__builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return pair(__builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
}

// Up to kTreeRows rows of a sequence, those of tile t.tile, over positions [lo, hi) of it, lo a multiple of kTile: rows 16 w .. of them by
// wave w of the workgroup. rec: the record that they leave, or nullptr where [lo, hi) is all they see: then their results are written. lds: kLds
// bytes at a multiple of 1024.
//
// Scores are K times Q^T (16 x 16 x 32 MFMAs): lane (c = lane % 16, g = lane / 16) holds, for row c, positions 4 g .. 4 g + 3 of 16, which
// are just what it supplies as B of V^T times P^T, 32 positions at a time, when V's transposing LDS reads fetch the same positions: P moves
// between no lanes, and a row's maximum, sum and outputs are its lanes'. P enters as two bf16 parts, which share V's fragments.
//
// bf16 tiles go from memory to LDS directly, into a ring of stages with one barrier a tile: the matrix cores and LDS have a third of the time that
// memory takes, so what counts is that loads pause as little as can be. At 64 and 128 dims three tiles stay on their way while a wave waits
// for one; at 256 dims, two stages, the next tile is asked for behind the wait and the barrier, and in between only the CU's other workgroup's loads
// are. E4M3 codes wait in registers and are widened on their way to LDS.
template <int D, bool E4M3>
__device__ __forceinline__ void tree_rows(const PagedView& c, const PagedTreeCall& a, const Piece& t, int kvh, int lo, int hi, float* rec, uint8_t* lds) {
    using T = TreeShape<D, E4M3>;
    constexpr int kTile = T::kTile, kSteps = D / 32, kDims = D / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int r0 = t.tile * kTreeRows, nr = min(kTreeRows, t.n * a.group - r0), tree0 = t.len - t.n;
    // x = factor (q . k): a negative factor's sign goes to q, so that the largest product is the largest x; and a factor of
    // zero stays above it, so that a product of -inf (a position that a row does not see) stays -inf (a NaN stays one)
    const float signed_factor = E4M3 ? c.k_scale[kvh] * a.scale_log2 : a.scale_log2;
    const float factor = fabsf(signed_factor) < 1.2e-38f ? 1.2e-38f : fabsf(signed_factor);
    const uint32_t flip = signed_factor < 0.0f ? 0x80008000u : 0u;
    // LDS byte addresses of a lane: K row l16, chunk tree_chunk; V's transposing reads, rows 4 g + ln / 4 % 4, chunk 2 d + ln / 2 % 2
    const int k_at = l16 * T::kRowBytes + ((tree_chunk<D>(0, g) ^ tree_swizzle<D>(l16)) * 16);
    const int v_row = 4 * g + (lane >> 2 & 3), v_at = v_row * T::kRowBytes + (((lane >> 1 & 1) ^ tree_swizzle<D>(v_row)) * 16) + (lane & 1) * 8;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_void*)lds;
    // the lane's row: where it lies, its query, and the positions that it, and all rows of the wave, see
    const int wrow = 16 * wave + l16;
    const bool is = wrow < nr, rows = 16 * wave < nr;
    const int row = r0 + min(wrow, nr - 1), node = row / a.group, m_row = t.row0 + node, head = kvh * a.group + row - node * a.group;
    uint4 qf[kSteps];
    int see_lo = 0, see_hi = 0, all_lo = 0, all_hi = 0;
    f32x4 o[kDims];
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, m_ref = -INFINITY, l_run = 0.0f;
    bool bad = false;

    const int32_t* table = c.table + t.s * c.table_stride;
    const uint8_t *kbase = c.k + kvh * c.k_head, *vbase = c.v + kvh * c.v_head;
    // Lane l looks after position l % kWaveRows of the wave's part of tile l / kWaveRows, kGroup tiles at once; the next
    // group's pages are asked for a group ahead.
    const int own = lane / T::kWaveRows * kTile + wave * T::kWaveRows + lane % T::kWaveRows;
    auto page_at = [&](int t0) { return t0 < hi ? table[page_of(c, min(t0 + own, hi - 1))] : 0; };
    int64_t koff = 0, voff = 0;
    auto place = [&](int page, int t0) {  // a bad page becomes page 0, and is remembered
        const int p = min(t0 + own, hi - 1);
        const bool in = page >= 0 && page < c.pages;
        bad |= !in;
        page = in ? page : 0;
        const uint32_t slot = p - page_of(c, p) * c.slots;
        koff = page * c.k_page + slot * c.k_slot;
        voff = page * c.v_page + slot * c.v_slot;
    };
    int page = 0, ti = 0, look = lo;  // the next group's pages; the next tile's place in its group, and its first position
    auto look_up = [&] {             // before each tile's loads
        if (ti == T::kGroup) {
            ti = 0;
            place(page, look);
            page = page_at(look + T::kGroup * kTile);
        }
    };
    // bf16: the wave's part of the next tile, straight into LDS
    auto load_tile = [&](uint32_t stage) __attribute__((always_inline)) {
        look_up();
        constexpr int kLanes = 64 / T::kRowsPerLoad;  // lanes of a row
        const int src0 = ti * T::kWaveRows + lane / kLanes;
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i) {
            const int row = wave * T::kWaveRows + i * T::kRowsPerLoad;
            const int at = ((lane % kLanes) ^ tree_swizzle<D>(row + lane / kLanes)) * 16, src = src0 + i * T::kRowsPerLoad;
            const uint32_t kd = lds_at + stage + row * T::kRowBytes, vd = kd + T::kStage / 2;
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
        ++ti, look += kTile;
    };
    // E4M3: the same positions' codes into registers, 16 a load, and from there into LDS as bf16, two chunks of a row. Eight lanes take half as
    // many columns of two rows four apart, whose swizzles differ in their lowest bit: so their writes fall on all banks.
    struct Codes { uint4 k[T::kCodeLoads], v[T::kCodeLoads]; };
    constexpr int kCodeLanes = D / 16, kCodeRows = 64 / kCodeLanes;  // lanes of a row, rows of a load
    const int code_col = (lane & 3) + (lane >> 3) % (kCodeLanes / 4) * 4;
    auto code_row = [&](int j) {
        const int x = (lane >> 3) / (kCodeLanes / 4) + j * (kCodeRows / 2);
        return (x & 3) + (lane >> 2 & 1) * 4 + (x >> 2) * 8;
    };
    auto load_codes = [&](Codes& x) __attribute__((always_inline)) {
        look_up();
#pragma unroll
        for (int j = 0; j < T::kCodeLoads; ++j) {
            const int src = ti * T::kWaveRows + code_row(j), at = code_col * 16;
            if (c.near) {
                const uint32_t ko = (uint32_t)__shfl((int)koff, src, kWave), vo = c.alike ? ko : (uint32_t)__shfl((int)voff, src, kWave);
                x.k[j] = ld16(kbase + (ko + at));
                x.v[j] = ld16(vbase + (vo + at));
            } else {
                x.k[j] = ld16(kbase + __shfl(koff, src, kWave) + at);
                x.v[j] = ld16(vbase + __shfl(voff, src, kWave) + at);
            }
        }
        ++ti, look += kTile;
    };
    auto store_codes = [&](const Codes& x, uint8_t* kd) __attribute__((always_inline)) {
        auto low = [](uint32_t w) { return bf16_pair_of_fp8(w); };
        auto high = [](uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)); };
        auto put = [&](uint8_t* d, const uint4& w, int row) {
            *reinterpret_cast<uint4*>(d + row * T::kRowBytes + ((2 * code_col) ^ tree_swizzle<D>(row)) * 16) =
                make_uint4(low(w.x), high(w.x), low(w.y), high(w.y));
            *reinterpret_cast<uint4*>(d + row * T::kRowBytes + ((2 * code_col + 1) ^ tree_swizzle<D>(row)) * 16) =
                make_uint4(low(w.z), high(w.z), low(w.w), high(w.w));
        };
#pragma unroll
        for (int j = 0; j < T::kCodeLoads; ++j) {
            const int row = wave * T::kWaveRows + code_row(j);
            put(kd, x.k[j], row);
            put(kd + T::kStage / 2, x.v[j], row);
        }
    };

    // the tile of positions t0 .. in LDS at `tile`, 16 positions at a time
    auto compute = [&](const uint8_t* tile, int t0) __attribute__((always_inline)) {
        if (!rows) return;
        // fragments are read kAhead steps before their MFMAs, in an order that the compiler keeps (left to it, each is waited for at once)
        f32x4 sc[T::kSub];
        {
            constexpr int kAhead = 2;
            bf16x8 kf[kAhead][T::kSub];
            auto read_k = [&](int s) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < T::kSub; ++b)
                    kf[s % kAhead][b] = *reinterpret_cast<const bf16x8*>(tile + (k_at ^ (D == 64 ? 32 * s : 16 * (s & 3))) + (D == 64 ? 0 : 256 * (s >> 2)) +
                                                                         16 * b * T::kRowBytes);
            };
#pragma unroll
            for (int b = 0; b < T::kSub; ++b) sc[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < kAhead; ++s) read_k(s);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int b = 0; b < T::kSub; ++b) sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[s % kAhead][b], as_bf16x8(qf[s]), sc[b], 0, 0, 0);
                if (s + kAhead < kSteps) read_k(s + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (t0 < all_lo || t0 + kTile > all_hi) {  // some row does not see all of it
            const uint64_t nodes = t0 + kTile > tree0 && t0 < hi && is ? node_bits(a, t, m_row, t0) : 0;
#pragma unroll
            for (int b = 0; b < T::kSub; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 16 * b + 4 * g + e, p = t0 + at;
                    const bool sees = (p >= see_lo && p < see_hi) || (nodes >> at & 1);
                    sc[b][e] = sees ? sc[b][e] : -INFINITY;
                }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < T::kSub; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[b][e]);
        mx = rows_max(mx);
        m_run = fmaxf(m_run, mx * factor);
        float scale = 1.0f;
        if (m_run > m_ref + kSlack) {
            scale = m_ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_ref - m_run);  // -inf: sum and out are zero
            m_ref = m_run;
        }
        if (__any(scale != 1.0f)) {
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d][e] *= scale;
        }
        const float mu = m_ref == -INFINITY ? 0.0f : m_ref;
        float sum = 0.0f;
        // step n: positions 32 (n / kDims) .., dims 16 (n % kDims) ..; the first V fragments are read beside the weights
        constexpr int kAhead = 4, kN = T::kSub / 2 * kDims;
        s16x4 vr[kAhead][2];
        auto read_v = [&](int n) __attribute__((always_inline)) {
            const int d = n % kDims, u = n / kDims;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                vr[n % kAhead][i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + T::kStage / 2 + (v_at ^ (32 * (d & (D == 64 ? 3 : 7)))) +
                                                                                          (D == 64 ? 0 : 256 * (d >> 3)) + 16 * (2 * u + i) * T::kRowBytes));
        };
#pragma unroll
        for (int n = 0; n < kAhead; ++n) read_v(n);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t pw[T::kSub][2][kParts];
#pragma unroll
        for (int b = 0; b < T::kSub; ++b)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[b][e], factor, -mu)), p1 = __builtin_amdgcn_exp2f(fmaf(sc[b][e + 1], factor, -mu));
                sum += p0 + p1;
                split_weights(p0, p1, pw[b][e / 2]);
            }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const int d = n % kDims, b = 2 * (n / kDims);
            const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(vr[n % kAhead][0], vr[n % kAhead][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int p = 0; p < kParts; ++p)
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, as_bf16x8(make_uint4(pw[b][0][p], pw[b][1][p], pw[b + 1][0][p], pw[b + 1][1][p])), o[d],
                                                               0, 0, 0);
            if (n + kAhead < kN) read_v(n + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
        l_run = fmaf(l_run, scale, sum);
    };

    const int tiles = (hi - lo + kTile - 1) / kTile;
    // what the part reads of its rows is asked for ahead of its tiles, and looked at when those are on their way
    uint64_t mask[kTreeMaxWords];
    {
        const uint16_t* qp = a.q + (int64_t)m_row * a.q_row + head * D;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[s] = ld16(qp + 8 * tree_chunk<D>(s, g));
#pragma unroll
        for (int w = 0; w < kTreeMaxWords; ++w) mask[w] = w < a.words ? a.masks[(int64_t)m_row * a.words + w] : 0;
    }
    if (tiles > 0) {
        place(page_at(lo), lo);
        page = page_at(lo + T::kGroup * kTile);
    }
    __syncthreads();  // the part before has read its flags
    Codes codes[E4M3 ? T::kAhead : 1];
    constexpr int kFlight = T::kStages - 2;  // bf16: tiles whose loads may be on their way while a tile is used
    if (tiles > 0) {
        if constexpr (E4M3) {
#pragma unroll
            for (int s = 0; s < T::kAhead; ++s) load_codes(codes[s]);
        } else {
            for (int s = 0; s <= kFlight && s < tiles; ++s) load_tile(s * T::kStage);
        }
    }
    {
        int depth = 0;
#pragma unroll
        for (int w = 0; w < kTreeMaxWords; ++w) {
            const int left = t.n - 64 * w;
            if (left > 0) depth += __popcll(mask[w] & (left >= 64 ? ~0ull : (1ull << left) - 1));
        }
        const int place = tree0 + depth - 1, from_here = a.window && place >= a.window ? place - a.window + 1 : 0;
        see_lo = all_lo = from_here, see_hi = all_hi = depth ? min(max(tree0, 0), hi) : 0;
        if (!is) see_lo = see_hi = 0;
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) all_lo = max(all_lo, __shfl_xor(all_lo, x)), all_hi = min(all_hi, __shfl_xor(all_hi, x));
        all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[s] = make_uint4(qf[s].x ^ flip, qf[s].y ^ flip, qf[s].z ^ flip, qf[s].w ^ flip);
    }
    if constexpr (E4M3) {
        // kAhead tiles a turn, the last of them perhaps behind the part
        for (int i = 0; i < tiles; i += T::kAhead) {
#pragma unroll
            for (int s = 0; s < T::kAhead; ++s) {
                uint8_t* tile = lds + (s & 1) * T::kStage;  // read by all two tiles ago
                store_codes(codes[s], tile);
                load_codes(codes[s]);
                __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                __asm__ volatile("" ::: "memory");
                if (i + s < tiles) compute(tile, lo + (i + s) * kTile);
            }
        }
    } else {
        uint32_t at = 0, into = (T::kStages - 1) * T::kStage;
        for (int i = 0; i < tiles; ++i) {
            // this wave's loads of the tile are done, and then everybody's; and everybody has read the tile before it
            if (i + kFlight < tiles) __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kFlight * 2 * T::kLoads) : "memory");
            else __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __asm__ volatile("" ::: "memory");
            if (i + T::kStages - 1 < tiles) load_tile(into);
            compute(lds + at, lo + i * kTile);
            into = at;
            at = at + T::kStage == T::kStages * T::kStage ? 0 : at + T::kStage;
        }
    }

    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    float most = 0.0f;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) most += fabsf(o[d][e]);
    uint32_t* flags = reinterpret_cast<uint32_t*>(lds);
    const uint32_t wave_flags = (__any(bad) ? 1u : 0u) | (__any(is && !(most < INFINITY)) ? 2u : 0u);
    __syncthreads();  // the last tile has been read
    if (lane == 0) flags[wave] = wave_flags;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) all |= flags[w];
    bad = all & 1;
    const bool odd = all & 2;  // the careful path writes, and reads q, which may be out
    if (is && (bad || !odd)) {
        if (rec) {
            float* to = rec + 2 * kTreeRows + wrow * D + 4 * g;
#pragma unroll
            for (int d = 0; d < kDims; ++d) *reinterpret_cast<float4*>(to + 16 * d) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
            if (g == 0) rec[wrow] = bad ? NAN : m_ref, rec[kTreeRows + wrow] = l_run;
        } else if (!bad) {
            const float inv = l_run == 0.0f ? 0.0f : (E4M3 ? c.v_scale[kvh] : 1.0f) / l_run;
            uint16_t* to = a.out + (int64_t)m_row * a.out_row + head * D + 4 * g;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
                *reinterpret_cast<uint2*>(to + 16 * d) = make_uint2(pk_bf16(o[d][0] * inv, o[d][1] * inv), pk_bf16(o[d][2] * inv, o[d][3] * inv));
        }
    }
    if (bad && threadIdx.x == 0) atomicOr(c.err, kErrPaged);
    if (odd && !bad)
        careful_piece<E4M3>(c, a, t, kvh, r0, nr, lo, hi, [&](int, const Row& x) { return a.q + x.m * a.q_row + x.h * D; }, rec, kTreeRows);
}

}  // namespace
}  // namespace moa
