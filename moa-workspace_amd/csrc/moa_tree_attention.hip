// moa_tree_attention.hip -- attention of drafted trees over the paged cache (include/moa_paged.h) for sequences of a few dozen rows.
//
// Every row of a tree sees the positions before it, so K and V of a sequence are read once for up to 16 RB rows, and the
// kernel is bound by their bytes: they go from memory to registers and never through LDS, each of four waves taking tiles of 16 or 32
// positions in turn, as in the kernel of few rows (moa_paged_attention.hip), whose lane layouts these are. What a wave
// has of K and V it uses for RB blocks of 16 rows, whose queries are in LDS and whose outputs in registers.
#include <algorithm>

#include "moa_paged_rows.h"

namespace moa {
namespace {

constexpr int kTreeMaxRows = 128;  // of a sequence: two passes over its K and V

template <int D, bool E4M3, int RB>  // RB: 2 or 4
struct TreeShape {
    static constexpr int kElem = E4M3 ? 1 : 2;
    static constexpr int kRows = 16 * RB;                                       // of a tile
    static constexpr int kSub = D * kElem >= 512 ? 1 : 2;                       // 16 positions each
    static constexpr int kTile = 16 * kSub;
    static constexpr int kHeld = RB * D <= 256 ? 2 : 1;                         // workgroups on a CU: waves per SIMD
    static constexpr int kKLoads = D * kElem / 64;                              // 16-byte loads of a K row per lane
    static constexpr int kVD = (E4M3 ? 16 : 8) < D / 16 ? (E4M3 ? 16 : 8) : D / 16;  // dims per V load
    static constexpr int kVB = D / (16 * kVD);                                  // V loads of a row per lane
    static constexpr int kVWords = kVD * kElem / 4;
    static constexpr int kQStride = D + 8;                                      // LDS row of Q: 16 rows start on 16 bank groups
    static constexpr int kQBytes = kRows * kQStride * 2;
    static constexpr int kLds = kQBytes + 4 * 16 * D * 4 + 2 * 4 * 16 * 4;
};

// The units of kTokenUnit positions of all sequences' tiles, a sequence's tiles behind each other, are one row of U, dealt out evenly: group
// w of `groups` takes units [w q, (w + 1) q), q = ceil(U / groups), crossing from tile to tile. A part that is not its whole tile leaves a
// record: number 2 w where it begins inside its tile, 2 w + 1 where it begins it, so split j of a tile that begins in group w0 is
// record 2 (w0 + j) + (j == 0).
struct TreeWalk {
    int64_t units, q;  // U, q
    int base;          // the 64 sequences looked at
    int64_t before;    // units before them
};

// Inclusive sums of numbers below 2^50: the low 20 bits and the others apart.
__device__ __forceinline__ int64_t scan_sum64(int64_t x) { return ((int64_t)scan_sum((int)(x >> 20)) << 20) + scan_sum((int)(x & 0xfffff)); }
__device__ __forceinline__ int64_t lane64(int64_t v, int l) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, l));
}
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {  // of numbers that are not negative; real calls' fit 32 bits
    return (a | b) >> 31 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

template <int R>
__device__ __forceinline__ int tree_tiles(const PagedTreeCall& a, const Seq& q) { return (q.n * a.group + R - 1) / R; }

template <int R>
__device__ TreeWalk tree_walk(const PagedView& c, const PagedTreeCall& a, int groups, int align) {
    TreeWalk w = {0, 1, 0, 0};
    bool bad = false;
    for (int base = 0; base < c.sequences; base += 64) {
        const Seq q = seq_of<true>(c, a, base + (threadIdx.x & 63), true, &bad);
        w.units += (int64_t)tree_tiles<R>(a, q) * token_units(a, q, align);
    }
    raise_bad(c, bad);
    w.units = lane64(scan_sum64(w.units), 63);
    w.q = quotient(w.units + groups - 1, groups);
    w.q = w.q ? w.q : 1;
    return w;
}

// The tile that unit u (not before an earlier call's) belongs to, its units and the first of them. u < w.units.
template <int R>
__device__ void tree_at(const PagedView& c, const PagedTreeCall& a, TreeWalk& w, int align, int64_t u, Piece* out, int* units, int64_t* first) {
    const int lane = threadIdx.x & 63;
    bool bad = false;
    for (;; w.base += 64) {
        const Seq q = seq_of<true>(c, a, w.base + lane, true, &bad);
        const int n = token_units(a, q, align);
        const int64_t all = (int64_t)tree_tiles<R>(a, q) * n, x = scan_sum64(all), end = lane64(x, 63);
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

// A row's weights are 2^(x - reference), the reference its largest x in the first tile where it sees anything: outputs are never rescaled,
// since a branch that does, however rarely, has the compiler move all of them between the matrix cores' and the vector registers in every
// step (64 rows of 256 dims: 476 moves). Weights may be large: f32 sums and pairs of bf16 keep their relative precision up to 2^kRise
// (times values of 2^60; beyond, the sums are infinite, and the careful path takes the rows). A wave that meets a larger x starts its part
// again with the largest x so far.
constexpr float kRise = 64.0f;

// Up to kRows rows of a sequence over a part of its positions.
template <int D, bool E4M3, int RB>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(TreeShape<D, E4M3, RB>::kHeld))) void paged_tree_kernel(
    PagedView c, PagedTreeCall a, float* part) {
    using T = TreeShape<D, E4M3, RB>;
    constexpr int NT = T::kSub;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
    uint16_t* qs = reinterpret_cast<uint16_t*>(lds);                   // [kRows][kQStride]
    float* os = reinterpret_cast<float*>(lds + T::kQBytes);            // [4 waves][16][D]
    float(*ms)[16] = reinterpret_cast<float(*)[16]>(os + 4 * 16 * D);
    float(*ls)[16] = ms + 4;
    const int groups = gridDim.x / c.kv_heads, kvh = blockIdx.x % c.kv_heads, group = blockIdx.x / c.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    // x = factor (q . k): a negative factor's sign goes to q, so that the largest product is the largest x; and a factor of
    // zero stays above it, so that a product of -inf (a position that a row does not see) stays -inf (a NaN stays one)
    const float signed_factor = E4M3 ? c.k_scale[kvh] * a.scale_log2 : a.scale_log2;
    const float factor = fabsf(signed_factor) < 1.2e-38f ? 1.2e-38f : fabsf(signed_factor);
    const uint32_t flip = signed_factor < 0.0f ? 0x80008000u : 0u;
    TreeWalk walk = tree_walk<T::kRows>(c, a, groups, T::kTile);
    const int64_t end = min(walk.units, (group + 1) * walk.q);
    for (int64_t unit = group * walk.q; unit < end;) {
        Piece t;
        int units;
        int64_t first;
        tree_at<T::kRows>(c, a, walk, T::kTile, unit, &t, &units, &first);
        const int off = (int)(unit - first), take = (int)min((int64_t)(units - off), end - unit);
        const bool whole = off == 0 && take == units;
        unit += take;
        const int r0 = t.tile * T::kRows, nr = min(T::kRows, t.n * a.group - r0), from = token_first(a, Seq{t.row0, t.n, t.len}, T::kTile);
        const int lo = from + off * kTokenUnit, hi = (int)min((int64_t)lo + (int64_t)take * kTokenUnit, (int64_t)t.len), tree0 = t.len - t.n;
        // as many blocks of 16 rows as there are
        auto run = [&](auto blocks) __attribute__((always_inline)) {
            constexpr int NB = decltype(blocks)::value;
            __syncthreads();  // the part before has been written out
            for (int i = threadIdx.x; i < 16 * NB * D / 8; i += 256) {
                const int r = i / (D / 8), j = i - r * (D / 8), row = r0 + min(r, nr - 1), node = row / a.group;
                const uint4 w = ld16(a.q + (int64_t)(t.row0 + node) * a.q_row + (kvh * a.group + row - node * a.group) * D + 8 * j);
                *reinterpret_cast<uint4*>(qs + r * T::kQStride + 8 * j) = make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
            }
            int see_lo[NB], see_hi[NB], mask_row[NB];  // of row 16 b + l16; -1: no row
            int all_lo = 0, all_hi = t.len;            // positions that all rows see
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const bool is = 16 * b + l16 < nr;
                const Row x = row_of(a, t, kvh, r0 + min(16 * b + l16, nr - 1));
                see_lo[b] = is ? x.lo : 0, see_hi[b] = is ? x.hi : 0, mask_row[b] = is ? (int)x.m : -1;
                all_lo = max(all_lo, x.lo), all_hi = min(all_hi, x.hi);
            }
#pragma unroll
            for (int b = 8; b > 0; b >>= 1) all_lo = max(all_lo, __shfl_xor(all_lo, b)), all_hi = min(all_hi, __shfl_xor(all_hi, b));
            all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
            __syncthreads();

            f32x4 o[NB][T::kVB][T::kVD];
            float m_run[NB], m_ref[NB], l_run[NB];
#pragma unroll
            for (int r = 0; r < NB; ++r) m_run[r] = -INFINITY;
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

            constexpr int kStep = 4 * T::kTile;
            bool over = false;
            do {
                int t0 = lo + wave * T::kTile;
                int page = page_at(t0), page1 = page_at(t0 + kStep);
                place(page, t0);
                if (t0 < hi) load_k();
#pragma unroll
                for (int r = 0; r < NB; ++r) {
                    m_ref[r] = m_run[r], l_run[r] = 0.0f;
#pragma unroll
                    for (int b = 0; b < T::kVB; ++b)
#pragma unroll
                        for (int d = 0; d < T::kVD; ++d) o[r][b][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
                over = false;
                for (; t0 < hi && !over; t0 += kStep) {
                    load_v();
                    if constexpr (NB * D > 256) __asm__ volatile("" ::: "memory");  // Q is read from LDS again: no registers for it
                    f32x4 sc[NB][NT];
#pragma unroll
                    for (int r = 0; r < NB; ++r)
#pragma unroll
                        for (int i = 0; i < NT; ++i) sc[r][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    // Q's dims follow the order K's 16-byte loads have: bf16 dims 32 j + 8 g, E4M3 dims 64 j + 16 g, two steps a load
#pragma unroll
                    for (int j = 0; j < T::kKLoads; ++j)
#pragma unroll
                        for (int h = 0; h < (E4M3 ? 2 : 1); ++h) {
                            bf16x8 kb[NT];
#pragma unroll
                            for (int i = 0; i < NT; ++i) {
                                if constexpr (E4M3) {
                                    const uint32_t w0 = h ? kf[i][j].z : kf[i][j].x, w1 = h ? kf[i][j].w : kf[i][j].y;
                                    kb[i] = as_bf16x8(make_uint4(bf16_pair_of_fp8(w0), bf16_pair_of_fp8(w0 >> 16), bf16_pair_of_fp8(w1), bf16_pair_of_fp8(w1 >> 16)));
                                } else {
                                    kb[i] = as_bf16x8(kf[i][j]);
                                }
                            }
#pragma unroll
                            for (int r = 0; r < NB; ++r) {
                                const bf16x8 qf = as_bf16x8(ld16(qs + (16 * r + l16) * T::kQStride + (E4M3 ? 64 * j + 16 * g + 8 * h : 32 * j + 8 * g)));
#pragma unroll
                                for (int i = 0; i < NT; ++i) sc[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb[i], qf, sc[r][i], 0, 0, 0);
                            }
                        }
                    // the next tile's K
                    page = page1;
                    page1 = page_at(t0 + 2 * kStep);
                    place(page, t0 + kStep);
                    if (t0 + kStep < hi) load_k();

                    const bool some = t0 < all_lo || t0 + T::kTile > all_hi;  // some row does not see all of it
                    uint32_t pw[NB][2 * NT][kParts];
#pragma unroll
                    for (int r = 0; r < NB; ++r) {
                        // weights of row 16 r + l16 at positions t0 + 16 i + 4 g + e
                        if (some) {
                            const uint32_t nodes = t0 + T::kTile > tree0 && mask_row[r] >= 0 ? (uint32_t)node_bits(a, t, mask_row[r], t0) : 0;
#pragma unroll
                            for (int i = 0; i < NT; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int p = t0 + 16 * i + 4 * g + e;
                                    const bool sees = (p >= see_lo[r] && p < see_hi[r]) || (nodes >> (16 * i + 4 * g + e) & 1);
                                    sc[r][i][e] = sees ? sc[r][i][e] : -INFINITY;
                                }
                        }
                        float mx = sc[r][0][0];
#pragma unroll
                        for (int i = 0; i < NT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[r][i][e]);
                        mx = fmaxf(mx, __shfl_xor(mx, 16));
                        mx = fmaxf(mx, __shfl_xor(mx, 32));
                        m_run[r] = fmaxf(m_run[r], mx * factor);
                        m_ref[r] = m_ref[r] == -INFINITY ? m_run[r] : m_ref[r];
                        over |= __any(m_run[r] > m_ref[r] + kRise);
                        const float mu = m_ref[r] == -INFINITY ? 0.0f : m_ref[r];
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < NT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; e += 2) {
                                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[r][i][e], factor, -mu)), p1 = __builtin_amdgcn_exp2f(fmaf(sc[r][i][e + 1], factor, -mu));
                                sum += p0 + p1;
                                split_weights(p0, p1, pw[r][2 * i + e / 2]);
                            }
                        l_run[r] += sum;
                    }
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
#pragma unroll
                            for (int r = 0; r < NB; ++r) {
                                if constexpr (NT == 1) {
                                    o[r][b][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(make_uint4(pw[r][0][0], pw[r][1][0], pw[r][0][1], pw[r][1][1])),
                                                                                         as_bf16x8(make_uint4(w[0], w[1], w[0], w[1])), o[r][b][d], 0, 0, 0);
                                } else {
#pragma unroll
                                    for (int p = 0; p < kParts; ++p)
                                        o[r][b][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(make_uint4(pw[r][0][p], pw[r][1][p], pw[r][2][p], pw[r][3][p])),
                                                                                             as_bf16x8(make_uint4(w[0], w[1], w[2], w[3])), o[r][b][d], 0, 0, 0);
                                }
                            }
                        }
                }
            } while (over);

            // the four waves' states into one, 16 rows at a time
            bad = __syncthreads_or(bad);
            float* rec = whole ? nullptr : part + ((int64_t)kvh * 2 * groups + 2 * group + (off == 0)) * record_floats(T::kRows, D);
            bool odd = false;
            const float vs = E4M3 ? c.v_scale[kvh] : 1.0f;
#pragma unroll
            for (int r = 0; r < NB; ++r) {
                if (16 * r >= nr) continue;
                if (r) __syncthreads();  // the rows before have been read
                l_run[r] += __shfl_xor(l_run[r], 16);
                l_run[r] += __shfl_xor(l_run[r], 32);
                if (g == 0) ms[wave][l16] = m_ref[r], ls[wave][l16] = l_run[r];
#pragma unroll
                for (int b = 0; b < T::kVB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int d = 0; d < T::kVD; d += 4)
                            *reinterpret_cast<float4*>(os + ((wave * 16 + 4 * g + e) * D + 16 * T::kVD * b + T::kVD * l16 + d)) =
                                make_float4(o[r][b][d][e], o[r][b][d + 1][e], o[r][b][d + 2][e], o[r][b][d + 3][e]);
                __syncthreads();
                const int here = min(16, nr - 16 * r);
                for (int i = threadIdx.x; i < here * (D / 4); i += 256) {
                    const int y = i / (D / 4), d = 4 * (i - y * (D / 4));
                    const float m = fmaxf(fmaxf(ms[0][y], ms[1][y]), fmaxf(ms[2][y], ms[3][y]));
                    float l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float f = ms[w][y] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms[w][y] - m);
                        const float4 z = *reinterpret_cast<const float4*>(os + (w * 16 + y) * D + d);
                        l = fmaf(f, ls[w][y], l);
                        v[0] = fmaf(f, z.x, v[0]), v[1] = fmaf(f, z.y, v[1]), v[2] = fmaf(f, z.z, v[2]), v[3] = fmaf(f, z.w, v[3]);
                    }
                    odd |= !(fabsf(v[0]) + fabsf(v[1]) + fabsf(v[2]) + fabsf(v[3]) < INFINITY);
                    const int row = 16 * r + y;
                    if (rec) {
                        if (d == 0) rec[row] = bad ? NAN : m, rec[T::kRows + row] = l;
                        *reinterpret_cast<float4*>(rec + 2 * T::kRows + row * D + d) = make_float4(v[0], v[1], v[2], v[3]);
                    } else if (!bad) {
                        const int node = (r0 + row) / a.group;
                        const float inv = l == 0.0f ? 0.0f : vs / l;
                        *reinterpret_cast<uint2*>(a.out + (int64_t)(t.row0 + node) * a.out_row + (kvh * a.group + r0 + row - node * a.group) * D + d) =
                            make_uint2(pk_bf16(v[0] * inv, v[1] * inv), pk_bf16(v[2] * inv, v[3] * inv));
                    }
                }
            }
            odd = __syncthreads_or(odd);
            if (bad && threadIdx.x == 0) atomicOr(c.err, kErrPaged);
            if (odd && !bad && flip) {  // q as it was
                for (int i = threadIdx.x; i < 16 * NB * D / 2; i += 256) reinterpret_cast<uint32_t*>(qs)[i / (D / 2) * (T::kQStride / 2) + i % (D / 2)] ^= flip;
                __syncthreads();
            }
            if (odd && !bad)
                careful_piece<E4M3>(c, a, t, kvh, r0, nr, lo, hi, [&](int r, const Row&) { return qs + r * T::kQStride; }, rec, T::kRows);
        };
        const int blocks = (nr + 15) / 16;
        if (blocks == 1) run(std::integral_constant<int, 1>{});
        if (blocks == 2) run(std::integral_constant<int, 2>{});
        if constexpr (RB == 4) {
            if (blocks == 3) run(std::integral_constant<int, 3>{});
            if (blocks == 4) run(std::integral_constant<int, 4>{});
        }
    }
}

// Rows of split tiles, four in a workgroup, a wave each.
constexpr int kTreeMergeRows = 4;

// Block `want` of the rows of the tiles that are split: its sequence, tile, parts, first record and first row in the tile. False: there are
// not that many.
template <int R>
__device__ bool tree_block(const PagedView& c, const PagedTreeCall& a, const TreeWalk& w, int align, int want, Piece* out) {
    const int lane = threadIdx.x & 63;
    bool bad = false;
    int64_t before = 0;
    for (int base = 0; base < c.sequences; base += 64) {
        const Seq q = seq_of<true>(c, a, base + lane, true, &bad);
        const int n = token_units(a, q, align), tiles = tree_tiles<R>(a, q), rows = q.n * a.group;
        const int64_t all = (int64_t)tiles * n, x = scan_sum64(all), first = before + x - all;
        // a sequence's tiles are split but for those that a group has whole; each is looked at below
        int blocks = 0;
        for (int i = 0; i < tiles; ++i) {
            const int64_t u = first + (int64_t)i * n;
            if (quotient(u, w.q) != quotient(u + n - 1, w.q)) blocks += (min(R, rows - i * R) + kTreeMergeRows - 1) / kTreeMergeRows;
        }
        const int xb = scan_sum(blocks);
        const uint64_t hit = __ballot(xb > want);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            int left = want - get(xb - blocks);
            const int64_t u0 = lane64(first, l);
            const int un = get(n), ur = get(rows);
            for (int i = 0;; ++i) {
                const int64_t u = u0 + (int64_t)i * un, w0 = quotient(u, w.q), w1 = quotient(u + un - 1, w.q);
                if (w0 == w1) continue;
                const int here = (min(R, ur - i * R) + kTreeMergeRows - 1) / kTreeMergeRows;
                if (left < here) {
                    *out = {base + l, get(q.row0), get(q.n), get(q.len), i, 0, (int)(w1 - w0) + 1, (int)(2 * w0), left * kTreeMergeRows};
                    return true;
                }
                left -= here;
            }
        }
        want -= __builtin_amdgcn_readlane(xb, 63);
        before += lane64(x, 63);
    }
    return false;
}

template <int D, bool E4M3, int RB>
__global__ __launch_bounds__(256) void paged_tree_merge_kernel(PagedView c, PagedTreeCall a, int groups, const float* part) {
    using T = TreeShape<D, E4M3, RB>;
    const int kvh = blockIdx.x % c.kv_heads;
    const TreeWalk walk = tree_walk<T::kRows>(c, a, groups, T::kTile);
    const int64_t size = record_floats(T::kRows, D);
    Piece t;
    for (int u = blockIdx.x / c.kv_heads; tree_block<T::kRows>(c, a, walk, T::kTile, u, &t); u += gridDim.x / c.kv_heads) {
        const float* base = part + ((int64_t)kvh * 2 * groups + t.record) * size;
        auto rec = [&](int j) { return base + (2 * j + (j == 0)) * size; };
        const int r = t.row + (threadIdx.x >> 6), row = t.tile * T::kRows + r;
        if (r < T::kRows && row < t.n * a.group) merge_row<D, E4M3>(c, a, t, kvh, rec, T::kRows, r, row);
    }
}

template <int D, bool E4M3, int RB>
hipError_t launch_tree(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx) {
    using T = TreeShape<D, E4M3, RB>;
    const int heads = c.kv_heads;
    const int64_t capacity = (int64_t)c.columns * c.slots, sequences = std::min(c.sequences, a.rows);
    const int64_t units = (a.window ? std::min<int64_t>(capacity, (int64_t)a.window + a.max_rows + kTokenUnit) : capacity) / kTokenUnit + 1;
    const int64_t tiles = (int64_t)a.rows * a.group / T::kRows + sequences;
    const int64_t most = (int64_t)kPagedChunkFloats / record_floats(T::kRows, D) / heads / 2;
    const int groups = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>((int64_t)ctx->cus * T::kHeld / heads, tiles * units), most));
    hipLaunchKernelGGL((paged_tree_kernel<D, E4M3, RB>), dim3((uint32_t)(groups * heads)), dim3(256), 0, s, c, a, ctx->paged_chunks);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || groups == 1) return e;
    // a split tile has a cut between two groups
    const int64_t blocks = std::min<int64_t>((int64_t)(groups - 1) * (T::kRows / kTreeMergeRows), (int64_t)a.rows * a.group / kTreeMergeRows + tiles);
    const int64_t wgs = std::min<int64_t>(blocks, std::max(1, 2048 / heads));
    hipLaunchKernelGGL((paged_tree_merge_kernel<D, E4M3, RB>), dim3((uint32_t)(wgs * heads)), dim3(256), 0, s, c, a, groups, ctx->paged_chunks);
    return hipGetLastError();
}

template <int D, int RB>
hipError_t launch_type(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx) {
    return c.k_scale ? launch_tree<D, true, RB>(c, a, s, ctx) : launch_tree<D, false, RB>(c, a, s, ctx);
}

template <int D>
hipError_t launch_rows(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx) {
    return a.max_rows * a.group <= 32 ? launch_type<D, 2>(c, a, s, ctx) : launch_type<D, 4>(c, a, s, ctx);
}

}  // namespace

hipError_t launch_paged_tree_attention(const PagedView& c, const PagedTreeCall& a, hipStream_t s, DevCtx* ctx) {
    const int rows = a.max_rows * a.group;
    if (rows <= kTokenRows || rows > kTreeMaxRows || c.head_dim > 256) return launch_paged_tree_rows(c, a, s, ctx);
    switch (c.head_dim) {
        case 64: return launch_rows<64>(c, a, s, ctx);
        case 128: return launch_rows<128>(c, a, s, ctx);
        default: return launch_rows<256>(c, a, s, ctx);
    }
}

}  // namespace moa
