// moa_search.hip -- tokens from logits (include/moa_search.h): the greedy verification of drafted trees, and the selection of
// beams. Both read every row of bf16 logits once, at the rate of memory (524 rows of 262144, 275 MB: 45 us, 6.1 TB/s; the 151 live rows of a
// selection, with exponentials and their f64 sums beside, 79 MB: 19 us, 4.2 TB/s); what is left of a row then fits a workgroup.
#include <algorithm>

#include "../../include/moa_search.h"
#include "moa_arrive.h"
#include "moa_checks.h"
#include "moa_device.h"
#include "moa_sync.h"

namespace moa {
namespace {

constexpr int kBlock = 256;
constexpr int kGroupLogits = 64;        // logits that share a key (their largest): 8 lanes' 16 bytes
constexpr int kSearchMaxVocab = 1 << 20;

constexpr unsigned kGroupTurn = 128;  // of the counters of a group's rows

typedef short s16x2 __attribute__((ext_vector_type(2)));

// Logits in the order of their values as 16-bit integers, -0 the same as 0 and every NaN below -infinity: negative ones have
// their other bits inverted and one added, which closes the gap that -0 leaves; then 127 are added, which carries the NaNs of positive
// sign around, and those of both signs end below -infinity, kNanKey at most.
constexpr short kNanKey = -32514;
__device__ __forceinline__ s16x2 ordered(uint32_t two) {
    const s16x2 b = __builtin_bit_cast(s16x2, two), sign = b >> 15;
    const s16x2 o = (b ^ (sign & (short)0x7fff)) - sign + (short)127;
    return __builtin_elementwise_max(o, (s16x2)kNanKey);
}
// The value of a key that is no NaN's.
__device__ __forceinline__ float key_value(int key) {
    const int o = key - 127;
    return bf2f((uint32_t)(o < 0 ? (o - 1) ^ 0x7fff : o) & 0xffffu);
}
constexpr int kLowestFinite = kNanKey + 2;  // behind NaN and -infinity

constexpr uint32_t kNan = 0xffffu, kMinusInfinity = 0xff80u;

// A row of logits in chunks of eight from its first on, wherever it lies: a row's sums then do not depend on its address, so that
// equal rows have equal totals. (Loads of 16 bytes need not be aligned.)
struct LogitRow {
    const uint16_t* p;
    int vocab;
    __device__ LogitRow(const uint16_t* logits, int64_t stride, int64_t row, int n) : p(logits + row * stride), vocab(n) {}
    // Elements behind the row are not read; they come as `outside`.
    __device__ uint4 chunk(int c, uint32_t outside) const {
        const int e = 8 * c;
        uint4 v;
        if (e + 8 <= vocab) {
            __builtin_memcpy(&v, p + e, 16);
            return v;
        }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = e + 2 * i;
            const uint32_t lo = x < vocab ? p[x] : outside, hi = x + 1 < vocab ? p[x + 1] : outside;
            w[i] = lo | hi << 16;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ int larger(const s16x2& m) { return max((int)m[0], (int)m[1]); }

__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, kWave));
    return v;
}

constexpr int kMaxParts = kSearchMaxVocab / (kBlock * 8 * 2);
// A row's parts: 256 threads of kLoads chunks each.
__host__ __device__ inline int parts_of(int vocab, int loads) { return (vocab + kBlock * 8 * loads - 1) / (kBlock * 8 * loads); }

// ---------------------------------------------------------------------------------------------- verify

// The largest logit of this workgroup's part of row blockIdx.y and its first place, as one number that orders by both, in thread 0.
template <int kLoads>
__device__ uint64_t verify_scan(const uint16_t* logits, int64_t stride, int vocab) {
    __shared__ int top[4];
    __shared__ uint32_t at[4];
    const LogitRow row(logits, stride, blockIdx.y, vocab);
    const int wave = threadIdx.x >> 6, first = blockIdx.x * kBlock * kLoads + threadIdx.x;
    uint4 w[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) w[j] = row.chunk(first + j * kBlock, kNan);
    s16x2 o[kLoads][4], m = (s16x2)(short)-32768;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        o[j][0] = ordered(w[j].x), o[j][1] = ordered(w[j].y), o[j][2] = ordered(w[j].z), o[j][3] = ordered(w[j].w);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, o[j][i]);
    }
    int most = wave_max(larger(m));
    if ((threadIdx.x & 63) == 0) top[wave] = most;
    __syncthreads();
    most = max(max(top[0], top[1]), max(top[2], top[3]));
    uint32_t place = ~0u;  // (places behind the row are larger than all in it)
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            place = min(place, o[j][i / 2][i & 1] == most ? (uint32_t)(8 * (first + j * kBlock) + i) : ~0u);
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) place = min(place, (uint32_t)__shfl_xor((int)place, k, kWave));
    if ((threadIdx.x & 63) == 0) at[wave] = place;
    __syncthreads();
    return (uint64_t)(uint32_t)(most + 32768) << 32 | ~min(min(at[0], at[1]), min(at[2], at[3]));
}

struct VerifyCall {
    const uint16_t* logits; int64_t stride;
    const int32_t* tokens; const int32_t* starts; const uint64_t* masks;
    int32_t* best; int32_t* leaves; int32_t* next;
    int words, rows, vocab, sequences;
    uint32_t* err;
};

// The rows of sequence s: false, with the sequence's outputs written, where it has none.
__device__ __forceinline__ bool verify_rows(const VerifyCall& c, int s, bool first, int* row0, int* n) {
    const int begin = c.starts[s], end = c.starts[s + 1];
    const bool out = !rows_in_range(begin, end, c.rows, 64 * c.words);
    *row0 = begin, *n = out ? 0 : end - begin;
    if (*n == 0 && first) {
        c.leaves[s] = c.next[s] = -1;
        if (out && begin != end) atomicOr(c.err, kErrPaged);
    }
    return *n > 0;
}

// The walk of a sequence of n rows by one wave, kWords nodes a lane: what it needs of the rows, asked for ahead of their tokens, and the
// walk along `named`, the rows' tokens. (Trees of up to 64 nodes have one word: the compares of four are most of a step.)
template <int kWords>
struct VerifyWalk {
    uint64_t mask[kWords][kWords];
    int32_t token[kWords];

    __device__ __forceinline__ void load(const VerifyCall& c, int row0, int n) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
            const int i = 64 * k + lane;
            token[k] = i < n ? c.tokens[row0 + i] : 0;
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                const int left = n - 64 * w;
                mask[k][w] = i < n && w < c.words && left > 0 ? c.masks[(int64_t)(row0 + i) * c.words + w] & (left >= 64 ? ~0ull : (1ull << left) - 1) : 0;
            }
        }
    }

    __device__ __forceinline__ void walk(const VerifyCall& c, int s, int n, const int32_t* named) {
        const int lane = threadIdx.x & 63;
        auto of = [&](uint64_t v, int l) {
            return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, l) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32;
        };
        if (!(of(mask[0][0], 0) & 1)) {  // node 0 is none
            if (lane == 0) c.leaves[s] = c.next[s] = -1;
            return;
        }
        int cur = 0;
        for (int step = 0; step < n; ++step) {
            const int want = named[cur];
            uint64_t sees[kWords];
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                uint64_t x = mask[0][w];
#pragma unroll
                for (int k = 1; k < kWords; ++k) x = cur >= 64 * k ? mask[k][w] : x;
                sees[w] = of(x, cur & 63);
            }
            int child = -1;
#pragma unroll
            for (int k = 0; k < kWords; ++k) {
                bool is = token[k] == want && (mask[k][k] >> lane & 1) && 64 * k + lane < n && !(sees[k] >> lane & 1);
#pragma unroll
                for (int w = 0; w < kWords; ++w) is = is && (mask[k][w] & ~(w == k ? 1ull << lane : 0ull)) == sees[w];
                const uint64_t hit = __ballot(is);
                if (child < 0 && hit) child = 64 * k + __builtin_ctzll(hit);
            }
            if (child < 0) break;
            cur = child;
        }
        if (lane == 0) c.leaves[s] = cur, c.next[s] = named[cur];
    }
};

template <int kLoads>
__global__ __launch_bounds__(kBlock) void verify_scan_kernel(VerifyCall c, uint64_t* part) {
    const uint64_t best = verify_scan<kLoads>(c.logits, c.stride, c.vocab);
    if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = best;
}

// One workgroup per sequence: its rows' parts into tokens, then the walk. (24 trees of 5 to 33 nodes: 6 us; 9.6 with four words of masks that are
// asked for behind the tokens.)
template <int kWords>
__global__ __launch_bounds__(kBlock) void verify_walk_kernel(VerifyCall c, const uint64_t* part, int parts) {
    __shared__ int32_t named[kTreeMaxNodes];
    const int s = blockIdx.x, t = threadIdx.x;
    int row0, n;
    if (!verify_rows(c, s, t == 0, &row0, &n)) return;
    VerifyWalk<kWords> tree;
    if (t < kWave) tree.load(c, row0, n);
    int lanes = 1;  // that share a row
    while (lanes < 64 && lanes < parts) lanes *= 2;
    for (int r = t / lanes; r < n; r += kBlock / lanes) {
        uint64_t key = 0;
        for (int i = t % lanes; i < parts; i += lanes) key = max(key, part[(int64_t)(row0 + r) * parts + i]);
        for (int o = lanes / 2; o > 0; o >>= 1) key = max(key, (uint64_t)__shfl_xor((long long)key, o, kWave));
        if (t % lanes == 0) c.best[row0 + r] = named[r] = (int32_t) ~(uint32_t)key;
    }
    __syncthreads();
    if (t < kWave) tree.walk(c, s, n, named);
}

// Few rows and sequences in one launch: the last part of a row to arrive names its token, the last row's workgroup walks, a wave per
// sequence. Against scan and walk as two launches, one sequence, us a call here / there at 8, 33, 64, 128 and 256 rows: 262144 logits 8.6 / 11.3,
// 9.1 / 11.4, 12.9 / 16.3, 20.6 / 27.6, 34.5 / 49.3; 32000 logits 8.8 / 11.5 up to 128 rows, 11.6 / 11.4 at 256. As a graph's nodes,
// where a second launch costs little, up to 8 rows are level at 262144 (6.8 both) and 32000 logits 0.6 to 0.9 slower (7.1 / 6.4 at 64).
constexpr int kFewSequences = 4;
template <int kWords>
__global__ __launch_bounds__(kBlock) void verify_few_kernel(VerifyCall c, uint64_t* part, uint32_t* row_best, uint32_t* tickets) {
    __shared__ int32_t named[kTreeMaxNodes];
    const int t = threadIdx.x, parts = gridDim.x, row = blockIdx.y;
    const uint64_t best = verify_scan<2>(c.logits, c.stride, c.vocab);
    if (t == 0) publish64(part + (int64_t)row * parts + blockIdx.x, best);
    if (!arrive_last<kRowTurn>(tickets + (int64_t)row * kTicketStride, blockIdx.x == 0, parts)) return;
    if (t < kWave) {
        uint64_t key = 0;
        for (int i = t; i < parts; i += kWave) key = max(key, collect64(part + (int64_t)row * parts + i));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) key = max(key, (uint64_t)__shfl_xor((long long)key, o, kWave));
        if (t == 0) publish32(row_best + row, ~(uint32_t)key);
    }
    if (!arrive_last<kRowTurn>(tickets + (int64_t)kTreeMaxNodes * kTicketStride, row == 0, c.rows)) return;
    if (t < c.rows) named[t] = (int32_t)__hip_atomic_load(row_best + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int s = t >> 6, lane = t & 63;
    int row0, n;
    if (s >= c.sequences || !verify_rows(c, s, lane == 0, &row0, &n)) return;
    VerifyWalk<kWords> tree;
    tree.load(c, row0, n);
    for (int i = lane; i < n; i += kWave) c.best[row0 + i] = named[row0 + i];
    tree.walk(c, s, n, named + row0);
}

// ---------------------------------------------------------------------------------------------- select

// Of a part of a row: the sum of e^(logit - ref), ref its lanes' largest reference.
struct PartSum { double sum; float ref; };

// What a selection keeps of each row of a launch: the keys of its groups of logits, its parts' sums, its candidates, and the counters of
// what has arrived.
struct SelectScratch {
    uint16_t* keys;        // [rows][key_stride]: the largest logit of a group, ordered() + 32768
    PartSum* parts;        // [rows][parts_n]
    uint64_t* totals;      // [rows][beams] f64, descending
    uint32_t* places;      // [rows][beams]
    uint32_t* tickets;     // a line for every group of beams
    int groups, key_stride, parts_n;  // of a row
};

struct SelectCall {
    const uint16_t* logits; int64_t stride;
    const float* scores; const int32_t* finished;
    float* out_scores; int32_t* out_finished; int32_t* parents; int32_t* tokens;
    int beams, vocab, eos, row0;  // first row of this launch
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 2.0f;  // what a logit may lie above its lane's reference: the larger, the more an exponential's argument is rounded

// A beam that adds candidates from its logits.
__device__ __forceinline__ bool grows(const SelectCall& c, int row) { return c.finished[row] == 0 && c.scores[row] > -INFINITY; }

// One pass over a part of a row: the keys of its groups, and its reference and sum.
template <int kLoads>
__global__ __launch_bounds__(kBlock) void select_scan_kernel(SelectCall c, SelectScratch k) {
    constexpr int kGroups = kBlock * kLoads / 8;  // of a part
    __shared__ double sums[4];
    __shared__ float top[4];
    __shared__ __attribute__((aligned(8))) uint16_t keys[kGroups];
    const int r = blockIdx.y;
    if (!grows(c, c.row0 + r)) return;
    const LogitRow row(c.logits, c.stride, c.row0 + r, c.vocab);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = blockIdx.x * kBlock * kLoads + threadIdx.x;
    uint4 w[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) w[j] = row.chunk(first + j * kBlock, kMinusInfinity);
    // The lane's sum stands against a reference that follows its largest logit so far, so that its first chunks are summed while the
    // others are on their way. It is f64 from the first exponential on: beside a logit that stands out every other one can be below f32's
    // last bit, and a beam whose total differs by their sum would come in the wrong place. (151 rows of 262144: 1 us more a call than f32
    // sums, 0.6 with exponentials added in pairs first.)
    float m = -INFINITY;
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        float x[8];
        bf16x8_to_f32(w[j], x);
        float most = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, x[i]);
        if (most > m + kSlack) {
            sum *= (double)__builtin_amdgcn_exp2f((m - most) * kLog2e);
            m = most;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += (double)__builtin_amdgcn_exp2f((x[i] - ref) * kLog2e);
#pragma unroll
        for (int o = 1; o < 8; o *= 2) most = fmaxf(most, __shfl_xor(most, o, kWave));
        if ((lane & 7) == 0) keys[(j * kBlock + threadIdx.x) / 8] = (uint16_t)(ordered(__float_as_uint(most) >> 16)[0] + 32768);
    }
    float all = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, kWave));
    if (m > -INFINITY) sum *= (double)__builtin_amdgcn_exp2f((m - all) * kLog2e);  // (a NaN in a lane without a finite logit stays)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (lane == 0) top[wave] = all, sums[wave] = sum;
    __syncthreads();
    const int at = (int)blockIdx.x * kGroups + 4 * (int)threadIdx.x;  // four keys a thread
    if ((int)threadIdx.x < kGroups / 4 && at < k.key_stride)
        *reinterpret_cast<uint64_t*>(k.keys + (int64_t)r * k.key_stride + at) = reinterpret_cast<const uint64_t*>(keys)[threadIdx.x];
    if (threadIdx.x == 0) {
        const float part = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) total += top[i] == -INFINITY ? sums[i] : sums[i] * (double)__builtin_amdgcn_exp2f((top[i] - part) * kLog2e);
        k.parts[(int64_t)r * k.parts_n + blockIdx.x] = {total, part};
    }
}

// The largest of the wave's values, the same in every lane: four shifts within rows of 16, then the rows' last lanes (DPP).
__device__ __forceinline__ uint32_t wave_largest(uint32_t x) {
    auto step = [&](uint32_t y) { x = max(x, y); };
    step(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, 63);
}

// The `want` largest of the workgroup's numbers (kN a thread; different but for 0, which is none), in descending order in `out`
// behind a barrier; returns how many there are. Each wave takes its own one after the other, and where a number stands among the
// four waves' lists is counted. lists: [4][kMaxBeams].
template <int kN>
__device__ int block_largest(uint32_t (&v)[kN], int want, uint32_t (*lists)[kMaxBeams], uint32_t* out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) mine = max(mine, v[i]);
    uint32_t kept = 0;  // lane i: number i of the wave's
    for (int i = 0; i < want; ++i) {
        const uint32_t best = wave_largest(mine);
        if (best == 0) break;
        if (lane == i) kept = best;
        if (mine == best) {
            mine = 0;
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                v[j] = v[j] == best ? 0 : v[j];
                mine = max(mine, v[j]);
            }
        }
    }
    __syncthreads();  // the lists of an earlier call have been read
    lists[wave][lane] = kept;
    __syncthreads();
    int rank = lane, n = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        for (int i = 0; i < want; ++i) {
            const uint32_t y = lists[w][i];
            n += y != 0;
            rank += w != wave && y > kept;
        }
    if (kept && rank < want) out[rank] = kept;
    __syncthreads();
    return min(n, want);
}

// The row's candidates: of the groups that come first by key and place, as many as beams (each holds a logit that comes before all of a
// later group's), then of their logits. Numbers order by key, then by place, the lower first.
template <int kKeys>
__device__ void select_row(const SelectCall& c, const SelectScratch& k, int r) {
    __shared__ uint32_t lists[4][kMaxBeams], found[kMaxBeams];
    __shared__ int groups[kMaxBeams];
    __shared__ double row_lse;
    const int row = c.row0 + r, t = threadIdx.x, lane = t & 63;
    uint64_t* totals = k.totals + (int64_t)r * c.beams;
    uint32_t* places = k.places + (int64_t)r * c.beams;
    const float score_f = c.scores[row];
    const int done = c.finished[row];
    const double score = score_f;
    auto put = [&](int i, double total, int place) {
        publish64(totals + i, __builtin_bit_cast(uint64_t, total + 0.0));  // (-0 ties with 0)
        publish32(places + i, (uint32_t)place);
    };
    constexpr int kMost = kMaxParts / kWave;
    PartSum part[kMost];  // the row's sums, in every wave
#pragma unroll
    for (int i = 0; i < kMost; ++i)
        part[i] = i * kWave + lane < k.parts_n ? k.parts[(int64_t)r * k.parts_n + i * kWave + lane] : PartSum{0.0, -INFINITY};
    constexpr uint32_t kLeast = kLowestFinite + 32768;
    const uint16_t* keys = k.keys + (int64_t)r * k.key_stride;
    uint64_t four[kKeys / 4];  // (of a row that adds none: of an earlier call)
#pragma unroll
    for (int j = 0; j < kKeys / 4; ++j) {
        const int at = 4 * (j * kBlock + t);
        four[j] = at < k.groups ? *reinterpret_cast<const uint64_t*>(keys + at) : 0;
    }
    if (done != 0 || !(score_f > -INFINITY)) {
        if (t < c.beams) put(t, t == 0 && c.eos >= 0 && done != 0 && score_f > -INFINITY ? score : -INFINITY, c.eos);
        return;
    }
    uint32_t v[kKeys];
#pragma unroll
    for (int j = 0; j < kKeys / 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 4 * (j * kBlock + t) + i;
            const uint32_t key = (uint32_t)(four[j] >> 16 * i) & 0xffffu;
            v[4 * j + i] = at < k.groups && key >= kLeast ? key << 16 | (0xffffu - at) : 0;
        }
    const int ng = block_largest<kKeys>(v, c.beams, lists, found);
    if (t < ng) {  // in ascending order
        const int g = 0xffff - (int)(found[t] & 0xffffu);
        int rank = 0;
        for (int i = 0; i < ng; ++i) rank += 0xffff - (int)(found[i] & 0xffffu) < g;
        groups[rank] = g;
    }
    __syncthreads();
    const LogitRow logits(c.logits, c.stride, row, c.vocab);
    uint32_t e[16];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = j * kBlock + t;  // 16 bytes of a group
        uint4 w = make_uint4(0, 0, 0, 0);
        if (i < 8 * ng) w = logits.chunk(groups[i / 8] * 8 + i % 8, kMinusInfinity);
        const uint32_t two[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const s16x2 o = ordered(two[h]);
#pragma unroll
            for (int x = 0; x < 2; ++x)
                e[8 * j + 2 * h + x] = i < 8 * ng && o[x] >= kLowestFinite ? (uint32_t)(o[x] + 32768) << 16 | (0xffffu - (8 * i + 2 * h + x)) : 0;
        }
    }
    if (t >= 3 * kWave) {  // the row's sum, by the wave that has no logits of up to 24 beams
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kMost; ++i) m = fmaxf(m, part[i].ref);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kMost; ++i)
            sum += part[i].ref == -INFINITY ? part[i].sum : part[i].sum * (double)__builtin_amdgcn_exp2f((part[i].ref - m) * kLog2e);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
        if (lane == 0) row_lse = sum > 0.0 && sum < INFINITY && m < INFINITY ? (double)m + log(sum) : -INFINITY;
    }
    const int n = block_largest<16>(e, c.beams, lists, found);
    if (t >= c.beams) return;
    if (t < n && row_lse > -INFINITY) {
        const int at = 0xffff - (int)(found[t] & 0xffffu);
        put(t, score + ((double)key_value((int)(found[t] >> 16) - 32768) - row_lse), groups[at / kGroupLogits] * kGroupLogits + at % kGroupLogits);
    } else {
        put(t, -INFINITY, -1);
    }
}

// A group's beams, a lane per row of one wave: the largest of the rows' next candidates, `beams` times. Totals are compared as 64-bit
// numbers in their order, 0 for none: high words first, then the low words of those that are equal. The candidates come to LDS at once.
__device__ void select_merge(const SelectCall& c, const SelectScratch& k, int r0) {
    __shared__ uint64_t orders[kMaxBeams * kMaxBeams];
    __shared__ uint32_t tokens[kMaxBeams * kMaxBeams];
    for (int i = threadIdx.x; i < c.beams * c.beams; i += kBlock) {
        const uint64_t b = collect64(k.totals + (int64_t)r0 * c.beams + i);
        tokens[i] = __hip_atomic_load(k.places + (int64_t)r0 * c.beams + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // (a total below f32's range would be a score of -infinity)
        orders[i] = (float)__builtin_bit_cast(double, b) > -INFINITY ? (b >> 63 ? ~b : b | 1ull << 63) : 0;
    }
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    const int lane = threadIdx.x, row = c.row0 + r0 + lane;
    const bool in = lane < c.beams;
    int next = 0;
    uint64_t order = in ? orders[lane * c.beams] : 0;  // the row's next candidate
    const int done = in ? c.finished[row] != 0 : 0;
    int out_parent = row, out_token = max(c.eos, 0), out_done = 1;
    uint64_t out = 0;
    for (int i = 0; i < c.beams; ++i) {
        const uint32_t hi = wave_largest((uint32_t)(order >> 32));
        if (hi == 0) break;
        const bool top = (uint32_t)(order >> 32) == hi;
        const uint32_t lo = wave_largest(top ? (uint32_t)order : 0);
        const int who = __builtin_ctzll(__ballot(top && (uint32_t)order == lo));  // the lowest row of equals
        const int token = (int)tokens[who * c.beams + __builtin_amdgcn_readlane(next, who)], was = __builtin_amdgcn_readlane(done, who);
        if (lane == i) {
            out = (uint64_t)hi << 32 | lo;
            out_parent = c.row0 + r0 + who;
            out_token = token;
            out_done = was || token == c.eos;
        }
        if (lane == who) order = ++next < c.beams ? orders[lane * c.beams + next] : 0;
    }
    if (!in) return;
    const double total = __builtin_bit_cast(double, out >> 63 ? out & ~(1ull << 63) : ~out);
    c.out_scores[row] = out ? (float)total : -INFINITY;
    c.parents[row] = out_parent;
    c.tokens[row] = out_token;
    c.out_finished[row] = out_done;
}

// A workgroup per row; the last of a group picks its beams. Latency bounds it (keys, logits of the groups found, arrival, candidates: 10.3 us for
// one group of 4, 12.6 for 20 of 8); one row of a group after the other in one workgroup would take its steps in turn.
template <int kKeys>
__global__ __launch_bounds__(kBlock) void select_rows_kernel(SelectCall c, SelectScratch k) {
    const int r = blockIdx.x, g = r / c.beams;
    select_row<kKeys>(c, k, r);
    if (!arrive_last<kGroupTurn>(k.tickets + (int64_t)g * kTicketStride, r == g * c.beams, c.beams)) return;
    select_merge(c, k, g * c.beams);
}

int check_logits(const uint16_t* logits, int64_t stride, int rows, int vocab) {
    int e;
    if ((e = check_ptr(logits, "logits", 2))) return e;
    if (rows > 1 && (stride < vocab || stride > (int64_t(1) << 40)))
        return bad_value("logit_row_stride must be at least vocab, got " + std::to_string(stride));
    return MOA_SUCCESS;
}

// Loads of a thread: four where two workgroups a CU are left then, else two, for more workgroups. (Selection of 20 groups of 8 beams of 262144, us a
// call: 29.7 with four, 31.0 with two, 31.3 with eight; of one group of 4: 13.5 with two, 15.5 with eight.)
int loads_of(int64_t rows, int vocab, int cus) { return rows * parts_of(vocab, 4) >= 2 * (int64_t)cus ? 4 : 2; }

static_assert(kMaxParts < (int)kRowTurn && kTreeMaxNodes < (int)kRowTurn && kTreeMaxNodes < kSearchRows && kMaxBeams < (int)kGroupTurn, "arrivals are fewer than a turn");
constexpr size_t kSearchBytes = kPagedChunkFloats * sizeof(float);

}  // namespace
}  // namespace moa

using namespace moa;

extern "C" {

int moa_tree_verify(const uint16_t* logits, int64_t logit_row_stride, const int32_t* tokens, const int32_t* row_starts,
                    const uint64_t* masks, int mask_words, int32_t* best, int32_t* leaves, int32_t* next_tokens, int rows,
                    int vocab, int sequences, void* stream) {
    int e;
    if ((e = check_range(rows, 0, 65535, "rows")) || (e = check_range(vocab, 1, kSearchMaxVocab, "vocab")) ||
        (e = check_range(sequences, 1, kPagedMaxSequences, "sequences")) || (e = check_range(mask_words, 1, kTreeMaxWords, "mask_words")) ||
        (e = check_ptr(row_starts, "row_starts", 4)) || (e = check_ptr(leaves, "leaves", 4)) || (e = check_ptr(next_tokens, "next_tokens", 4)))
        return e;
    if (rows && ((e = check_logits(logits, logit_row_stride, rows, vocab)) || (e = check_ptr(tokens, "tokens", 4)) ||
                 (e = check_ptr(masks, "masks", 8)) || (e = check_ptr(best, "best", 4))))
        return e;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const VerifyCall c{logits, logit_row_stride, tokens, row_starts, masks, best, leaves, next_tokens, mask_words, rows, vocab, sequences, ctx->err};
    uint64_t* part = reinterpret_cast<uint64_t*>(ctx->paged_chunks);
    if (rows && rows <= kTreeMaxNodes && sequences <= kFewSequences) {
        const int parts = parts_of(vocab, 2);
        hipLaunchKernelGGL(mask_words == 1 ? verify_few_kernel<1> : verify_few_kernel<kTreeMaxWords>, dim3(parts, rows), dim3(kBlock), 0, s, c, part, reinterpret_cast<uint32_t*>(part + (size_t)rows * parts),
                           ctx->search_tickets + (size_t)kSearchRows * kTicketStride);
        return call_result(hipGetLastError(), "tree_verify launch");
    }
    const int loads = loads_of(rows, vocab, ctx->cus), parts = parts_of(vocab, loads);
    if (rows) {
        auto* f = loads == 4 ? verify_scan_kernel<4> : verify_scan_kernel<2>;
        hipLaunchKernelGGL(f, dim3(parts, rows), dim3(kBlock), 0, s, c, part);
        if ((e = call_result(hipGetLastError(), "tree_verify launch"))) return e;
    }
    hipLaunchKernelGGL(mask_words == 1 ? verify_walk_kernel<1> : verify_walk_kernel<kTreeMaxWords>, dim3(sequences), dim3(kBlock), 0, s, c, part, parts);
    return call_result(hipGetLastError(), "tree_verify launch");
}

int moa_beam_select(const uint16_t* logits, int64_t logit_row_stride, const float* scores, const int32_t* finished,
                    float* out_scores, int32_t* out_finished, int32_t* parents, int32_t* tokens, int groups, int beams,
                    int vocab, int eos, void* stream) {
    int e;
    if ((e = check_range(beams, 1, kMaxBeams, "beams")) || (e = check_range(groups, 0, 65535 / beams, "groups")) ||
        (e = check_range(vocab, 1, kSearchMaxVocab, "vocab")) || (e = check_range(eos, -1, vocab - 1, "eos")))
        return e;
    if (groups == 0) return MOA_SUCCESS;
    const int rows = groups * beams;
    if ((e = check_logits(logits, logit_row_stride, rows, vocab)) || (e = check_ptr(scores, "scores", 4)) ||
        (e = check_ptr(finished, "finished", 4)) || (e = check_ptr(out_scores, "out_scores", 4)) ||
        (e = check_ptr(out_finished, "out_finished", 4)) || (e = check_ptr(parents, "parents", 4)) || (e = check_ptr(tokens, "tokens", 4)))
        return e;
    DevCtx* ctx = paged_context(&e);
    if (!ctx) return e;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int loads = loads_of(rows, vocab, ctx->cus);
    SelectScratch k;
    k.groups = (vocab + kGroupLogits - 1) / kGroupLogits;
    k.key_stride = (k.groups + 3) / 4 * 4;
    k.parts_n = parts_of(vocab, loads);
    // the groups of rows that the scratch and its counters hold at once
    const size_t row_bytes = (size_t)beams * 12 + (size_t)k.parts_n * sizeof(PartSum) + (size_t)k.key_stride * 2;
    const int most = (int)std::min<size_t>(groups, std::min<size_t>(kSearchBytes / (row_bytes * beams), kSearchRows / beams));
    uint8_t* at = reinterpret_cast<uint8_t*>(ctx->paged_chunks);
    const size_t held = (size_t)most * beams;
    k.totals = reinterpret_cast<uint64_t*>(at);
    k.parts = reinterpret_cast<PartSum*>(at + held * beams * 8);
    k.keys = reinterpret_cast<uint16_t*>(at + held * (beams * 8 + k.parts_n * sizeof(PartSum)));
    k.places = reinterpret_cast<uint32_t*>(at + held * (beams * 8 + k.parts_n * sizeof(PartSum) + k.key_stride * 2));
    k.tickets = ctx->search_tickets;
    auto* scan = loads == 4 ? select_scan_kernel<4> : select_scan_kernel<2>;
    auto* pick = k.groups > 16 * kBlock ? select_rows_kernel<64> : select_rows_kernel<16>;
    for (int g = 0; g < groups; g += most) {
        const int here = std::min(most, groups - g);
        const SelectCall c{logits, logit_row_stride, scores, finished, out_scores, out_finished, parents, tokens, beams, vocab, eos, g * beams};
        hipLaunchKernelGGL(scan, dim3(k.parts_n, here * beams), dim3(kBlock), 0, s, c, k);
        hipLaunchKernelGGL(pick, dim3(here * beams), dim3(kBlock), 0, s, c, k);
        if ((e = call_result(hipGetLastError(), "beam_select launch"))) return e;
    }
    return MOA_SUCCESS;
}

}  // extern "C"
