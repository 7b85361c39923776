// moa_search.hip -- tokens from logits (include/moa_search.h): the greedy verification of drafted trees, and the selection of
// beams. Both read every row of bf16 logits once; what is left of a row then fits a workgroup.
#include <algorithm>

#include "../../include/moa_search.h"
#include "moa_checks.h"
#include "moa_device.h"
#include "moa_paged_plan.h"

namespace moa {
namespace {

constexpr int kBlock = 256;
constexpr int kGroupLogits = 64;        // logits that share a key (their largest): 8 lanes' 16 bytes
constexpr int kSearchMaxVocab = 1 << 20;
constexpr int kMaxGroups = kSearchMaxVocab / kGroupLogits;

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

// A row's parts: 256 threads of kLoads chunks each.
__host__ __device__ inline int parts_of(int vocab, int loads) { return (vocab + kBlock * 8 * loads - 1) / (kBlock * 8 * loads); }

// ---------------------------------------------------------------------------------------------- verify

// The largest logit of a part of a row and its first place, as one number that orders by both.
template <int kLoads>
__global__ __launch_bounds__(kBlock) void verify_scan_kernel(const uint16_t* logits, int64_t stride, int vocab, uint64_t* best) {
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
    if (threadIdx.x == 0)
        best[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = (uint64_t)(uint32_t)(most + 32768) << 32 | ~min(min(at[0], at[1]), min(at[2], at[3]));
}

// One workgroup per sequence: its rows' parts into tokens, then the walk by one wave, four nodes a lane.
__global__ __launch_bounds__(kBlock) void verify_walk_kernel(const uint64_t* part, int parts, const int32_t* tokens, const int32_t* starts,
                                                             const uint64_t* masks, int words, int32_t* best, int32_t* leaves,
                                                             int32_t* next, int rows, uint32_t* err) {
    __shared__ int32_t named[kTreeMaxNodes];
    const int s = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const int row0 = starts[s], end = starts[s + 1];
    const bool out = !rows_in_range(row0, end, rows, 64 * words);
    if (out || row0 == end) {
        if (t == 0) {
            leaves[s] = next[s] = -1;
            if (out && row0 != end) atomicOr(err, kErrPaged);
        }
        return;
    }
    const int n = end - row0;
    int lanes = 1;  // that share a row
    while (lanes < 64 && lanes < parts) lanes *= 2;
    for (int r = t / lanes; r < n; r += kBlock / lanes) {
        uint64_t key = 0;
        for (int i = t % lanes; i < parts; i += lanes) key = max(key, part[(int64_t)(row0 + r) * parts + i]);
        for (int o = lanes / 2; o > 0; o >>= 1) key = max(key, (uint64_t)__shfl_xor((long long)key, o, kWave));
        if (t % lanes == 0) best[row0 + r] = named[r] = (int32_t) ~(uint32_t)key;
    }
    __syncthreads();
    if (t >= 64) return;
    uint64_t mask[4][kTreeMaxWords];
    int32_t token[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = 64 * k + lane;
        token[k] = i < n ? tokens[row0 + i] : 0;
#pragma unroll
        for (int w = 0; w < kTreeMaxWords; ++w) {
            const int left = n - 64 * w;
            mask[k][w] = i < n && w < words && left > 0 ? masks[(int64_t)(row0 + i) * words + w] & (left >= 64 ? ~0ull : (1ull << left) - 1) : 0;
        }
    }
    auto of = [&](uint64_t v, int l) {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, l) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32;
    };
    if (!(of(mask[0][0], 0) & 1)) {  // node 0 is none
        if (lane == 0) leaves[s] = next[s] = -1;
        return;
    }
    int cur = 0;
    for (int step = 0; step < n; ++step) {
        const int want = named[cur];
        uint64_t sees[kTreeMaxWords];
#pragma unroll
        for (int w = 0; w < kTreeMaxWords; ++w) {
            const uint64_t x = cur < 64 ? mask[0][w] : cur < 128 ? mask[1][w] : cur < 192 ? mask[2][w] : mask[3][w];
            sees[w] = of(x, cur & 63);
        }
        int child = -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            bool is = token[k] == want && (mask[k][k] >> lane & 1) && 64 * k + lane < n && !(sees[k] >> lane & 1);
#pragma unroll
            for (int w = 0; w < kTreeMaxWords; ++w) is = is && (mask[k][w] & ~(w == k ? 1ull << lane : 0ull)) == sees[w];
            const uint64_t hit = __ballot(is);
            if (child < 0 && hit) child = 64 * k + __builtin_ctzll(hit);
        }
        if (child < 0) break;
        cur = child;
    }
    if (lane == 0) leaves[s] = cur, next[s] = named[cur];
}

// ---------------------------------------------------------------------------------------------- select

// What a selection keeps of each row: the keys of its groups of logits, its parts' maxima and sums, and its candidates.
struct SelectScratch {
    uint16_t* keys;      // [rows][groups]: the largest logit of a group, ordered() + 32768
    float2* parts;       // [rows][parts]: largest logit, sum of e^(logit - largest)
    double* totals;      // [rows][beams], descending
    int32_t* places;     // [rows][beams]
    int groups, parts_n; // of a row
};

struct SelectCall {
    const uint16_t* logits; int64_t stride;
    const float* scores; const int32_t* finished;
    float* out_scores; int32_t* out_finished; int32_t* parents; int32_t* tokens;
    int beams, vocab, eos, row0;  // first row of this launch
};

constexpr float kLog2e = 1.4426950408889634f;

// A beam that adds candidates from its logits.
__device__ __forceinline__ bool grows(const SelectCall& c, int row) { return c.finished[row] == 0 && c.scores[row] > -INFINITY; }

// One pass over a part of a row: the keys of its groups, and its largest logit and sum.
template <int kLoads>
__global__ __launch_bounds__(kBlock) void select_scan_kernel(SelectCall c, SelectScratch k) {
    __shared__ float top[4], sums[4];
    if (!grows(c, c.row0 + blockIdx.y)) return;
    const LogitRow row(c.logits, c.stride, c.row0 + (int)blockIdx.y, c.vocab);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = blockIdx.x * kBlock * kLoads + threadIdx.x;
    uint4 w[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) w[j] = row.chunk(first + j * kBlock, kMinusInfinity);
    int most = -32768;
    uint16_t* keys = k.keys + (int64_t)blockIdx.y * k.groups;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const s16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(ordered(w[j].x), ordered(w[j].y)),
                                                  __builtin_elementwise_max(ordered(w[j].z), ordered(w[j].w)));
        int g = larger(m);
        most = max(most, g);
#pragma unroll
        for (int o = 1; o < 8; o *= 2) g = max(g, __shfl_xor(g, o, kWave));
        const int at = (first + j * kBlock) / 8;
        if ((lane & 7) == 0 && at < k.groups) keys[at] = (uint16_t)(g + 32768);
    }
    const float m = most >= kLowestFinite ? key_value(most) : -INFINITY, ref = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        float x[8];
        bf16x8_to_f32(w[j], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * kLog2e);
    }
    float all = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, kWave));
    sum = wave_sum(m == -INFINITY ? sum : sum * __builtin_amdgcn_exp2f((m - all) * kLog2e));  // (a NaN in a lane without a finite logit stays)
    if (lane == 0) top[wave] = all, sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    const float part = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) total += top[i] == -INFINITY ? sums[i] : sums[i] * __builtin_amdgcn_exp2f((top[i] - part) * kLog2e);
    k.parts[(int64_t)blockIdx.y * k.parts_n + blockIdx.x] = make_float2(part, total);
}

// The sum of v over the workgroup, in every thread. lds: 4 numbers that no earlier call may still read.
template <class T>
__device__ T block_total(T v, T* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// The positions of the `want` largest of n keys in LDS that are at least `least`, ties to the lowest position, in any order;
// returns how many there are. The smallest of them is found by halving the range of keys.
__device__ int largest_keys(const uint16_t* keys, int n, int want, int least, int* out, int* lds) {
    const int t = threadIdx.x, per = (n + kBlock - 1) / kBlock, from = min(t * per, n), to = min(from + per, n);
    auto count = [&](int least) {
        int c = 0;
        for (int i = from; i < to; ++i) c += keys[i] >= least;
        return block_total(c, lds);
    };
    int lo = least, hi = 65536;  // at least `want` keys are lo or more (or lo is `least`); fewer are hi or more
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (count(mid) >= want) lo = mid;
        else hi = mid;
    }
    int above = 0, equal = 0;
    for (int i = from; i < to; ++i) above += keys[i] > lo, equal += keys[i] == lo;
    // both prefix sums at once: neither passes 2^16
    int x = above << 16 | equal, before = 0;
    const int mine = x, lane = t & 63, wave = t >> 6;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(x, o, kWave);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    for (int i = 0; i < wave; ++i) before += lds[i];
    const int total = lds[0] + lds[1] + lds[2] + lds[3], tops = total >> 16;
    before += x - mine;
    int a = before >> 16, e = tops + (before & 0xffff);
    for (int i = from; i < to; ++i) {
        if (keys[i] > lo) out[a++] = i;
        else if (keys[i] == lo) {
            if (e < want) out[e] = i;
            ++e;
        }
    }
    __syncthreads();
    return min(want, tops + (total & 0xffff));
}

// One workgroup per row: its sum, the groups that hold its `beams` largest logits (of the groups that come first by key and place,
// since each holds a logit that comes before all of a later group), those logits, and their totals in descending order.
__global__ __launch_bounds__(kBlock) void select_row_kernel(SelectCall c, SelectScratch k) {
    __shared__ uint16_t keys[kMaxGroups > kMaxBeams * kGroupLogits ? kMaxGroups : kMaxBeams * kGroupLogits];
    __shared__ int groups[kMaxBeams], chosen[kMaxBeams], lds[4];
    __shared__ double sums[4];
    __shared__ float top[4];
    const int r = blockIdx.x, row = c.row0 + r, t = threadIdx.x, lane = t & 63;
    double* totals = k.totals + (int64_t)r * c.beams;
    int32_t* places = k.places + (int64_t)r * c.beams;
    const double score = c.scores[row];
    if (!grows(c, row)) {
        if (t < c.beams) {
            totals[t] = t == 0 && c.eos >= 0 && score > -INFINITY ? score : -INFINITY;
            places[t] = c.eos;
        }
        return;
    }
    float m = -INFINITY;
    for (int i = t; i < k.parts_n; i += kBlock) m = fmaxf(m, k.parts[(int64_t)r * k.parts_n + i].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
    if (lane == 0) top[t >> 6] = m;
    for (int i = t; i < k.groups; i += kBlock) keys[i] = k.keys[(int64_t)r * k.groups + i];
    __syncthreads();
    m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    double sum = 0.0;
    for (int i = t; i < k.parts_n; i += kBlock) {
        const float2 p = k.parts[(int64_t)r * k.parts_n + i];
        sum += p.x == -INFINITY ? (double)p.y : (double)p.y * exp((double)p.x - (double)m);
    }
    sum = block_total(sum, sums);
    const bool alive = sum > 0.0 && sum < INFINITY && m < INFINITY;
    const double lse = (double)m + log(sum);
    constexpr int kLeast = kLowestFinite + 32768;
    const int ng = alive ? largest_keys(keys, k.groups, c.beams, kLeast, groups, lds) : 0;
    // their logits, groups in ascending order
    const LogitRow logits(c.logits, c.stride, row, c.vocab);
    __syncthreads();
    if (t < 64) {
        const int g = lane < ng ? groups[lane] : 0x7fffffff;
        int rank = 0;
        for (int i = 0; i < ng; ++i) rank += __shfl(g, i, kWave) < g;
        if (lane < ng) chosen[rank] = g;
    }
    __syncthreads();
    for (int i = t; i < ng * 8; i += kBlock) {
        const uint4 w = logits.chunk(chosen[i / 8] * 8 + i % 8, kMinusInfinity);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const s16x2 o = ordered(v[j]);
            keys[8 * i + 2 * j] = (uint16_t)(o[0] + 32768), keys[8 * i + 2 * j + 1] = (uint16_t)(o[1] + 32768);
        }
    }
    __syncthreads();
    const int n = ng ? largest_keys(keys, ng * kGroupLogits, c.beams, kLeast, groups, lds) : 0;
    if (t >= 64) return;
    int key = 0, at = 0x7fffffff;
    if (lane < n) key = keys[groups[lane]], at = groups[lane];
    int rank = 0;
    for (int i = 0; i < n; ++i) {
        const int y = __shfl(key, i, kWave), z = __shfl(at, i, kWave);
        rank += y > key || (y == key && z < at);
    }
    if (lane < n) {
        totals[rank] = score + ((double)key_value(key - 32768) - lse);
        places[rank] = chosen[at / kGroupLogits] * kGroupLogits + at % kGroupLogits;
    } else if (lane < c.beams) {
        totals[lane] = -INFINITY;
        places[lane] = -1;
    }
}

// One wave per group, a lane per row: the largest of the rows' next candidates, `beams` times.
__global__ __launch_bounds__(kWave) void select_merge_kernel(SelectCall c, SelectScratch k) {
    const int lane = threadIdx.x, r0 = blockIdx.x * c.beams, row = c.row0 + r0 + lane;
    const double* totals = k.totals + (int64_t)(r0 + lane) * c.beams;
    const int32_t* places = k.places + (int64_t)(r0 + lane) * c.beams;
    const bool in = lane < c.beams;
    int next = 0, place = in ? places[0] : 0, out_parent = row, out_token = max(c.eos, 0);
    double total = in ? totals[0] : -INFINITY, out_total = -INFINITY;
    if (total != total) total = -INFINITY;
    const int done = in ? c.finished[row] != 0 : 0;
    int out_done = 1;
    for (int i = 0; i < c.beams; ++i) {
        double best = total;
        int who = lane;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double y = __shfl_xor(best, o, kWave);
            const int z = __shfl_xor(who, o, kWave);
            if (y > best || (y == best && z < who)) best = y, who = z;
        }
        if (best == -INFINITY) break;
        const int token = __shfl(place, who, kWave), was = __shfl(done, who, kWave);
        if (lane == i) {
            out_total = best;
            out_parent = c.row0 + r0 + who;
            out_token = token;
            out_done = was || token == c.eos;
        }
        if (lane == who) {
            ++next;
            total = next < c.beams ? totals[next] : -INFINITY;
            place = next < c.beams ? places[next] : 0;
            if (total != total) total = -INFINITY;
        }
    }
    if (!in) return;
    c.out_scores[row] = (float)out_total;
    c.parents[row] = out_parent;
    c.tokens[row] = out_token;
    c.out_finished[row] = out_done;
}

int check_logits(const uint16_t* logits, int64_t stride, int rows, int vocab) {
    int e;
    if ((e = check_ptr(logits, "logits", 2))) return e;
    if (rows > 1 && (stride < vocab || stride > (int64_t(1) << 40)))
        return bad_value("logit_row_stride must be at least vocab, got " + std::to_string(stride));
    return MOA_SUCCESS;
}

// Loads of a thread: eight where two workgroups a CU are left then, else two, for more workgroups.
int loads_of(int64_t rows, int vocab, int cus) { return rows * parts_of(vocab, 8) >= 2 * (int64_t)cus ? 8 : 2; }

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
    const int loads = loads_of(rows, vocab, ctx->cus), parts = parts_of(vocab, loads);
    uint64_t* part = reinterpret_cast<uint64_t*>(ctx->paged_chunks);
    if (rows) {
        auto* f = loads == 8 ? verify_scan_kernel<8> : verify_scan_kernel<2>;
        hipLaunchKernelGGL(f, dim3(parts, rows), dim3(kBlock), 0, s, logits, logit_row_stride, vocab, part);
        if ((e = call_result(hipGetLastError(), "tree_verify launch"))) return e;
    }
    hipLaunchKernelGGL(verify_walk_kernel, dim3(sequences), dim3(kBlock), 0, s, part, parts, tokens, row_starts, masks, mask_words, best,
                       leaves, next_tokens, rows, ctx->err);
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
    k.parts_n = parts_of(vocab, loads);
    // the groups of rows that the scratch holds at once (all but always: it holds 2000 rows of the largest vocabulary)
    const size_t row_bytes = (size_t)beams * 12 + (size_t)k.parts_n * 8 + (size_t)k.groups * 2;
    const int most = (int)std::min<size_t>(groups, kSearchBytes / (row_bytes * beams));
    uint8_t* at = reinterpret_cast<uint8_t*>(ctx->paged_chunks);
    const size_t held = (size_t)most * beams;
    k.totals = reinterpret_cast<double*>(at);
    k.parts = reinterpret_cast<float2*>(at + held * beams * 8);
    k.places = reinterpret_cast<int32_t*>(at + held * (beams * 8 + k.parts_n * 8));
    k.keys = reinterpret_cast<uint16_t*>(at + held * (beams * 12 + k.parts_n * 8));
    for (int g = 0; g < groups; g += most) {
        const int here = std::min(most, groups - g), n = here * beams;
        const SelectCall c{logits, logit_row_stride, scores, finished, out_scores, out_finished, parents, tokens, beams, vocab, eos, g * beams};
        auto* f = loads == 8 ? select_scan_kernel<8> : select_scan_kernel<2>;
        hipLaunchKernelGGL(f, dim3(k.parts_n, n), dim3(kBlock), 0, s, c, k);
        hipLaunchKernelGGL(select_row_kernel, dim3(n), dim3(kBlock), 0, s, c, k);
        hipLaunchKernelGGL(select_merge_kernel, dim3(here), dim3(kWave), 0, s, c, k);
        if ((e = call_result(hipGetLastError(), "beam_select launch"))) return e;
    }
    return MOA_SUCCESS;
}

}  // extern "C"
