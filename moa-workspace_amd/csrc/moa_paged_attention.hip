// moa_paged_attention.hip -- attention of new rows over the paged cache (include/moa_paged.h).
//
// Row i of a sequence's n new rows stands at p = len - n + i and sees positions max(0, p - window + 1) .. p. With
// x_t = scale (q . k_t) it gives sum_t e^(x_t - m) v_t / sum_t e^(x_t - m), m the largest x_t, in one pass over the
// positions with a running m and sum. E4M3 pages: k_t and v_t are codes times the head's scale; K's joins the
// factor of x_t, V's the last division.
#include "moa_device.h"
#include "moa_paged.h"

namespace moa {
namespace {

constexpr int kMaxDim = 512;

// One row (m, head h) by one wave, any type and shape: 64 positions at a time, a lane each for the scores; then the lanes
// hold head_dim / 64 dims each and take the 64 weights in turn. Positions outside the row's range are never used.
template <bool E4M3>
__global__ __launch_bounds__(256) void paged_attention_row_kernel(PagedView c, PagedAttentionCall a) {
    __shared__ float qs[4][kMaxDim];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
    const int m = (int)(unit / a.q_heads), h = (int)(unit - (int64_t)m * a.q_heads), kvh = h / a.group;
    if (m >= a.rows) return;
    const int s = sequence_of(a.starts, c.sequences, m);
    if (s < 0 || s >= c.sequences) return;
    const int start = a.starts[s], end = a.starts[s + 1], len = c.lens[s];
    if (end <= m) return;
    if (start < 0 || end > a.rows || end - start > a.max_rows || len < 0 || len > paged_capacity(c)) {
        if (lane == 0) atomicOr(c.err, kErrPaged);
        return;
    }
    const int p = len - (end - m), lo = a.window && p >= a.window ? p - a.window + 1 : 0;
    const int d = c.head_dim;
    for (int i = lane; i < d; i += 64) qs[wave][i] = bf2f(a.q[m * a.q_row + h * d + i]);
    const float ks = E4M3 ? c.k_scale[kvh] * a.scale_log2 : a.scale_log2;
    const int per = d / 64;
    float o[kMaxDim / 64] = {}, mx = -INFINITY, sum = 0.0f;
    bool bad = false;
    for (int t0 = lo; t0 <= p; t0 += 64) {
        const int t = t0 + lane;
        int page = 0, slot = 0;
        float x = -INFINITY;
        if (t <= p) {
            const uint32_t i = page_of(c, t);
            slot = t - i * c.slots;
            page = c.table[s * c.table_stride + i];
            if (page < 0 || page >= c.pages) bad = true;
            else {
                const uint8_t* kp = c.k + page * c.k_page + slot * c.k_slot + kvh * c.k_head;
                float acc = 0.0f;
                for (int j = 0; j < d; j += 8) {
                    float e[8];
                    if (E4M3) {
                        const uint2 w = *reinterpret_cast<const uint2*>(kp + j);
                        fp8x4_to_f32(w.x, e);
                        fp8x4_to_f32(w.y, e + 4);
                    } else {
                        bf16x8_to_f32(ld16(kp + 2 * j), e);
                    }
#pragma unroll
                    for (int i2 = 0; i2 < 8; ++i2) acc = fmaf(e[i2], qs[wave][j + i2], acc);
                }
                x = acc * ks;
            }
        }
        if (__any(bad)) break;
        float mn = x;
#pragma unroll
        for (int o2 = 32; o2 > 0; o2 >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o2, kWave));
        mn = fmaxf(mn, mx);
        const float f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mn);
        const float w = t <= p && mn != -INFINITY ? __builtin_amdgcn_exp2f(x - mn) : 0.0f;
        mx = mn;
        sum = fmaf(sum, f, wave_sum(w));
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) o[i] *= f;
        const int n = min(64, p - t0 + 1);
        for (int j = 0; j < n; ++j) {
            const float wj = __shfl(w, j, kWave);
            const uint8_t* vp = c.v + __shfl(page, j, kWave) * c.v_page + __shfl(slot, j, kWave) * c.v_slot + kvh * c.v_head;
#pragma unroll
            for (int i = 0; i < kMaxDim / 64; ++i)
                if (i < per)
                    o[i] = fmaf(wj, E4M3 ? e4m3_to_f32(vp[lane * per + i]) : bf2f(reinterpret_cast<const uint16_t*>(vp)[lane * per + i]), o[i]);
        }
    }
    if (__any(bad)) {
        if (lane == 0) atomicOr(c.err, kErrPaged);
        return;
    }
    const float vs = E4M3 ? c.v_scale[kvh] : 1.0f;
    const float inv = sum == 0.0f ? 0.0f : vs / sum;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i)
        if (i < per) a.out[m * a.out_row + h * d + lane * per + i] = (uint16_t)f2bf(o[i] * inv);
}

}  // namespace

hipError_t launch_paged_attention(const PagedView& c, const PagedAttentionCall& a, hipStream_t s, DevCtx*) {
    const int64_t units = (int64_t)a.rows * a.q_heads;
    auto* f = c.k_scale ? paged_attention_row_kernel<true> : paged_attention_row_kernel<false>;
    hipLaunchKernelGGL(f, dim3((uint32_t)((units + 3) / 4)), dim3(256), 0, s, c, a);
    return hipGetLastError();
}

}  // namespace moa
