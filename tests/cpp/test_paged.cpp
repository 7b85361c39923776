// test_paged.cpp -- the paged KV cache over the C++ host interface (moa-workspace_amd/host/moa_ops.hpp).
//
// TEST INFRASTRUCTURE. A run of the calls as a host program makes them: three sequences are given prompts (reserve,
// append, attention), one of them is forked, all take single tokens, one ends and the pool is compacted, with the
// attention of every step and layer checked against a plain evaluation in double from the host's own copy of every
// sequence's rows, and the lengths and reference counts against a plain count. E4M3 pages hold values that are codes times
// the scale exactly, so one check serves both types. At last, calls with tensors of the wrong shape throw.
//
//   test_paged            on device 0
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "moa_ops.hpp"

using moa::bf16;
using moa::Device;
using moa::HbmTensor;

namespace {

constexpr size_t kLayers = 2, kPages = 40, kSlots = 16, kHeads = 2, kGroup = 3, kDim = 64, kSeqs = 5, kColumns = 12;
constexpr size_t kKv = kHeads * kDim, kQ = kHeads * kGroup * kDim;
constexpr float kScale = 0.125f, kPageScale = 0.25f;

uint32_t state = 12345;
uint32_t next_random() { return state = state * 1664525u + 1013904223u; }
// sixteenths up to 1.5: bf16 values that are E4M3 codes times kPageScale (at most three significant bits)
float value() {
    static const float v[8] = {0.0625f, 0.125f, 0.1875f, 0.25f, 0.375f, 0.5f, 0.75f, 1.5f};
    const uint32_t r = next_random() >> 20;
    return r & 8 ? -v[r & 7] : v[r & 7];
}
bf16 to_bf16(float f) {  // exact here
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return bf16{static_cast<uint16_t>(u >> 16)};
}
float to_f32(bf16 b) {
    const uint32_t u = static_cast<uint32_t>(b.bits) << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}
std::vector<float> values(size_t n) {
    std::vector<float> v(n);
    for (float& x : v) x = value();
    return v;
}
HbmTensor<bf16> upload(const Device& d, const std::vector<float>& v, std::vector<size_t> shape) {
    std::vector<bf16> b(v.size());
    std::transform(v.begin(), v.end(), b.begin(), to_bf16);
    return HbmTensor<bf16>::from_host(d, b, std::move(shape));
}
HbmTensor<int32_t> ints(const Device& d, const std::vector<int32_t>& v) { return HbmTensor<int32_t>::from_host(d, v, {v.size()}); }

template <class T>
struct Run {
    const Device& d;
    HbmTensor<T> k, v;
    HbmTensor<int32_t> table, lens, refs;
    HbmTensor<float> scale;
    moa::PagedCache<T> cache;
    std::vector<float> kept[kSeqs][kLayers][2];  // K and V rows of every sequence
    int failed = 0;

    explicit Run(const Device& dev)
        : d(dev), k(dev, {kLayers, kPages, kSlots, kHeads, kDim}), v(dev, {kLayers, kPages, kSlots, kHeads, kDim}),
          table(dev, {kSeqs, kColumns}), lens(dev, {kSeqs}), refs(dev, {kPages}),
          scale(HbmTensor<float>::from_host(dev, std::vector<float>(kLayers * kHeads, kPageScale), {kLayers, kHeads})),
          cache(k, v, table, lens, refs, std::is_same<T, bf16>::value ? nullptr : &scale, std::is_same<T, bf16>::value ? nullptr : &scale) {}

    size_t length(size_t s) const { return kept[s][0][0].size() / kKv; }

    // fresh[s] new rows for every sequence: reserve, then append and attend in both layers
    void step(const char* name, const std::vector<int32_t>& fresh, int window) {
        std::vector<int32_t> starts{0};
        int most = 1;
        for (int32_t n : fresh) {
            starts.push_back(starts.back() + n);
            most = std::max(most, n);
        }
        const size_t rows = static_cast<size_t>(starts.back());
        const auto dn = ints(d, fresh), ds = ints(d, starts);
        moa::ops::paged_cache_reserve(d, cache, dn);
        double worst = 0.0;
        for (size_t layer = 0; layer < kLayers; ++layer) {
            const auto hk = values(rows * kKv), hv = values(rows * kKv), hq = values(rows * kQ);
            for (size_t s = 0; s < kSeqs; ++s)
                for (int which = 0; which < 2; ++which) {
                    const auto& from = which ? hv : hk;
                    kept[s][layer][which].insert(kept[s][layer][which].end(), from.begin() + starts[s] * kKv, from.begin() + starts[s + 1] * kKv);
                }
            const auto dk = upload(d, hk, {rows, kHeads, kDim}), dv = upload(d, hv, {rows, kHeads, kDim});
            const auto dq = upload(d, hq, {rows, kHeads * kGroup, kDim});
            HbmTensor<bf16> out(d, {rows, kHeads * kGroup, kDim});
            moa::ops::paged_cache_append(d, cache, dk, dv, ds, static_cast<int>(layer));
            moa::ops::paged_attention(d, dq, cache, ds, out, static_cast<int>(layer), window, kScale, most);
            worst = std::max(worst, check(out.to_host(d), hq, starts, layer, window));
        }
        std::vector<int32_t> want;
        for (size_t s = 0; s < kSeqs; ++s) want.push_back(static_cast<int32_t>(length(s)));
        report(name, worst <= 1.0 && lens.to_host(d) == want, worst);
    }

    // The largest error over its bound: bf16 weights move a result by at most 2^-8 of the attention of |v|, the
    // rounding to bf16 by 2^-8 of it; exact values, so the scores' and sums' f32 roundings stay below 2^-14 of it.
    double check(const std::vector<bf16>& out, const std::vector<float>& q, const std::vector<int32_t>& starts, size_t layer, int window) const {
        double worst = 0.0;
        for (size_t s = 0; s < kSeqs; ++s) {
            const int n = starts[s + 1] - starts[s], len = static_cast<int>(length(s));
            const auto &ks = kept[s][layer][0], &vs = kept[s][layer][1];
            for (int i = 0; i < n; ++i)
                for (size_t h = 0; h < kHeads * kGroup; ++h) {
                    const int p = len - n + i, lo = window ? std::max(0, p - window + 1) : 0;
                    const size_t row = starts[s] + i, kvh = h / kGroup;
                    std::vector<double> x;
                    for (int t = lo; t <= p; ++t) {
                        double dot = 0.0;
                        for (size_t j = 0; j < kDim; ++j) dot += static_cast<double>(q[row * kQ + h * kDim + j]) * ks[t * kKv + kvh * kDim + j];
                        x.push_back(dot * kScale);
                    }
                    const double m = *std::max_element(x.begin(), x.end());
                    double sum = 0.0;
                    for (double& e : x) sum += e = std::exp(e - m);
                    for (size_t j = 0; j < kDim; ++j) {
                        double want = 0.0, spread = 0.0;
                        for (int t = lo; t <= p; ++t) {
                            const double y = x[t - lo] / sum * vs[t * kKv + kvh * kDim + j];
                            want += y;
                            spread += std::fabs(y);
                        }
                        const double got = to_f32(out[row * kQ + h * kDim + j]);
                        const double tol = std::ldexp(std::fabs(want), -8) + (1 + std::ldexp(1.0, -8)) * spread * (std::ldexp(1.0, -8) + std::ldexp(1.0, -14)) + 1e-30;
                        const double over = std::fabs(got - want) / tol;
                        worst = std::isfinite(got) ? std::max(worst, over) : 1e30;
                    }
                }
        }
        return worst;
    }

    void report(const char* name, bool ok, double worst) {
        std::printf("[%-12s %-30s] error %.3f of its bound -> %s\n", std::is_same<T, bf16>::value ? "bf16 pages" : "E4M3 pages", name, worst,
                    ok ? "PASS" : "FAIL");
        failed += ok ? 0 : 1;
    }

    // Reference counts: the table entries in use that name each page.
    void count(const char* name, bool compacted) {
        const auto t = table.to_host(d), n = lens.to_host(d), r = refs.to_host(d);
        std::vector<int32_t> want(kPages, 0);
        for (size_t s = 0; s < kSeqs; ++s)
            for (size_t i = 0; i < (n[s] + kSlots - 1) / kSlots; ++i) ++want[t[s * kColumns + i]];
        const auto live = static_cast<size_t>(std::count_if(want.begin(), want.end(), [](int32_t x) { return x > 0; }));
        const bool front = std::all_of(want.begin(), want.begin() + live, [](int32_t x) { return x > 0; });
        report(name, r == want && (!compacted || front), 0.0);
    }

    int all() {
        step("prompts", {35, 1, 0, 70, 0}, 0);
        count("counts", false);
        step("tokens", {1, 1, 0, 1, 0}, 0);
        const auto parents = ints(d, {3, 3}), children = ints(d, {2, 4});
        moa::ops::paged_cache_fork(d, cache, parents, children);
        for (int c : {2, 4})
            for (size_t l = 0; l < kLayers; ++l)
                for (int w = 0; w < 2; ++w) kept[c][l][w] = kept[3][l][w];
        count("counts after the fork", false);
        step("tokens of the copies", {1, 1, 1, 1, 2}, 0);
        const auto gone = ints(d, {0, 3, 3});
        moa::ops::paged_cache_free(d, cache, gone);
        for (int s : {0, 3})
            for (size_t l = 0; l < kLayers; ++l)
                for (int w = 0; w < 2; ++w) kept[s][l][w].clear();
        moa::ops::paged_cache_compact(d, cache);
        count("counts after the compaction", true);
        step("chunks in a window", {20, 17, 9, 0, 1}, 24);
        step("tokens in a window", {1, 1, 1, 0, 1}, 24);
        return failed;
    }
};

template <class F>
bool throws(const char* name, F&& f) {
    int code = 0;
    try {
        f();
    } catch (const moa::Error& e) {
        code = e.code();
    }
    std::printf("[refused: %-32s] code %d -> %s\n", name, code, code == MOA_ERROR_INVALID_VALUE ? "PASS" : "FAIL");
    return code == MOA_ERROR_INVALID_VALUE;
}

int refusals(const Device& d) {
    Run<bf16> r(d);
    const auto two = ints(d, {1, 1});
    const auto starts = ints(d, {0, 1, 1, 1, 1, 1});
    HbmTensor<bf16> q(d, {1, 6, kDim}), small(d, {1, 6, 32}), rows(d, {1, kHeads, kDim});
    HbmTensor<int32_t> flat(d, {kSeqs * kColumns});
    int failed = 0;
    failed += !throws("new_tokens of two", [&] { moa::ops::paged_cache_reserve(d, r.cache, two); });
    failed += !throws("row_starts of two", [&] { moa::ops::paged_cache_append(d, r.cache, rows, rows, two); });
    failed += !throws("a layer too many", [&] { moa::ops::paged_cache_append(d, r.cache, rows, rows, starts, 2); });
    failed += !throws("heads of 32 dims", [&] { moa::ops::paged_attention(d, small, r.cache, starts, small); });
    failed += !throws("more max_rows than rows", [&] { moa::ops::paged_attention(d, q, r.cache, starts, q, 0, 0, 1.0f, 2); });
    failed += !throws("children of another count", [&] { moa::ops::paged_cache_fork(d, r.cache, two, starts); });
    failed += !throws("a flat page table", [&] { moa::PagedCache<bf16> c(r.k, r.v, flat, r.lens, r.refs); });
    failed += !throws("scales with bf16 pages", [&] {
        moa::PagedCache<bf16> c(r.k, r.v, r.table, r.lens, r.refs, &r.scale, &r.scale);
        moa::ops::paged_cache_compact(d, c);
    });
    return failed;
}

}  // namespace

int main() {
    try {
        Device device(0);
        int failed = Run<bf16>(device).all() + Run<moa::f8e4m3>(device).all() + refusals(device);
        const uint32_t bits = device.device_errors();
        if (bits) {
            std::printf("device error bits 0x%x -> FAIL\n", bits);
            ++failed;
        }
        std::printf("%s: %d checks failed\n", failed ? "FAIL" : "PASS", failed);
        return failed ? 1 : 0;
    } catch (const moa::Error& e) {
        std::printf("FAIL: %s (code %d)\n", e.what(), e.code());
        return 1;
    }
}
