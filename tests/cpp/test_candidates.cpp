// test_candidates.cpp -- drafted trees and beams over the C++ host interface (moa-workspace_amd/host/moa_ops.hpp).
//
// TEST INFRASTRUCTURE. Two runs as a host program makes them, on bf16 and on E4M3 pages. Speculative: sequences get prompts, then
// trees of drafted tokens (reserve, append, attention of the nodes), their logits are verified and the paths committed; the next tokens'
// attention reads what the commit moved. Beams: two groups select their next tokens and take over their parents' sequences, then
// attend again. Every step's attention is checked in both layers against a plain evaluation in double from the host's own copy
// of every sequence's rows, the other results against plain counts. At last, calls with tensors of the wrong shape throw.
//
//   test_candidates       on device 0
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

constexpr size_t kLayers = 2, kPages = 40, kSlots = 16, kHeads = 2, kGroup = 3, kDim = 64, kSeqs = 4, kColumns = 12, kVocab = 301;
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

HbmTensor<uint64_t> words(const Device& d, const std::vector<uint64_t>& v) { return HbmTensor<uint64_t>::from_host(d, v, {v.size(), 1}); }

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

    // fresh[s] new rows of every sequence, which see the nodes of their masks: reserve, then append and attend in both layers.
    // Rows that see themselves and the earlier ones go through the tree's attention as well.
    void step(const char* name, const std::vector<int32_t>& fresh, const std::vector<uint64_t>& masks, int window) {
        std::vector<int32_t> starts{0};
        for (int32_t n : fresh) starts.push_back(starts.back() + n);
        const int most = std::max(1, *std::max_element(fresh.begin(), fresh.end()));
        const size_t rows = static_cast<size_t>(starts.back());
        const auto dn = ints(d, fresh), ds = ints(d, starts);
        const auto dm = words(d, masks);
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
            moa::ops::paged_tree_attention(d, dq, cache, ds, dm, out, static_cast<int>(layer), window, kScale, most);
            worst = std::max(worst, check(out.to_host(d), hq, starts, masks, layer, window));
        }
        report(name, worst <= 1.0 && lens.to_host(d) == lengths(), worst);
    }

    // Every sequence of the batch takes a token.
    void tokens(const char* name, int window) { step(name, std::vector<int32_t>(kSeqs, 1), std::vector<uint64_t>(kSeqs, 1), window); }

    std::vector<int32_t> lengths() const {
        std::vector<int32_t> n;
        for (size_t s = 0; s < kSeqs; ++s) n.push_back(static_cast<int32_t>(length(s)));
        return n;
    }

    // The largest error over its bound: bf16 weights move a result by at most 2^-8 of the attention of |v|, the
    // rounding to bf16 by 2^-8 of it; exact values, so the scores' and sums' f32 roundings stay below 2^-14 of it.
    double check(const std::vector<bf16>& out, const std::vector<float>& q, const std::vector<int32_t>& starts,
                 const std::vector<uint64_t>& masks, size_t layer, int window) const {
        double worst = 0.0;
        for (size_t s = 0; s < kSeqs; ++s) {
            const int n = starts[s + 1] - starts[s], base = static_cast<int>(length(s)) - n;
            const auto &ks = kept[s][layer][0], &vs = kept[s][layer][1];
            for (int i = 0; i < n; ++i) {
                const size_t row = starts[s] + i;
                std::vector<int> sees;
                int depth = 0;
                for (int j = 0; j < n; ++j) depth += masks[row] >> j & 1;
                for (int t = window ? std::max(0, base + depth - window) : 0; t < base; ++t) sees.push_back(t);
                for (int j = 0; j < n; ++j)
                    if (masks[row] >> j & 1) sees.push_back(base + j);
                for (size_t h = 0; h < kHeads * kGroup; ++h) {
                    const size_t kvh = h / kGroup;
                    std::vector<double> x;
                    for (int t : sees) {
                        double dot = 0.0;
                        for (size_t j = 0; j < kDim; ++j) dot += static_cast<double>(q[row * kQ + h * kDim + j]) * ks[t * kKv + kvh * kDim + j];
                        x.push_back(dot * kScale);
                    }
                    const double m = *std::max_element(x.begin(), x.end());
                    double sum = 0.0;
                    for (double& e : x) sum += e = std::exp(e - m);
                    for (size_t j = 0; j < kDim; ++j) {
                        double want = 0.0, spread = 0.0;
                        for (size_t t = 0; t < sees.size(); ++t) {
                            const double y = x[t] / sum * vs[sees[t] * kKv + kvh * kDim + j];
                            want += y;
                            spread += std::fabs(y);
                        }
                        const double got = to_f32(out[row * kQ + h * kDim + j]);
                        const double tol = std::ldexp(std::fabs(want), -8) + (1 + std::ldexp(1.0, -8)) * spread * (std::ldexp(1.0, -8) + std::ldexp(1.0, -14)) + 1e-30;
                        worst = std::isfinite(got) ? std::max(worst, std::fabs(got - want) / tol) : 1e30;
                    }
                }
            }
        }
        return worst;
    }

    void report(const char* name, bool ok, double worst = 0.0) {
        std::printf("[%-12s %-34s] error %.3f of its bound -> %s\n", std::is_same<T, bf16>::value ? "bf16 pages" : "E4M3 pages", name, worst,
                    ok ? "PASS" : "FAIL");
        failed += ok ? 0 : 1;
    }

    // Reference counts: the table entries in use that name each page.
    void count(const char* name) {
        const auto t = table.to_host(d), n = lens.to_host(d), r = refs.to_host(d);
        std::vector<int32_t> want(kPages, 0);
        for (size_t s = 0; s < kSeqs; ++s)
            for (size_t i = 0; i < (n[s] + kSlots - 1) / kSlots; ++i) ++want[t[s * kColumns + i]];
        report(name, r == want && n == lengths());
    }

    static std::vector<uint64_t> chain(const std::vector<int32_t>& fresh) {
        std::vector<uint64_t> m;
        for (int32_t n : fresh)
            for (int32_t i = 0; i < n; ++i) m.push_back(~0ull >> (63 - i));
        return m;
    }

    // Trees of 5, 1, 0 and 3 nodes. The logits' largest lead from node 0 of the first to its second child (node 2) and that one's child
    // (node 4), whose own token nothing drafted; the second has its root alone; the third of the last's nodes continues the second.
    void speculate() {
        const std::vector<int32_t> starts{0, 5, 6, 6, 9}, drafted{7, 10, 11, 12, 13, 20, 30, 31, 32};
        const std::vector<uint64_t> masks{1, 3, 5, 9, 21, 1, 1, 3, 7};
        const std::vector<int32_t> largest{11, 1, 13, 2, 300, 40, 31, 0, 5}, leaf{4, 0, -1, 1}, next{300, 40, -1, 0};
        step("trees", {5, 1, 0, 3}, masks, 0);
        std::vector<float> x = values(9 * kVocab);
        for (size_t r = 0; r < 9; ++r) x[r * kVocab + largest[r]] = 4.0f;
        const auto logits = upload(d, x, {9, kVocab});
        const auto tokens = ints(d, drafted), ds = ints(d, starts);
        const auto dm = words(d, masks);
        HbmTensor<int32_t> best(d, {9}), leaves(d, {kSeqs}), nexts(d, {kSeqs});
        moa::ops::tree_verify(d, logits, tokens, ds, dm, best, leaves, nexts);
        report("verification", best.to_host(d) == largest && leaves.to_host(d) == leaf && nexts.to_host(d) == next);
        moa::ops::paged_tree_commit(d, cache, ds, dm, leaves);
        for (size_t s = 0; s < kSeqs; ++s) {
            const int n = starts[s + 1] - starts[s];
            if (!n) continue;
            for (size_t l = 0; l < kLayers; ++l)
                for (int w = 0; w < 2; ++w) {
                    auto& rows = kept[s][l][w];
                    const size_t base = rows.size() / kKv - n;
                    std::vector<float> path(rows.begin(), rows.begin() + base * kKv);
                    for (int j = 0; j < n; ++j)
                        if (masks[starts[s] + leaf[s]] >> j & 1) path.insert(path.end(), rows.begin() + (base + j) * kKv, rows.begin() + (base + j + 1) * kKv);
                    rows = path;
                }
        }
        count("counts after the commit");
        this->tokens("tokens behind the paths", 0);
    }

    // Groups of two beams: scores far apart, or logits, that make both children the second beam's in the first group and swap the beams
    // of the second.
    void beams() {
        const std::vector<int32_t> want_parents{1, 1, 3, 2}, want_tokens{9, 100, 300, 17}, want_finished{0, 0, 1, 0};
        std::vector<float> x(kSeqs * kVocab, 0.0f);
        x[1 * kVocab + 9] = 16.0f, x[1 * kVocab + 100] = 15.0f, x[2 * kVocab + 17] = 16.0f, x[3 * kVocab + 300] = 16.0f;
        const auto logits = upload(d, x, {kSeqs, kVocab});
        const auto scores = HbmTensor<float>::from_host(d, {-1.0f, -1.0f, -2.0f, -1.0f}, {kSeqs});
        HbmTensor<int32_t> finished(d, {kSeqs}), ended(d, {kSeqs}), parents(d, {kSeqs}), next(d, {kSeqs});
        HbmTensor<float> totals(d, {kSeqs});
        moa::ops::beam_select(d, logits, scores, finished, totals, ended, parents, next, 2, 300);
        const auto got = totals.to_host(d);
        double worst = 0.0;
        for (size_t r = 0; r < kSeqs; ++r) {
            const int p = want_parents[r];
            const float* row = &x[p * kVocab];
            double sum = 0.0;
            for (size_t t = 0; t < kVocab; ++t) sum += std::exp(static_cast<double>(row[t]));
            const double want = (p == 2 ? -2.0 : -1.0) + row[want_tokens[r]] - std::log(sum);
            // exponentials and their sum in f32 (301 terms, a few steps of 2^-24 each: below 2^-14 of the sum), one rounding
            worst = std::max(worst, std::fabs(got[r] - want) / (std::ldexp(1.0, -14) + std::ldexp(std::fabs(want), -24)));
        }
        report("selection", worst <= 1.0 && parents.to_host(d) == want_parents && next.to_host(d) == want_tokens && ended.to_host(d) == want_finished,
               worst);
        moa::ops::paged_cache_reorder(d, cache, parents, 2);
        std::vector<float> was[kSeqs][kLayers][2];
        for (size_t s = 0; s < kSeqs; ++s)
            for (size_t l = 0; l < kLayers; ++l)
                for (int w = 0; w < 2; ++w) was[s][l][w] = kept[s][l][w];
        for (size_t s = 0; s < kSeqs; ++s)
            for (size_t l = 0; l < kLayers; ++l)
                for (int w = 0; w < 2; ++w) kept[s][l][w] = was[want_parents[s]][l][w];
        count("counts after the reorder");
        tokens("tokens of the chosen beams", 24);
    }

    int all() {
        const std::vector<int32_t> prompts{35, 13, 1, 60};
        step("prompts", prompts, chain(prompts), 0);
        speculate();
        beams();
        tokens("tokens in a window", 24);
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
    const auto starts = ints(d, {0, 1, 1, 1, 1}), two = ints(d, {1, 1}), three = ints(d, {0, 0, 0});
    const auto one = words(d, {1}), masks = words(d, {1, 1});
    HbmTensor<bf16> q(d, {1, 6, kDim}), small(d, {1, 6, 32}), logits(d, {2, kVocab}), flat(d, {2 * kVocab});
    HbmTensor<uint64_t> wide(d, {1, 5});
    HbmTensor<int32_t> a(d, {2}), b(d, {2}), c(d, {2}), e(d, {2}), leaves(d, {kSeqs});
    HbmTensor<float> f(d, {2}), g(d, {3});
    int failed = 0;
    failed += !throws("heads of 32 dims", [&] { moa::ops::paged_tree_attention(d, small, r.cache, starts, one, small); });
    failed += !throws("masks of two rows", [&] { moa::ops::paged_tree_attention(d, q, r.cache, starts, masks, q); });
    failed += !throws("masks of five words", [&] { moa::ops::paged_tree_attention(d, q, r.cache, starts, wide, q); });
    failed += !throws("a window below max_rows", [&] {
        HbmTensor<bf16> rows(d, {2, 6, kDim});
        moa::ops::paged_tree_attention(d, rows, r.cache, starts, masks, rows, 0, 1);
    });
    failed += !throws("leaves of two", [&] { moa::ops::paged_tree_commit(d, r.cache, starts, one, two); });
    failed += !throws("three parents of pairs", [&] { moa::ops::paged_cache_reorder(d, r.cache, three, 2); });
    failed += !throws("flat logits", [&] { moa::ops::tree_verify(d, flat, two, starts, masks, a, leaves, b); });
    failed += !throws("next tokens of two", [&] { moa::ops::tree_verify(d, logits, two, starts, masks, a, leaves, b); });
    failed += !throws("rows that are no groups", [&] { moa::ops::beam_select(d, logits, f, a, f, b, c, e, 3); });
    failed += !throws("scores of three", [&] { moa::ops::beam_select(d, logits, g, a, f, b, c, e, 2); });
    failed += !throws("an eos past the vocabulary", [&] { moa::ops::beam_select(d, logits, f, a, f, b, c, e, 2, kVocab); });
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
