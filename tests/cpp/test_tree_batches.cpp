// test_tree_batches.cpp -- batches of drafted trees over the C++ host interface (moa-workspace_amd/host/moa_ops.hpp) that leave max_rows
// to its default.
//
// TEST INFRASTRUCTURE. Sequences of as many nodes each, more rows in all than a tree has mask bits: the call without max_rows gives
// the bits of the call that says how many rows a sequence has, in rows that all hold something else before.
//
//   test_tree_batches     on device 0
#include <cstdio>
#include <string>
#include <vector>

#include "moa_ops.hpp"

using moa::bf16;
using moa::Device;
using moa::HbmTensor;

namespace {

constexpr size_t kSlots = 16, kHeads = 2, kDim = 64;

uint32_t state = 7;
std::vector<bf16> values(size_t n) {  // bf16 numbers between 1/8 and 1, of both signs
    std::vector<bf16> v(n);
    for (bf16& x : v) {
        state = state * 1664525u + 1013904223u;
        x.bits = static_cast<uint16_t>(0x3e00u + (state >> 16 & 0x8000u) + (state >> 8 & 0x17fu));
    }
    return v;
}

// `seqs` chains of n nodes before which nothing lies, masks of `words` words.
bool batch(const Device& d, size_t seqs, size_t n, size_t words) {
    const size_t columns = (n + kSlots - 1) / kSlots, pages = seqs * columns, rows = seqs * n;
    HbmTensor<bf16> k(d, {1, pages, kSlots, kHeads, kDim}), v(d, {1, pages, kSlots, kHeads, kDim});
    HbmTensor<int32_t> table(d, {seqs, columns}), lens(d, {seqs}), refs(d, {pages});
    moa::PagedCache<bf16> cache(k, v, table, lens, refs);
    std::vector<int32_t> starts;
    std::vector<uint64_t> masks(rows * words, 0);
    for (size_t s = 0; s <= seqs; ++s) starts.push_back(static_cast<int32_t>(s * n));
    for (size_t r = 0; r < rows; ++r)
        for (size_t j = 0; j <= r % n; ++j) masks[r * words + j / 64] |= 1ull << j % 64;
    const auto ds = HbmTensor<int32_t>::from_host(d, starts, {seqs + 1});
    const auto dm = HbmTensor<uint64_t>::from_host(d, masks, {rows, words});
    moa::ops::paged_cache_reserve(d, cache, HbmTensor<int32_t>::from_host(d, std::vector<int32_t>(seqs, static_cast<int32_t>(n)), {seqs}));
    const auto dk = HbmTensor<bf16>::from_host(d, values(rows * kHeads * kDim), {rows, kHeads, kDim});
    const auto dv = HbmTensor<bf16>::from_host(d, values(rows * kHeads * kDim), {rows, kHeads, kDim});
    const auto dq = HbmTensor<bf16>::from_host(d, values(rows * kHeads * kDim), {rows, kHeads, kDim});
    moa::ops::paged_cache_append(d, cache, dk, dv, ds);
    auto out = HbmTensor<bf16>::from_host(d, std::vector<bf16>(rows * kHeads * kDim, bf16{0x7fc0}), {rows, kHeads, kDim});
    auto want = HbmTensor<bf16>::from_host(d, std::vector<bf16>(rows * kHeads * kDim, bf16{0x7fc0}), {rows, kHeads, kDim});
    int code = 0;
    try {
        moa::ops::paged_tree_attention(d, dq, cache, ds, dm, out);
    } catch (const moa::Error& e) {
        code = e.code();
    }
    moa::ops::paged_tree_attention(d, dq, cache, ds, dm, want, 0, 0, 1.0f, static_cast<int>(n));
    const auto a = out.to_host(d), b = want.to_host(d);
    bool ok = code == 0;
    for (size_t i = 0; i < a.size(); ++i) ok = ok && a[i].bits == b[i].bits && (a[i].bits & 0x7f80) != 0x7f80;
    std::printf("[%zu chains of %zu, %zu words] code %d -> %s\n", seqs, n, words, code, ok ? "PASS" : "FAIL");
    return ok;
}

}  // namespace

int main() {
    try {
        Device device(0);
        int failed = 0;
        for (const auto& c : {std::vector<size_t>{1, 2, 1}, {3, 40, 1}, {40, 17, 1}, {2, 128, 2}, {5, 200, 4}})
            failed += !batch(device, c[0], c[1], c[2]);
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
