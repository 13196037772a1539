// overlap_check.cpp -- CPU check of macrograd_b200/csrc/mg_overlap.h against all pairs of
// elements of small random views. Built and run by tests/test_overlap.py; prints "ok" or the
// first failure.
#include <cstdio>
#include <random>
#include <set>

#include "mg_overlap.h"

using mg::View;

static std::set<int64_t> bytes_of(const View& v)
{
    std::set<int64_t> all;
    for (int64_t a = 0; a < v.n[0]; ++a)
        for (int64_t b = 0; b < v.n[1]; ++b)
            for (int64_t c = 0; c < v.n[2]; ++c)
                for (int64_t d = 0; d < v.n[3]; ++d)
                    for (int e = 0; e < v.elem; ++e)
                        all.insert((int64_t)(intptr_t)v.at + e +
                                   v.elem * (a * v.stride[0] + b * v.stride[1] + c * v.stride[2] + d * v.stride[3]));
    return all;
}

static View view(int64_t at, int elem, std::initializer_list<int64_t> n, std::initializer_list<int64_t> stride)
{
    View v = {(const void*)(intptr_t)at, elem, {1, 1, 1, 1}, {0, 0, 0, 0}};
    std::copy(n.begin(), n.end(), v.n);
    std::copy(stride.begin(), stride.end(), v.stride);
    return v;
}

int main()
{
    std::mt19937 rng(1);
    const auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    int met = 0;
    for (int round = 0; round < 60000; ++round) {
        View v[2];
        for (View& x : v) {
            x = view(1000 + pick(0, 60), pick(0, 1) ? 2 : 4, {}, {});
            for (int i = 0; i < 4; ++i) {
                x.n[i] = pick(0, 9) ? pick(1, 4) : 0;
                x.stride[i] = pick(0, 3) ? pick(0, 40) : -pick(0, 12);
            }
            x.stride[3] = pick(0, 4) ? 1 : x.stride[3];
        }
        const std::set<int64_t> a = bytes_of(v[0]), b = bytes_of(v[1]);
        bool want = false;
        for (int64_t x : a) want = want || b.count(x);
        met += want;
        const mg::Span s = mg::span_of(v[0]);
        if (!a.empty() && (s.lo != *a.begin() || s.hi != *a.rbegin() + 1)) {
            std::printf("FAIL span, round %d\n", round);
            return 1;
        }
        if (mg::views_meet(v[0], v[1]) != want || mg::views_meet(v[1], v[0]) != want) {
            std::printf("FAIL round %d, want %d\n", round, want);
            return 1;
        }
    }
    // large views, as they are passed: slices of a packed projection [4, 8192, 3, 32, 128], its rows next to one another
    const int64_t L = 3 * 32 * 128;
    const auto heads = [&](int64_t at) { return view(4096 + 2 * at, 2, {4, 32, 8192, 128}, {8192 * L, 128, L, 1}); };
    const View q = heads(0), k = heads(32 * 128), v = heads(2 * 32 * 128);
    // a pool of keys and values side by side, 2^31 elements and more
    const auto pool = [&](int64_t at) { return view(4096 + 2 * at, 2, {70000, 16, 8, 128}, {16 * 8 * 256, 8 * 256, 256, 1}); };
    const View all = view(4096, 2, {4, 32, 8192, 384}, {8192 * L, 384, L, 1});
    if (mg::views_meet(q, k) || mg::views_meet(k, v) || mg::views_meet(q, v) || !mg::views_meet(q, q) ||
        !mg::views_meet(k, heads(32 * 128 + 1)) || !mg::views_meet(all, v) || mg::views_meet(pool(0), pool(128)) ||
        !mg::views_meet(pool(0), pool(127)) || !mg::same_view(q, q) || mg::same_view(q, k)) {
        std::printf("FAIL large views\n");
        return 1;
    }
    // sizes and strides whose product leaves 64 bits
    const int64_t far = INT64_MAX / 4;
    if (mg::views_meet(view(4096, 2, {INT32_MAX, 1, 1, 8}, {far, 0, 0, 1}), view(0, 4, {8, 1, 1, 8}, {8, 0, 0, 1}))) {
        std::printf("FAIL far strides\n");
        return 1;
    }
    // strides that fit no order: an answer, if it is only that they may meet
    const View odd[2] = {view(0, 2, {30000, 30011, 30013, 2}, {60013, 60017, 120011, 1}),
                         view(1 << 20, 2, {30000, 30011, 30013, 2}, {60029, 70001, 110017, 1})};
    if (!mg::views_meet(odd[0], odd[1])) {
        std::printf("FAIL undecided\n");
        return 1;
    }
    std::printf("ok: %d of 60000 pairs meet\n", met);
    return 0;
}
