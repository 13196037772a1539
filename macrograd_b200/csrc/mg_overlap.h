// mg_overlap.h -- whether two strided views of memory have a byte in common.
//
// Views of one buffer may span the same bytes without sharing any (the queries, keys and
// values of a packed projection), so spans alone do not tell. With all strides made positive
// the distance of two elements is D + sum c_k z_k, 0 <= z_k <= m_k, one term for each dim of
// either view, and the views meet if some distance lies within an element's size. The terms
// are tried from the largest stride down: what the smaller ones can still reach leaves one
// or two values of z_k where strides are nested, and where they reach everywhere (to the
// size of an element) the answer is known.
#pragma once

#include <algorithm>
#include <cstdint>

namespace mg {

struct View {
    const void* at;
    int elem;                    // bytes of an element
    int64_t n[4], stride[4];     // dims (1 where there are fewer) and strides in elements
};

namespace overlap {

typedef __int128 wide;           // no product of a stride and a size overflows

struct Terms {
    wide c[8], m[8], reach[9], gap[9];     // reach, gap: of the terms from k on; largest step between two sums
    int count;
    int64_t budget;
};

inline bool within(Terms& t, int k, wide lo, wide hi)
{
    if (hi < 0 || lo > t.reach[k]) return false;
    if (hi - lo + 1 >= t.gap[k]) return true;
    const wide c = t.c[k], below = t.reach[k + 1];
    wide z = lo > below ? (lo - below + c - 1) / c : 0;
    for (const wide last = std::min(t.m[k], hi / c); z <= last; ++z) {
        if (--t.budget < 0) return true;   // not decided: taken as an overlap
        if (within(t, k + 1, lo - z * c, hi - z * c)) return true;
    }
    return false;
}

}  // namespace overlap

// The bytes [lo, hi) that a view spans; none where it has no element.
struct Span {
    overlap::wide lo, hi;
};

inline Span span_of(const View& v)
{
    Span s = {(overlap::wide)(intptr_t)v.at, (overlap::wide)(intptr_t)v.at + v.elem};
    for (int i = 0; i < 4; ++i) {
        if (v.n[i] <= 0) return {0, 0};
        const overlap::wide far = (overlap::wide)v.stride[i] * v.elem * (v.n[i] - 1);
        (far < 0 ? s.lo : s.hi) += far;
    }
    return s;
}

inline bool views_meet(const View& a, const View& b)
{
    using overlap::wide;
    for (int i = 0; i < 4; ++i)
        if (a.n[i] <= 0 || b.n[i] <= 0) return false;
    overlap::Terms t;
    t.count = 0;
    t.budget = 1 << 16;
    wide start = (wide)(intptr_t)a.at - (wide)(intptr_t)b.at;      // of the smallest distance
    for (int i = 0; i < 8; ++i) {
        const View& v = i < 4 ? a : b;
        const wide m = v.n[i % 4] - 1, s = (wide)v.stride[i % 4] * v.elem * (i < 4 ? 1 : -1), c = s < 0 ? -s : s;
        if (m == 0 || c == 0) continue;
        if (s < 0) start += s * m;
        int k = 0;
        while (k < t.count && t.c[k] > c) ++k;
        if (k < t.count && t.c[k] == c) {
            t.m[k] += m;
            continue;
        }
        for (int j = t.count++; j > k; --j) t.c[j] = t.c[j - 1], t.m[j] = t.m[j - 1];
        t.c[k] = c, t.m[k] = m;
    }
    t.reach[t.count] = t.gap[t.count] = 0;
    for (int k = t.count - 1; k >= 0; --k) {
        t.reach[k] = t.reach[k + 1] + t.c[k] * t.m[k];
        t.gap[k] = std::max(t.gap[k + 1], t.c[k] - t.reach[k + 1]);
    }
    // an element of a starts less than b's size behind one of b's, and less than its own before it
    return overlap::within(t, 0, 1 - a.elem - start, b.elem - 1 - start);
}

// The same elements in the same places.
inline bool same_view(const View& a, const View& b)
{
    if (a.at != b.at || a.elem != b.elem) return false;
    for (int i = 0; i < 4; ++i)
        if (a.n[i] != b.n[i] || (a.n[i] > 1 && a.stride[i] != b.stride[i])) return false;
    return true;
}

}  // namespace mg
