// Whether operands of a call share memory: host checks of the entry points that may not write over what they read.
#pragma once

#include <algorithm>
#include <cstdint>

namespace b200 {

using wide = __int128;  // (strides are the caller's and unchecked)
// n1 runs, s1 bytes apart, of n2 runs, s2 bytes apart, of `width` bytes each.
struct Runs {
    wide base;
    uint64_t n1, s1, n2, s2, width;
    wide extent;
    Runs(const void* p, uint64_t n1, uint64_t s1, uint64_t n2, uint64_t s2, uint64_t width)
        : base(reinterpret_cast<uintptr_t>(p)), n1(n1), s1(s1), n2(n2), s2(s2), width(width),
          extent(static_cast<wide>(n1 - 1) * s1 + static_cast<wide>(n2 - 1) * s2 + width) {}
};
inline wide floor_div(wide a, wide b) { return a / b - (a % b < 0 ? 1 : 0); }
// Whether two operands share a byte: exactly where their strides are the same (interleaved halves, layers, K and V of one buffer do
// not), by the whole extent of the levels whose strides differ otherwise.
inline bool share_bytes(Runs a, Runs b) {
    const wide apart = b.base - a.base;
    if (a.n1 == 1) a.s1 = b.s1;  // a level of one run has any stride
    if (b.n1 == 1) b.s1 = a.s1;
    if (a.n2 == 1) a.s2 = b.s2;
    if (b.n2 == 1) b.s2 = a.s2;
    if (a.s1 != b.s1) return true;
    wide aw = a.width, bw = b.width;
    if (a.s2 != b.s2) {
        aw += static_cast<wide>(a.n2 - 1) * a.s2;
        bw += static_cast<wide>(b.n2 - 1) * b.s2;
        a.n2 = b.n2 = 1;
    }
    // Some run of a, i1 and i2, and some of b, j1 and j2: apart + (j1 - i1) s1 + (j2 - i2) s2 in (-bw, aw)?
    auto steps = [](wide low, wide high, wide stride, uint64_t an, uint64_t bn, wide* first, wide* last) {  // j - i with low < (j - i) stride < high
        *first = -static_cast<wide>(an - 1);
        *last = bn - 1;
        if (stride == 0) return;
        *first = std::max(*first, floor_div(low, stride) + 1);
        *last = std::min(*last, -floor_div(-high, stride) - 1);
    };
    wide f1, l1, f2, l2;
    steps(-bw - static_cast<wide>(b.n2 - 1) * b.s2 - apart, aw + static_cast<wide>(a.n2 - 1) * a.s2 - apart, a.s1, a.n1, b.n1, &f1, &l1);
    if (l1 - f1 > 64) return true;  // (not looked at one by one)
    for (wide k = f1; k <= l1; ++k) {
        const wide at = apart + k * a.s1;
        steps(-bw - at, aw - at, a.s2, a.n2, b.n2, &f2, &l2);
        if (f2 <= l2 && (a.s2 != 0 || (at > -bw && at < aw))) return true;
    }
    return false;
}
inline bool share_memory(const Runs& a, const Runs& b) { return a.base < b.base + b.extent && b.base < a.base + a.extent && share_bytes(a, b); }

}  // namespace b200
