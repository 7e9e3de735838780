// Where the rows of a tensor lie in memory, so that a call whose outputs lie over its inputs is refused beforehand (its workgroups
// would race).  Host code without HIP.
#pragma once

#include <stdint.h>

namespace llmops {

typedef __int128 Wide;  // (strides are the caller's: products of them have to fit)

// Rows of `width` bytes at base + i * step[0] + j * step[1], i < count[0], j < count[1]; steps not negative, step[0] the larger one
struct Extent {
    Wide base, step[2], width;
    int64_t count[2];

    Extent(const void* p, int64_t n0, Wide step0, int64_t n1, Wide step1, Wide bytes) : base((Wide) reinterpret_cast<uintptr_t>(p)), width(bytes) {
        const int64_t n[2] = {n0, n1};
        Wide s[2] = {n0 > 1 ? step0 : 0, n1 > 1 ? step1 : 0};
        for (int d = 0; d < 2; d++)
            if (s[d] < 0) base += (n0 > 0 && n1 > 0 ? n[d] - 1 : 0) * s[d], s[d] = -s[d];
        const int first = s[0] >= s[1] ? 0 : 1;
        for (int d = 0; d < 2; d++) step[d] = s[first ^ d], count[d] = n[first ^ d];
    }
    Extent(const void* p, Wide bytes) : Extent(p, 1, 0, 1, 0, bytes) {}

    bool empty() const { return count[0] <= 0 || count[1] <= 0 || width <= 0; }
    Wide inner() const { return (count[1] - 1) * step[1] + width; }  // what the rows of one i span
    Wide end() const { return base + (count[0] - 1) * step[0] + inner(); }
    // rows one behind the other: those of one i, and those of i behind those of i - 1
    bool nested() const { return (count[1] == 1 || step[1] >= width) && (count[0] == 1 || step[0] >= inner()); }
    // a nested one: does a row meet [from, from + bytes)?
    bool meets(Wide from, Wide bytes) const {
        from -= base;
        const Wide i = from < inner() ? 0 : count[0] == 1 ? 1 : (from - inner()) / step[0] + 1;  // the first whose span ends behind `from`
        if (i >= count[0] || i * step[0] >= from + bytes) return false;
        if (i + 1 < count[0] && (i + 1) * step[0] < from + bytes) return true;  // (the next one's first row starts inside)
        from -= i * step[0];
        const Wide j = from < width ? 0 : count[1] == 1 ? 1 : (from - width) / step[1] + 1;
        return j < count[1] && j * step[1] < from + bytes;
    }
};

// no row of x lies over another of x
inline bool rows_apart(const Extent& x) {
    if (x.empty() || x.nested()) return true;
    // rows (0, 0) and (i, -j) or (i, j): for each j the two i whose row starts nearest
    for (int64_t j = 0; j < x.count[1]; j++)
        for (int up = 0; up < 2; up++) {
            const Wide i = x.step[0] > 0 ? j * x.step[1] / x.step[0] + up : up;
            if (i == 0 && j == 0) continue;
            const Wide gap = i * x.step[0] - j * x.step[1];
            if (i < x.count[0] && gap < x.width && -gap < x.width) return false;
        }
    return true;
}

// no row of x lies over one of y.  (Where their spans meet, y's rows are looked at one by one; an x that is not nested then counts as lying over y.)
inline bool apart(const Extent& x, const Extent& y) {
    if (x.empty() || y.empty() || x.end() <= y.base || y.end() <= x.base) return true;
    if (!x.nested()) return false;
    const bool whole = y.count[1] == 1 || y.step[1] == y.width;  // (rows without a gap)
    const Wide bytes = whole ? y.inner() : y.width;
    for (int64_t i = 0; i < y.count[0]; i++)
        for (int64_t j = 0; j < (whole ? 1 : y.count[1]); j++)
            if (x.meets(y.base + i * y.step[0] + j * y.step[1], bytes)) return false;
    return true;
}

}  // namespace llmops
