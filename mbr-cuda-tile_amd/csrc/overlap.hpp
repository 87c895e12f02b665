// Whether two sets of rows in memory share a byte: the check of entry points that refuse an output within an input.
#pragma once

#include <stdint.h>

#include <utility>

namespace mbrt {

// n rows of len bytes, one every step bytes.
struct MemRows {
    const void* at;
    int64_t step, len, n;
};

// Whether two such sets share a byte.  Rows of one set between those of the other (columns of one wider matrix) do not.
inline bool rows_meet(MemRows a, MemRows b) {
    if (a.n <= 0 || b.n <= 0 || a.len <= 0 || b.len <= 0) return false;
    typedef __int128 wide;
    auto begin = [](const MemRows& r) { return (wide) reinterpret_cast<uintptr_t>(r.at); };
    auto end = [&](const MemRows& r) { return begin(r) + (wide)(r.n - 1) * r.step + r.len; };
    if (end(a) <= begin(b) || end(b) <= begin(a)) return false;
    for (MemRows* r : {&a, &b})  // rows that touch or overlap: one row
        if (r->step <= r->len) *r = MemRows{r->at, 0, (int64_t)(end(*r) - begin(*r)), 1};
    if (a.n > b.n) std::swap(a, b);
    // row i of a against the first row of b that ends behind its beginning
    auto row_meets = [&](wide i) {
        const wide lo = begin(a) + i * a.step, past = lo - begin(b) - b.len;
        const wide j = past < 0 || b.n == 1 ? (past < 0 ? 0 : 1) : past / b.step + 1;
        return j < b.n && begin(b) + j * b.step < lo + a.len;
    };
    if (b.n > 1 && a.step == b.step) {  // equal steps: a pair that meets can be moved until one of the two is its set's first row
        const wide d = begin(b) - begin(a), i = d >= 0 ? d / a.step : -1;
        return row_meets(0) || (i >= 0 && i < a.n && row_meets(i)) || (i + 1 >= 0 && i + 1 < a.n && row_meets(i + 1));
    }
    for (int64_t i = 0; i < a.n; ++i)
        if (row_meets(i)) return true;
    return false;
}

}  // namespace mbrt
