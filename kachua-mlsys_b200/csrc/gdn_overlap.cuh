// gdn_overlap.cuh -- whether two tensors of evenly spaced rows share memory
// (host code, plain C++).
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace gdn {

// `width` bytes at p, p + step, ...
struct Rows {
    const void* p;
    int64_t rows, step, width;
};

inline bool same_rows(const Rows& a, const Rows& b) {
    return a.p == b.p && a.rows == b.rows && a.width == b.width && (a.rows <= 1 || a.step == b.step);
}

// Exact where one of the two is contiguous or both have one step, so for two
// column blocks of a buffer.  With other steps rows of both come by at every
// multiple of the steps' common divisor, which is taken for any such distance:
// two tensors that miss each other only by where they end count as meeting.
inline bool rows_meet(Rows a, Rows b) {
    using I = __int128;  // strides are the caller's
    if (!a.p || !b.p || a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1) return false;
    for (Rows* t : {&a, &b})
        if (t->rows > 1 && t->step == t->width) t->width *= t->rows, t->rows = 1;
    if (a.rows == 1) {
        const Rows t = a;
        a = b;
        b = t;
    }
    const auto floor_div = [](I n, I d) { return n / d - (n % d < 0); };  // d > 0
    const I pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    if (pa + (a.rows - 1) * I(a.step) + a.width <= pb || pb + (b.rows - 1) * I(b.step) + b.width <= pa) return false;
    if (a.rows == 1) return true;
    if (b.rows > 1 && a.step != b.step) {
        I g = a.step;
        for (I r = b.step; r != 0;) {
            const I t = g % r;
            g = r;
            r = t;
        }
        const I d = pb - pa - floor_div(pb - pa, g) * g;  // from a row of a to the next of b
        return d < a.width || g - d < b.width;
    }
    // the difference of a row of a and one of b takes every multiple of the step here
    const I first = pa - (b.rows - 1) * I(a.step), rows = I(a.rows) + b.rows - 1;
    I lo = floor_div(pb - a.width - first, a.step) + 1, hi = -floor_div(-(pb + b.width - first), a.step) - 1;
    if (lo < 0) lo = 0;
    if (hi > rows - 1) hi = rows - 1;
    return lo <= hi;
}

// An output meets no other output, and an input only where it may be that
// input itself (`in_place`), row for row.
struct Operands {
    static constexpr int kMost = 16;
    Rows in[kMost], out[kMost];
    bool in_place[kMost];
    int ins = 0, outs = 0;
    void read(const void* p, int64_t rows, int64_t step, int64_t width) { in[ins++] = {p, rows, step, width}; }
    void write(const void* p, int64_t rows, int64_t step, int64_t width, bool may_be_input = false) {
        in_place[outs] = may_be_input;
        out[outs++] = {p, rows, step, width};
    }
    bool apart() const {
        for (int i = 0; i < outs; ++i) {
            for (int j = 0; j < i; ++j)
                if (rows_meet(out[i], out[j])) return false;
            for (int j = 0; j < ins; ++j)
                if (rows_meet(out[i], in[j]) && !(in_place[i] && same_rows(out[i], in[j]))) return false;
        }
        return true;
    }
};

}  // namespace gdn
