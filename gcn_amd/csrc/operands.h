// Where the operands of a call lie: a result that shares memory with what other workgroups still read, or with another
// result, is refused on the host, whatever views of one buffer the two are.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace gcn {

// rows of `width` bytes, `pitch` bytes apart
struct Place {
    intptr_t at;
    int64_t rows, width, pitch;
};

template <class T>
inline Place place(const T* p, int64_t rows, int64_t cols, int64_t ld) {
    const int64_t size = (int64_t)sizeof(T);
    if (!p) rows = 0;
    return {(intptr_t)p, rows, cols * size, (rows > 1 ? ld : cols) * size};
}
template <class T>
inline Place place(const T* p, int64_t n) {
    return place(p, 1, n, n);
}

inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); }      // b > 0

// whether a byte belongs to rows of both
inline bool share_memory(Place a, Place b) {
    if (a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1) return false;
    if (a.rows > b.rows) std::swap(a, b);
    const int64_t a_bytes = (a.rows - 1) * a.pitch + a.width, b_bytes = (b.rows - 1) * b.pitch + b.width;
    if (a.at + a_bytes <= b.at || b.at + b_bytes <= a.at) return false;
    // row i of a: b's row j meets it where  at - b.width < j b.pitch < at + a.width,  at = its address from b's on.  At equal
    // pitches a row later is a row later in b: the rows that could meet b's at all begin or end inside it
    auto meets = [&](int64_t i) {
        const int64_t at = a.at + i * a.pitch - b.at;
        const int64_t j = std::max<int64_t>(0, floor_div(at - b.width, b.pitch) + 1);
        return j < b.rows && j * b.pitch < at + a.width;
    };
    const int64_t first = std::max<int64_t>(0, floor_div(b.at - a.at, a.pitch) - 1);
    const int64_t last = std::min(a.rows - 1, floor_div(b.at + b_bytes - a.at, a.pitch) + 1);
    if (a.pitch == b.pitch) return meets(first) || meets(std::min(first + 1, last)) || meets(std::min(first + 2, last));
    for (int64_t i = first; i <= last; ++i)
        if (meets(i)) return true;
    return false;
}

// the same rows: a result over an operand that every row reads before it writes
inline bool same_rows(const Place& a, const Place& b) { return a.at == b.at && (a.rows == 1 || a.pitch == b.pitch); }

// a result that may be the operand itself but lie no other way over it
inline bool lies_across(const Place& out, const Place& in) { return share_memory(out, in) && !same_rows(out, in); }

}  // namespace gcn
