// Whether two buffers of a request share a byte: what an operator writes may
// not be what it reads or writes elsewhere.  Plain C++, checked on the host.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <utility>

namespace qwn {

// `rows` rows of `width` bytes, `stride` bytes apart; a null pointer is no buffer.
struct Rows {
    const void *data = nullptr;
    uint64_t rows = 0, width = 0, stride = 0;

    uint64_t at() const { return reinterpret_cast<uintptr_t>(data); }
    bool none() const { return !data || rows == 0 || width == 0; }
    uint64_t end() const { return at() + (rows - 1) * stride + width; }
    bool dense() const { return rows == 1 || width == stride; }
};

inline Rows row_block(const void *data, uint64_t rows, uint64_t cols, uint64_t stride, uint64_t element) {
    return Rows{data, rows, cols * element, stride * element};
}
inline Rows list_of_bytes(const void *data, uint64_t bytes) { return Rows{data, 1, bytes, bytes}; }

// A row of r in the bytes [from, to): the first that ends past `from` begins before `to`.
inline bool row_within(const Rows &r, uint64_t from, uint64_t to) {
    const uint64_t reach = r.at() + r.width;
    const uint64_t i = reach > from ? 0 : (from - reach) / r.stride + 1;
    return i < r.rows && r.at() + i * r.stride < to;
}

inline bool overlap(Rows a, Rows b) {
    if (a.none() || b.none() || a.end() <= b.at() || b.end() <= a.at()) return false;
    if (a.dense()) return row_within(b, a.at(), a.end());
    if (b.dense()) return row_within(a, b.at(), b.end());
    if (a.at() > b.at()) std::swap(a, b);
    if (a.stride == b.stride) {  // columns of one buffer: b's begin in a's, or reach a's next row
        const uint64_t d = (b.at() - a.at()) % a.stride;
        return d < a.width || d + b.width > a.stride;
    }
    if (a.rows > b.rows) std::swap(a, b);
    for (uint64_t i = 0; i < a.rows; ++i) {
        const uint64_t from = a.at() + i * a.stride;
        if (row_within(b, from, from + a.width)) return true;
    }
    return false;
}

// The same elements in the same places: a result in place of its input.
inline bool in_place(const Rows &a, const Rows &b) {
    return a.data == b.data && a.width == b.width && (a.stride == b.stride || a.rows == 1);
}

inline bool overlaps_any(const Rows &out, std::initializer_list<Rows> others) {
    for (const Rows &r : others)
        if (overlap(out, r)) return true;
    return false;
}

}  // namespace qwn
