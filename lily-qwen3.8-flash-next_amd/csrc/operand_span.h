// operand_span.h - an operand as memory: whether it can be where it is said to be, and what it shares
// with another.
#pragma once

#include <cstdint>

#include "../../include/lily_sampler.h"

namespace lily {

// An operand as memory: `rows` rows of `width` bytes, `stride` bytes apart.
struct Span {
    uint64_t at = 0, rows = 0, width = 0, stride = 0;
    uint32_t dtype = 0;
};

inline uint64_t size_of(uint32_t dtype) { return dtype == LILY_F32 ? 4u : dtype == LILY_BF16 ? 2u : 1u; }

inline Span span(const void* p, uint64_t rows, uint64_t columns, uint64_t stride, uint32_t dtype) {
    const uint64_t e = size_of(dtype);
    Span s;
    s.at = reinterpret_cast<uintptr_t>(p);
    s.rows = p != nullptr ? rows : 0u;
    s.width = columns * e;
    // (one row: its stride says nothing; one beyond all memory stays there in bytes)
    s.stride = rows <= 1u ? columns * e : stride < (1ull << 59) ? stride * e : 1ull << 63;
    s.dtype = dtype;
    return s;
}

inline bool aligned(const Span& s) { return s.rows == 0u || (s.at % 16u == 0u && s.stride % 16u == 0u); }

// The last byte behind a span must be an address.
inline bool fits(const Span& s) {
    if (s.rows == 0u) {
        return true;
    }
    const unsigned __int128 end = (unsigned __int128)s.at + (unsigned __int128)(s.rows - 1u) * s.stride + s.width;
    return end <= (unsigned __int128)1 << 63;
}

// Whether two operands share a byte.  Rows of one stride are compared within it, so that columns of a
// wider buffer side by side are apart; otherwise the whole ranges are.
inline bool overlap(const Span& a, const Span& b) {
    if (a.rows == 0u || b.rows == 0u) {
        return false;
    }
    const uint64_t end_a = a.at + (a.rows - 1u) * a.stride + a.width, end_b = b.at + (b.rows - 1u) * b.stride + b.width;
    if (end_a <= b.at || end_b <= a.at) {
        return false;
    }
    if (a.stride == b.stride && a.rows > 1u && b.rows > 1u) {
        const uint64_t s = a.stride, off = b.at >= a.at ? (b.at - a.at) % s : (s - (a.at - b.at) % s) % s;
        return !(off >= a.width && off + b.width <= s);
    }
    return true;
}

// An output may be an input itself: then every element is read by the thread that writes it, or a
// row is read whole before any of it is written.
inline bool same(const Span& a, const Span& b) {
    return a.at == b.at && a.dtype == b.dtype && a.stride == b.stride && a.width == b.width;
}

}  // namespace lily
