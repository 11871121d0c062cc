// Whether the memory that a call writes lies apart from all else it is given (host side, nothing is read): a kernel whose
// CTAs write while others still read would answer by chance where a caller lets two of its tensors share memory.
#pragma once
#include <stdint.h>

#include <initializer_list>

struct PrbRange {
    const void* at;
    long bytes;                              // none where the call does without it
};

// bytes from the first of `rows` rows to the end of the last
inline long prb_span(long rows, long stride, long width) { return rows > 0 ? (rows - 1) * stride + width : 0; }

inline bool prb_overlap(const PrbRange& a, const PrbRange& b) {
    if (a.at == nullptr || b.at == nullptr || a.bytes <= 0 || b.bytes <= 0) return false;
    const uintptr_t x = (uintptr_t)a.at, y = (uintptr_t)b.at;
    return x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}

// every range that is written lies apart from every other range
inline bool prb_apart(std::initializer_list<PrbRange> written, std::initializer_list<PrbRange> read) {
    for (auto w = written.begin(); w != written.end(); ++w) {
        for (auto o = w + 1; o != written.end(); ++o)
            if (prb_overlap(*w, *o)) return false;
        for (const PrbRange& r : read)
            if (prb_overlap(*w, r)) return false;
    }
    return true;
}

// two sets of rows of `width` bytes lie apart: anywhere, or as column slices of one tensor (of one stride)
inline bool prb_rows_apart(const void* a, long a_stride, const void* b, long b_stride, long rows, long width) {
    if (!prb_overlap({a, prb_span(rows, a_stride, width)}, {b, prb_span(rows, b_stride, width)})) return true;
    if (a_stride != b_stride || a_stride <= 0) return false;
    const long ahead = (((long)((uintptr_t)b - (uintptr_t)a)) % a_stride + a_stride) % a_stride;
    return ahead >= width && ahead <= a_stride - width;
}
