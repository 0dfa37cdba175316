// Byte ranges of a call's arrays, and whether something that is written meets something else.
#pragma once

#include <cstddef>
#include <cstdint>

namespace chroma_ranges {

struct Range {
    const void* begin;
    uint64_t bytes;
    bool written;
};

// Null ranges and empty ones meet nothing.
inline bool meet(const Range& a, const Range& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.begin), y = reinterpret_cast<uintptr_t>(b.begin);
    return x && y && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
}

template <size_t N> bool overlap(const Range (&ranges)[N]) {
    for (size_t i = 0; i < N; ++i) {
        for (size_t j = i + 1; j < N; ++j) {
            if ((ranges[i].written || ranges[j].written) && meet(ranges[i], ranges[j])) {
                return true;
            }
        }
    }
    return false;
}

}  // namespace chroma_ranges
