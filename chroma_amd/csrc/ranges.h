// Byte ranges of a call's arrays, and whether something that is written meets something else.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

namespace chroma_ranges {

struct Range {
    const void* begin;
    uint64_t bytes;
    bool written;
};

struct Axis {
    int64_t count, stride;
};

// Bytes from an array's first element to its last one's end, of ``size`` bytes each; past 2^62 as 2^62, which meets all that
// lies behind.
inline uint64_t bytes_of(std::initializer_list<Axis> axes, uint64_t size) {
    unsigned __int128 last = 0;
    for (const Axis& axis : axes) {
        last += static_cast<unsigned __int128>(axis.count - 1) * uint64_t(axis.stride);
    }
    const unsigned __int128 bytes = (last + 1u) * size;
    return bytes >> 62 ? uint64_t(1) << 62 : uint64_t(bytes);
}

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
