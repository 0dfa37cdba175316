// ``chroma_hip_cache_move``: rows of keys and values copied between caches, or between pages of one, in every layer.
//
// The moves travel as kernel arguments (up to kMoves a launch), so that nothing is uploaded and a captured call replays
// them. What bounds it: a step's rows the launch, pages the memory (each byte read and written once).
#include "cache.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <exception>
#include <type_traits>
#include <vector>

namespace {

constexpr int kMoves = 256;
constexpr int kThreads = 256;

struct Move {
    uint32_t from, to, rows;
};

struct Moves {
    const char* source_keys;
    const char* source_values;
    char* target_keys;
    char* target_values;
    uint64_t source_pitch, target_pitch, row_bytes;  // pitches between layers
    Move move[kMoves];
};
static_assert(sizeof(Moves) <= 4096, "kernel arguments hold 4 KiB");

typedef uint32_t Aligned __attribute__((ext_vector_type(4)));  // 16 bytes
typedef Aligned Bytes __attribute__((aligned(1)));             // at any address

// grid: (pieces of the longest move, moves, layers x keys or values). A thread copies 16 bytes, and what a move's length
// leaves of its last 16 bytes goes byte by byte. Loads and stores are non-temporal: 1500 pages of 16 rows of 1 KiB in 24
// layers (2.4 GB read and written in all) 387 us against 454 through the caches (64 threads: 370 and 437, but 100 pages of
// differing fill 21 us against 12; 4 loads under way a thread: 421 and 478).
template <bool ALIGNED> __global__ void __launch_bounds__(kThreads) move_rows(Moves m) {
    using Unit = std::conditional_t<ALIGNED, Aligned, Bytes>;
    const Move move = m.move[blockIdx.y];
    const uint64_t layer = blockIdx.z / 2u, bytes = move.rows * m.row_bytes, units = bytes / 16u;
    const char* from = (blockIdx.z % 2u ? m.source_values : m.source_keys) + layer * m.source_pitch + move.from * m.row_bytes;
    char* to = (blockIdx.z % 2u ? m.target_values : m.target_keys) + layer * m.target_pitch + move.to * m.row_bytes;
    for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < units; i += uint64_t(gridDim.x) * kThreads) {
        __builtin_nontemporal_store(__builtin_nontemporal_load(reinterpret_cast<const Unit*>(from) + i), reinterpret_cast<Unit*>(to) + i);
    }
    if (blockIdx.x == 0 && threadIdx.x < bytes % 16u) {
        to[units * 16u + threadIdx.x] = from[units * 16u + threadIdx.x];
    }
}

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "cache_move: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

// Whether two of the ranges [begin, end) that are written, or one that is written and one that is read, meet.
struct Range {
    int64_t begin, end;
    bool written;
};
bool clash(std::vector<Range>& ranges) {
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    int64_t read_end = -1, written_end = -1;
    for (const Range& r : ranges) {
        if (r.begin < written_end || (r.written && r.begin < read_end)) {
            return true;
        }
        int64_t& end = r.written ? written_end : read_end;
        end = std::max(end, r.end);
    }
    return false;
}

const char* mistake(const chroma_hip_cache_rows& to, const chroma_hip_cache_rows& from, int64_t layers, int64_t row_bytes,
                    const int64_t* moves, int64_t count) {
    constexpr int64_t kRows = int64_t(1) << 32, kBytes = int64_t(1) << 46;
    if (layers < 1 || layers > 32767 || row_bytes < 1 || row_bytes > (int64_t(1) << 30) || count < 0) {
        return "want 1 to 32767 layers and rows of at least a byte";
    }
    if (!to.keys || !to.values || !from.keys || !from.values || (count && !moves)) {
        return "null pointer";
    }
    for (const chroma_hip_cache_rows* cache : {&to, &from}) {
        if (cache->rows < 1 || cache->rows >= kRows || cache->rows > kBytes / row_bytes) {
            return "a cache's rows are out of range";
        }
        if (cache->layer_pitch < 0 || cache->layer_pitch > kBytes || (layers > 1 && cache->layer_pitch < cache->rows * row_bytes)) {
            return "a cache's layer pitch is smaller than its rows";
        }
    }
    const bool same = to.keys == from.keys && to.values == from.values && (layers == 1 || to.layer_pitch == from.layer_pitch);
    const auto begin = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    const auto bytes = [&](const chroma_hip_cache_rows& c) { return uintptr_t((layers - 1) * c.layer_pitch + c.rows * row_bytes); };
    const auto meet = [&](const void* a, uintptr_t size_a, const void* b, uintptr_t size_b) {
        return begin(a) < begin(b) + size_b && begin(b) < begin(a) + size_a;
    };
    if (meet(to.keys, bytes(to), to.values, bytes(to)) || (same && meet(from.keys, bytes(from), from.values, bytes(from)))) {
        return "keys and values overlap";
    }
    if (!same && (meet(to.keys, bytes(to), from.keys, bytes(from)) || meet(to.keys, bytes(to), from.values, bytes(from)) ||
                  meet(to.values, bytes(to), from.keys, bytes(from)) || meet(to.values, bytes(to), from.values, bytes(from)))) {
        return "caches that overlap must be the same";
    }
    std::vector<Range> ranges;
    ranges.reserve(size_t(count) * (same ? 2 : 1));
    for (int64_t i = 0; i < count; ++i) {
        const int64_t source = moves[3 * i], target = moves[3 * i + 1], rows = moves[3 * i + 2];
        if (source < 0 || target < 0 || rows < 0 || rows > from.rows || source > from.rows - rows || rows > to.rows || target > to.rows - rows) {
            return "a move leaves its cache";
        }
        if (rows) {
            ranges.push_back({target, target + rows, true});
            if (same) {
                ranges.push_back({source, source + rows, false});
            }
        }
    }
    return clash(ranges) ? "a row is written twice, or written and read" : nullptr;
}

int move(const chroma_hip_cache_rows& to, const chroma_hip_cache_rows& from, int64_t layers, int64_t row_bytes, const int64_t* moves,
         int64_t count, hipStream_t stream, char* error, size_t error_size) {
    if (const char* wrong = mistake(to, from, layers, row_bytes, moves, count)) {
        return refuse(wrong, error, error_size);
    }
    Moves all;
    all.source_keys = static_cast<const char*>(from.keys);
    all.source_values = static_cast<const char*>(from.values);
    all.target_keys = static_cast<char*>(to.keys);
    all.target_values = static_cast<char*>(to.values);
    all.source_pitch = uint64_t(from.layer_pitch);
    all.target_pitch = uint64_t(to.layer_pitch);
    all.row_bytes = uint64_t(row_bytes);
    const bool wide = ((reinterpret_cast<uintptr_t>(from.keys) | reinterpret_cast<uintptr_t>(from.values) | reinterpret_cast<uintptr_t>(to.keys) |
                        reinterpret_cast<uintptr_t>(to.values) | (layers > 1 ? all.source_pitch | all.target_pitch : 0u) | all.row_bytes) & 15u) == 0;
    for (int64_t i = 0; i < count;) {
        uint32_t n = 0;
        uint64_t most = 0;
        for (; i < count && n < uint32_t(kMoves); ++i) {
            if (moves[3 * i + 2]) {
                all.move[n++] = {uint32_t(moves[3 * i]), uint32_t(moves[3 * i + 1]), uint32_t(moves[3 * i + 2])};
                most = std::max<uint64_t>(most, uint64_t(moves[3 * i + 2]));
            }
        }
        if (!n) {
            break;
        }
        const uint64_t pieces = (most * all.row_bytes / 16u + kThreads - 1) / kThreads;
        const dim3 grid(unsigned(std::clamp<uint64_t>(pieces, 1u, 4096u)), n, unsigned(2 * layers));
        if (wide) {
            move_rows<true><<<grid, kThreads, 0, stream>>>(all);
        } else {
            move_rows<false><<<grid, kThreads, 0, stream>>>(all);
        }
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) {
            return refuse(hipGetErrorString(status), error, error_size);
        }
    }
    return CHROMA_HIP_OK;
}

}  // namespace

namespace chroma_cache {

int launch_cache_move(const chroma_hip_cache_rows* to, const chroma_hip_cache_rows* from, int64_t layers, int64_t row_bytes,
                      const int64_t* moves, int64_t count, hipStream_t stream, char* error, size_t error_size) {
    if (!to || !from) {
        return refuse("null cache", error, error_size);
    }
    try {
        return move(*to, *from, layers, row_bytes, moves, count, stream, error, error_size);
    } catch (const std::exception& e) {
        return refuse(e.what(), error, error_size);
    }
}

}  // namespace chroma_cache

extern "C" __attribute__((visibility("default"))) int chroma_hip_cache_move(const chroma_hip_cache_rows* to, const chroma_hip_cache_rows* from,
                                                                            int64_t layers, int64_t row_bytes, const int64_t* moves,
                                                                            int64_t count, void* stream, char* error, size_t error_size) {
    return chroma_cache::launch_cache_move(to, from, layers, row_bytes, moves, count, static_cast<hipStream_t>(stream), error, error_size);
}
