// ``chroma_hip_cache_store``: new rows of keys and values stored at the slots that a device array holds, in every layer.
//
// A row goes in 16-byte units, one to a thread, so that a wave writes whole lines of it; what its length leaves of the last
// unit goes byte by byte. Row and slot are requested together. What bounds it: a decode step's rows the launch (64 rows of 1 KB
// 2.6 us), a prompt's the memory, each byte read and written once: 8000 rows of 1 KB in 24 layers 124 us, 6.3 TB/s. Nothing is
// read again here, so loads and stores leave the caches to others.
#include "../../include/chroma_hip.h"

#include <hip/hip_runtime.h>

#include "ranges.h"

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <type_traits>

namespace {

using Call = chroma_hip_cache_store_call;

constexpr int kThreads = 256;

typedef uint32_t Aligned __attribute__((ext_vector_type(4)));  // 16 bytes
typedef Aligned Bytes __attribute__((aligned(1)));             // at any address

// grid: (pieces of the units of all rows, layers x keys or values)
template <bool ALIGNED> __global__ void __launch_bounds__(kThreads) store_rows(Call c) {
    using Unit = std::conditional_t<ALIGNED, Aligned, Bytes>;
    const uint64_t layer = blockIdx.y / 2u;
    const char* from = static_cast<const char*>(blockIdx.y % 2u ? c.new_values : c.new_keys) + layer * c.new_layer_pitch;
    char* to = static_cast<char*>(blockIdx.y % 2u ? c.values : c.keys) + layer * c.layer_pitch;
    const uint32_t row_bytes = uint32_t(c.row_bytes), units = row_bytes / 16u, tail = row_bytes % 16u, per_row = units + (tail ? 1u : 0u);
    const uint64_t all = uint64_t(c.count) * per_row;
    for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < all; i += uint64_t(gridDim.x) * kThreads) {
        const uint64_t row = i / per_row;
        const uint32_t unit = uint32_t(i - row * per_row);
        const char* source = from + row * c.new_row_pitch + unit * 16ull;
        const int64_t slot = c.slots[row];
        const bool stored = uint64_t(slot) < uint64_t(c.rows);
        char* target = to + (stored ? slot : 0) * row_bytes + unit * 16ull;
        if (unit < units) {
            const Aligned value = __builtin_nontemporal_load(reinterpret_cast<const Unit*>(source));
            if (stored) {
                __builtin_nontemporal_store(value, reinterpret_cast<Unit*>(target));
            }
        } else if (stored) {
            for (uint32_t k = 0; k < tail; ++k) {
                target[k] = source[k];
            }
        }
    }
}

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "cache_store: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

const char* mistake(const Call& c) {
    constexpr int64_t kRows = int64_t(1) << 32, kBytes = int64_t(1) << 46;
    if (c.layers < 1 || c.layers > 32767 || c.row_bytes < 1 || c.row_bytes > (int64_t(1) << 30)) {
        return "want 1 to 32767 layers and rows of 1 to 1073741824 bytes";
    }
    if (c.rows < 1 || c.rows >= kRows || c.rows > kBytes / c.row_bytes || c.count < 0 || c.count >= kRows || c.count > kBytes / c.row_bytes) {
        return "rows or count out of range";
    }
    if (c.layer_pitch < 0 || c.layer_pitch > kBytes || c.new_layer_pitch < 0 || c.new_layer_pitch > kBytes || c.new_row_pitch < 0 ||
        c.new_row_pitch > kBytes || (c.count && c.new_row_pitch > kBytes / c.count)) {
        return "a pitch is out of range";
    }
    if ((c.layers > 1 && c.layer_pitch < c.rows * c.row_bytes) || (c.count > 1 && c.new_row_pitch < c.row_bytes)) {
        return "a pitch is smaller than what lies in it";
    }
    if (!c.keys || !c.values || (c.count && (!c.new_keys || !c.new_values || !c.slots))) {
        return "null device pointer";
    }
    if (!c.count) {
        return nullptr;
    }
    const uint64_t held = uint64_t((c.layers - 1) * c.layer_pitch + c.rows * c.row_bytes);
    const uint64_t fresh = uint64_t((c.layers - 1) * c.new_layer_pitch + (c.count - 1) * c.new_row_pitch + c.row_bytes);
    const chroma_ranges::Range ranges[] = {{c.keys, held, true}, {c.values, held, true}, {c.new_keys, fresh, false},
                                           {c.new_values, fresh, false}, {c.slots, uint64_t(c.count) * 8u, false}};
    return chroma_ranges::overlap(ranges) ? "the cache's keys or values overlap another array" : nullptr;
}

}  // namespace

extern "C" __attribute__((visibility("default"))) int chroma_hip_cache_store(const Call* call, void* stream, char* error, size_t error_size) {
    if (!call) {
        return refuse("null call", error, error_size);
    }
    const Call& c = *call;
    if (const char* wrong = mistake(c)) {
        return refuse(wrong, error, error_size);
    }
    if (!c.count) {
        return CHROMA_HIP_OK;
    }
    const uint64_t addresses = reinterpret_cast<uintptr_t>(c.keys) | reinterpret_cast<uintptr_t>(c.values) | reinterpret_cast<uintptr_t>(c.new_keys) |
                               reinterpret_cast<uintptr_t>(c.new_values) | uint64_t(c.row_bytes) | (c.count > 1 ? uint64_t(c.new_row_pitch) : 0u) |
                               (c.layers > 1 ? uint64_t(c.layer_pitch | c.new_layer_pitch) : 0u);
    const uint64_t pieces = (uint64_t(c.count) * uint64_t((c.row_bytes + 15) / 16) + kThreads - 1) / kThreads;
    const dim3 grid(unsigned(std::min<uint64_t>(pieces, 1u << 20)), unsigned(2 * c.layers));
    if (addresses & 15u) {
        store_rows<false><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(c);
    } else {
        store_rows<true><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(c);
    }
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? CHROMA_HIP_OK : refuse(hipGetErrorString(status), error, error_size);
}
