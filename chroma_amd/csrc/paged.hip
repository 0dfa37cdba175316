// ``chroma_hip_paged_attention``: attention of one new token per sequence over a paged cache (attention_paged.h) on
// device memory that a caller owns.
#include "../../include/chroma_hip.h"

#include <hip/hip_runtime.h>

#include <chroma_hip/attention_paged.h>

#include <algorithm>
#include <cstdio>
#include <type_traits>

namespace {

using Call = chroma_hip_paged_attention_call;

template <class T, int DP, uint32_t KEYS, uint32_t WAVES>
__global__ void __launch_bounds__(64 * WAVES) paged_attention_whole(chroma::PagedOperands<T> a) {
    chroma::attention_paged_whole<T, DP, KEYS, WAVES>(a);
}

template <class T, int DP, bool STREAM>
__global__ void __launch_bounds__(256) paged_attention_shares(chroma::PagedOperands<T> a, uint32_t ranges, float* scratch) {
    chroma::attention_paged_shares<T, DP, chroma::paged_keys<T, DP>(), STREAM>(a, ranges, scratch);
}

template <class T, int DP, uint32_t WAVES>
__global__ void __launch_bounds__(256) paged_attention_combine(chroma::PagedOperands<T> a, uint32_t ranges, float* scratch) {
    chroma::attention_paged_combine<T, DP, chroma::paged_keys<T, DP>(), WAVES>(a, ranges, scratch);
}

constexpr int64_t kMost = int64_t(1) << 31;  // extents that the kernels count in 32 bits stay below this

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "paged_attention: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

// What is wrong with the call, or null.
const char* mistake(const Call& c) {
    if (c.dtype != CHROMA_HIP_FLOAT32 && c.dtype != CHROMA_HIP_BFLOAT16) {
        return "dtype must be CHROMA_HIP_FLOAT32 or CHROMA_HIP_BFLOAT16";
    }
    if (c.sequences < 1 || c.sequences > 65535 || c.kv_heads < 1 || c.kv_heads > 65535 || c.group < 1 || c.group > 1024) {
        return "want 1 to 65535 sequences and KV heads and 1 to 1024 query heads of a KV head";
    }
    if (c.dim < 8 || c.dim > 256 || c.dim % 8) {
        return "the head dimension must be a multiple of 8 from 8 to 256";
    }
    if (c.pages < 1 || c.pages >= kMost || c.page_rows < 1 || c.page_rows >= kMost || c.longest < 0 || c.longest >= kMost - 4096) {
        return "pages, page_rows or longest out of range";
    }
    if (c.sequences * (c.longest / 16 + 2) >= kMost || c.sequences * c.kv_heads * c.group > (int64_t(1) << 24)) {
        return "more sequences of this length, or more query heads, than the kernels count";
    }
    if (c.window < 0 || c.first < 0) {
        return "window and first must not be negative";
    }
    if ((c.k_new == nullptr) != (c.v_new == nullptr)) {
        return "k_new and v_new come together";
    }
    if (c.table_stride < (c.longest + c.page_rows - 1) / c.page_rows) {
        return "a table row is shorter than the longest sequence's pages";
    }
    const int64_t chunk = c.dtype == CHROMA_HIP_BFLOAT16 ? 8 : 4, heads = c.kv_heads * c.group * c.dim;
    if (c.q_stride < heads || c.out_stride < heads || (c.k_new && c.new_stride < c.kv_heads * c.dim) || c.page_stride < 0 ||
        c.row_stride < c.dim || c.head_stride < 0 || (c.kv_heads > 1 && c.head_stride < c.dim)) {
        return "a stride is smaller than what lies in it";
    }
    if ((c.q_stride | c.out_stride | c.page_stride | c.row_stride | c.head_stride | (c.k_new ? c.new_stride : 0)) % chunk) {
        return "strides must be whole 16-byte chunks";
    }
    return nullptr;
}

template <class T> chroma::PagedOperands<T> operands(const Call& c) {
    chroma::PagedOperands<T> a;
    a.q = static_cast<const T*>(c.q);
    a.k = static_cast<const T*>(c.k_pages);
    a.v = static_cast<const T*>(c.v_pages);
    a.k_new = static_cast<const T*>(c.k_new);
    a.v_new = static_cast<const T*>(c.v_new);
    a.sinks = static_cast<const T*>(c.sinks);
    a.table = c.table;
    a.lengths = c.lengths;
    a.out = static_cast<T*>(c.out);
    a.page_stride = uint64_t(c.page_stride);
    a.row_stride = uint64_t(c.row_stride);
    a.head_stride = uint64_t(c.head_stride);
    a.q_stride = uint64_t(c.q_stride);
    a.new_stride = uint64_t(c.new_stride);
    a.out_stride = uint64_t(c.out_stride);
    a.table_stride = uint64_t(c.table_stride);
    a.pages = uint64_t(c.pages);
    a.page_rows = uint32_t(c.page_rows);
    a.longest = uint32_t(c.longest);
    // a window or first rows past the longest sequence are all of it
    a.window = uint32_t(c.window < kMost ? c.window : kMost - 1);
    a.first = uint32_t(c.first < kMost ? c.first : kMost - 1);
    a.sequences = uint32_t(c.sequences);
    a.kv_heads = uint32_t(c.kv_heads);
    a.group = uint32_t(c.group);
    a.dim = uint32_t(c.dim);
    a.scale = c.scale;
    return a;
}

// Whether a call of these types and head dimension runs on the kernels of padded dimension DP.
template <class T, int DP> bool fits(const Call& c) { return c.dim <= DP && (DP == (sizeof(T) == 2 ? 32 : 16) || c.dim > DP / 2); }

// How a call is cut. Up to kPasses key blocks for every wave of a sequence's workgroup one launch takes whole sequences: 8 KV
// heads of 8 heads of 64, us for whole sequences and for shares: one of 900 rows 8.9 and 11.3, of 1400 10.5 and 10.7, of
// 2000 14.2 and 10.7; 8 mixed ones up to 900 9.1 and 11.8, up to 2000 15.8 and 14.2; 32 up to 900 11.3 and 16.5, up to 2000
// 18.5 and 23.5, up to 4096 36.8 and 34.8; 128 up to 1000 31 and 37, up to 2000 69 and 62. Beyond, all blocks are cut into as
// many shares as bring kWaves waves, those that the chip holds at once: 1024 / 2048 / 4096 waves take 64 sequences of 8192
// 201 / 185 / 192 us and 32 mixed ones up to 4096 37 / 35 / 40.
constexpr int64_t kPasses = 6, kWaves = 2048;
struct Cut {
    int64_t heads, tiles;
    int64_t ranges;  // shares; 0: whole sequences
};
template <class T, int DP> Cut cut_of(const Call& c) {
    Cut cut;
    cut.tiles = (c.group + 15) / 16;
    cut.heads = c.kv_heads * c.group;
    // the most blocks of ``keys`` rows that a sequence can have
    const auto most_blocks = [&](int64_t keys) {
        const int64_t rows = c.longest + 1, blocks = (rows + keys - 1) / keys;
        if (!c.window) {
            return blocks;
        }
        return std::min(blocks + 1, (std::min(c.first, c.longest) + keys - 1) / keys + (std::min(c.window, rows) + keys - 1) / keys);
    };
    const int64_t wanted = (kWaves + c.kv_heads * cut.tiles - 1) / (c.kv_heads * cut.tiles);
    cut.ranges = most_blocks(chroma::paged_whole_keys<T, DP>()) <= kPasses * int64_t(chroma::paged_whole_waves<T, DP>())
                     ? 0
                     : std::min(wanted, c.sequences * most_blocks(chroma::paged_keys<T, DP>()));
    return cut;
}

template <class T, int DP> size_t scratch_bytes(const Call& c) {
    const Cut cut = cut_of<T, DP>(c);
    return cut.ranges ? size_t(cut.ranges + c.sequences) * size_t(cut.heads) * (DP + 2) * sizeof(float) : 0;
}

template <class T, int DP> void launch(const Call& c, float* scratch, hipStream_t stream) {
    const Cut cut = cut_of<T, DP>(c);
    const chroma::PagedOperands<T> a = operands<T>(c);
    if (!cut.ranges) {
        const dim3 grid(unsigned(c.kv_heads * cut.tiles), unsigned(c.sequences));
        constexpr uint32_t keys = chroma::paged_whole_keys<T, DP>(), waves = chroma::paged_whole_waves<T, DP>();
        paged_attention_whole<T, DP, keys, waves><<<grid, 64 * waves, 0, stream>>>(a);
        return;
    }
    const uint32_t ranges = uint32_t(cut.ranges);
    const int64_t waves = cut.ranges * c.kv_heads * cut.tiles;
    if (cut.tiles == 1 && c.dim * sizeof(T) % 128 == 0) {
        paged_attention_shares<T, DP, true><<<unsigned((waves + 3) / 4), 256, 0, stream>>>(a, ranges, scratch);
    } else {
        paged_attention_shares<T, DP, false><<<unsigned((waves + 3) / 4), 256, 0, stream>>>(a, ranges, scratch);
    }
    const int64_t units = c.sequences * cut.heads;
    if (cut.ranges > 32 * c.sequences && units < 2048) {  // many parts and few heads: a workgroup for a head
        paged_attention_combine<T, DP, 4><<<unsigned(units), 256, 0, stream>>>(a, ranges, scratch);
    } else {
        paged_attention_combine<T, DP, 1><<<unsigned((units + 3) / 4), 256, 0, stream>>>(a, ranges, scratch);
    }
}

// f(type, padded dimension) of the call's kernels.
template <class F> auto with_kernels(const Call& c, F f) {
    if (c.dtype == CHROMA_HIP_BFLOAT16) {
        using T = uint16_t;
        return fits<T, 32>(c) ? f(T(), std::integral_constant<int, 32>()) : fits<T, 64>(c) ? f(T(), std::integral_constant<int, 64>())
             : fits<T, 128>(c) ? f(T(), std::integral_constant<int, 128>()) : f(T(), std::integral_constant<int, 256>());
    }
    using T = float;
    return fits<T, 16>(c) ? f(T(), std::integral_constant<int, 16>()) : fits<T, 32>(c) ? f(T(), std::integral_constant<int, 32>())
         : fits<T, 64>(c) ? f(T(), std::integral_constant<int, 64>()) : fits<T, 128>(c) ? f(T(), std::integral_constant<int, 128>())
                                                                                      : f(T(), std::integral_constant<int, 256>());
}

}  // namespace

extern "C" {

__attribute__((visibility("default"))) size_t chroma_hip_paged_attention_workspace(const Call* call) {
    if (!call || mistake(*call)) {
        return 0;
    }
    return with_kernels(*call, [&](auto type, auto dim) { return scratch_bytes<decltype(type), decltype(dim)::value>(*call); });
}

__attribute__((visibility("default"))) int chroma_hip_paged_attention(const Call* call, void* workspace, size_t workspace_bytes, void* stream,
                                                                      char* error, size_t error_size) {
    if (!call) {
        return refuse("null call", error, error_size);
    }
    const Call& c = *call;
    if (const char* wrong = mistake(c)) {
        return refuse(wrong, error, error_size);
    }
    if (!c.q || !c.k_pages || !c.v_pages || !c.lengths || !c.out || (!c.table && c.longest)) {
        return refuse("null device pointer", error, error_size);
    }
    if ((reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.k_pages) | reinterpret_cast<uintptr_t>(c.v_pages) |
         reinterpret_cast<uintptr_t>(c.k_new) | reinterpret_cast<uintptr_t>(c.v_new) | reinterpret_cast<uintptr_t>(c.out)) & 15u) {
        return refuse("q, pages, new rows and out must start on 16 bytes", error, error_size);
    }
    const size_t need = chroma_hip_paged_attention_workspace(call);
    if (need && (!workspace || workspace_bytes < need)) {
        return refuse("workspace smaller than chroma_hip_paged_attention_workspace", error, error_size);
    }
    if (need && (reinterpret_cast<uintptr_t>(workspace) & 15u)) {
        return refuse("the workspace must start on 16 bytes", error, error_size);
    }
    with_kernels(c, [&](auto type, auto dim) {
        launch<decltype(type), decltype(dim)::value>(c, static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
        return 0;
    });
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? CHROMA_HIP_OK : refuse(hipGetErrorString(status), error, error_size);
}

}  // extern "C"
