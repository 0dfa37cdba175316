// ``chroma_hip_paged_chunk_attention``: attention of a chunk of new tokens of every sequence over a paged cache
// (attention_chunk.h) on device memory that a caller owns.
#include "../../include/chroma_hip.h"

#include <hip/hip_runtime.h>

#include <chroma_hip/attention_chunk.h>

#include "ranges.h"

#include <algorithm>
#include <cstdio>
#include <type_traits>

namespace {

using Call = chroma_hip_paged_chunk_call;

template <class T, int DP, uint32_t KEYS, uint32_t WAVES>
__global__ void __launch_bounds__(64 * WAVES) paged_chunk_tiles(chroma::ChunkOperands<T> a, uint32_t splits, float* scratch) {
    chroma::attention_chunk_tiles<T, DP, KEYS, WAVES>(a, splits, scratch);
}

// (two waves a SIMD, or three with heads up to 64)
template <int DP, uint32_t KEYS, uint32_t WAVES, bool FULL>
__global__ void __launch_bounds__(64 * WAVES, DP <= 64 ? 3 : DP == 256 ? 1 : 2) paged_chunk_wide(chroma::ChunkOperands<uint16_t> a, uint32_t splits,
                                                                                                 float* scratch) {
    chroma::attention_chunk_wide<DP, KEYS, WAVES, FULL>(a, splits, scratch);
}

template <class T, int DP, uint32_t ROWS, bool LOG2>
__global__ void __launch_bounds__(256) paged_chunk_combine(chroma::ChunkOperands<T> a, uint32_t splits, float* scratch) {
    chroma::attention_chunk_combine<T, DP, ROWS, LOG2>(a, splits, scratch);
}

constexpr int64_t kMost = int64_t(1) << 31;  // extents that the kernels count in 32 bits stay below this

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "paged_chunk_attention: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

// What is wrong with the call's extents, or null.
const char* mistake(const Call& c) {
    if (c.dtype != CHROMA_HIP_FLOAT32 && c.dtype != CHROMA_HIP_BFLOAT16) {
        return "dtype must be CHROMA_HIP_FLOAT32 or CHROMA_HIP_BFLOAT16";
    }
    if (c.sequences < 1 || c.sequences > 65535 || c.kv_heads < 1 || c.kv_heads > 65535 || c.group < 1 || c.group > 1024) {
        return "want 1 to 65535 sequences and KV heads and 1 to 1024 query heads of a KV head";
    }
    if (c.tokens < 1 || c.tokens > (int64_t(1) << 24)) {
        return "want 1 to 16777216 tokens";
    }
    if (c.dim < 8 || c.dim > 256 || c.dim % 8) {
        return "the head dimension must be a multiple of 8 from 8 to 256";
    }
    if (c.pages < 1 || c.pages >= kMost || c.page_rows < 1 || c.page_rows >= kMost || c.longest < 0 || c.longest >= kMost - 4096 - c.tokens) {
        return "pages, page_rows or longest out of range";
    }
    // (a launch holds fewer than 2^32 threads: the most tiles, 2^22 full ones and 2^22 sequences' last ones, have 512 each)
    if (c.tokens * c.kv_heads * c.group >= (int64_t(1) << 26) || c.sequences * c.kv_heads > (int64_t(1) << 22)) {
        return "more query rows, or KV heads of sequences, than the kernels count";
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
    constexpr int64_t kStride = int64_t(1) << 40;
    const int64_t chunk = c.dtype == CHROMA_HIP_BFLOAT16 ? 8 : 4, heads = c.kv_heads * c.group * c.dim;
    if (c.table_stride > kStride || c.q_stride > kStride || c.out_stride > kStride || c.new_stride > kStride || c.page_stride > kStride ||
        c.row_stride > kStride || c.head_stride > kStride) {
        return "a stride is out of range";
    }
    if (c.q_stride < heads || c.out_stride < heads || (c.k_new && c.new_stride < c.kv_heads * c.dim) || c.page_stride < 0 ||
        c.row_stride < c.dim || c.head_stride < 0 || (c.kv_heads > 1 && c.head_stride < c.dim)) {
        return "a stride is smaller than what lies in it";
    }
    if ((c.q_stride | c.out_stride | c.page_stride | c.row_stride | c.head_stride | (c.k_new ? c.new_stride : 0)) % chunk) {
        return "strides must be whole 16-byte chunks";
    }
    return nullptr;
}

template <class T> chroma::ChunkOperands<T> operands(const Call& c) {
    chroma::ChunkOperands<T> a;
    a.q = static_cast<const T*>(c.q);
    a.k = static_cast<const T*>(c.k_pages);
    a.v = static_cast<const T*>(c.v_pages);
    a.k_new = static_cast<const T*>(c.k_new);
    a.v_new = static_cast<const T*>(c.v_new);
    a.sinks = static_cast<const T*>(c.sinks);
    a.table = c.table;
    a.lengths = c.lengths;
    a.starts = c.starts;
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
    a.tokens = uint32_t(c.tokens);
    a.kv_heads = uint32_t(c.kv_heads);
    a.group = uint32_t(c.group);
    a.dim = uint32_t(c.dim);
    a.scale = c.scale;
    return a;
}

// Whether a call of these types and head dimension runs on the kernels of padded dimension DP.
template <class T, int DP> bool fits(const Call& c) { return c.dim <= DP && (DP == (sizeof(T) == 2 ? 32 : 16) || c.dim > DP / 2); }

// How a call is cut: tiles of 32 rows a wave (``waves`` 4 or 8, bfloat16) or of 16 rows (``waves`` 0), at most this many of all
// sequences, and workgroups for each of them.
struct Cut {
    int waves;
    int64_t tiles, splits;
    int64_t rows() const { return waves ? 32 * waves : 16; }
};

// Measured with 8 KV heads of 8 heads of 64 (D 64) or of 4 of 128 (D 128), in microseconds:
//
// The 16-row tiles have eight waves share a tile's keys: quick where there are few rows, while the tiles of 128 rows read each
// key 8 times less often. 32 tokens over 900 rows 12.5 (16 rows) and 19.8 (128 rows), over 8000 33 and 25; 64 over 2000 20 and
// 20, over 8000 54 and 32; 256 over 900 35 and 22; 32 sequences of 16 over 2000 100 and 52; but below 64 rows a sequence most of
// a large tile is empty: 32 of 4 tokens over 2000 31 and 39. D 128, 64 tokens over 2000: 21 and 25; 32 over
// 16000 58 and 54.
// Eight waves a tile read the keys half as often, once tiles are many: D 128, 2 x 2048 tokens over 4000 419 with four and 378;
// 512 over 900 37 with four and 52. With D 64 they gain nothing.
//
// Keys are split for 512 workgroups (with 256, 8 x 32 tokens over 2000 take 41 instead of 35; with 1024, D 128, 4 x 512 over 900
// 97 instead of 72), but not into so little that the second launch costs more: five blocks of a large tile (256 over 900 in
// three parts 24, in four 22), two blocks a wave of a small one and at most 32 parts (one token over 30000 rows, 58 parts 40,
// 32 parts 31), no parts for 256 small tiles or more (64 over 900 in two 16, in one 13), and with D 128, whose parts are
// larger, four blocks a wave where there are 256 workgroups (64 over 2000 in four 25, in two 20).
template <class T, int DP> Cut cut_of(const Call& c) {
    constexpr int64_t wide = chroma::chunk_wide_keys<DP>(), few = chroma::paged_whole_keys<T, DP>(), few_waves = chroma::paged_whole_waves<T, DP>();
    Cut cut;
    const auto tiles_of = [&](int64_t rows) { return c.tokens * c.group / rows + std::min(c.sequences, c.tokens); };
    const int64_t rows = c.longest + (c.k_new ? c.tokens : 0);
    const auto most_blocks = [&](int64_t keys) {
        const int64_t blocks = (rows + keys - 1) / keys + 1;
        return c.window ? std::min(blocks, (std::min(c.first, rows) + std::min(c.window, rows)) / keys + 3) : blocks;
    };
    const int64_t heads = c.tokens * c.group * c.kv_heads;
    cut.waves = sizeof(T) != 2 || c.tokens * c.group < 64 * c.sequences || (heads < 128 * 64 && heads * most_blocks(wide) * wide < 10000000) ? 0
              : DP == 128 && tiles_of(256) * c.kv_heads >= 512 ? 8 : 4;
    cut.tiles = tiles_of(cut.rows());
    const int64_t units = cut.tiles * c.kv_heads, wanted = (512 + units - 1) / units, rounds = most_blocks(few) / few_waves;
    const int64_t most = cut.waves ? most_blocks(wide) / 5
                       : units >= 256 ? 1
                       : DP < 128 ? std::min<int64_t>(rounds / 2, 32) : std::max(std::min(256 / units, rounds / 2), (rounds + 2) / 4);
    cut.splits = std::max<int64_t>(1, std::min(wanted, most));
    return cut;
}

template <class T, int DP> size_t scratch_bytes(const Call& c) {
    const Cut cut = cut_of<T, DP>(c);
    return cut.splits > 1 ? size_t(cut.tiles * c.kv_heads * cut.splits) * size_t(cut.rows() * (DP + 2)) * sizeof(float) : 0;
}

template <int DP, uint32_t WAVES, bool FULL, class A> void launch_wide(const A& a, dim3 grid, float* scratch, hipStream_t stream) {
    paged_chunk_wide<DP, chroma::chunk_wide_keys<DP>(), WAVES, FULL><<<grid, 64 * WAVES, 0, stream>>>(a, grid.y, scratch);
}

template <class T, int DP> void launch(const Call& c, float* scratch, hipStream_t stream) {
    const Cut cut = cut_of<T, DP>(c);
    const chroma::ChunkOperands<T> a = operands<T>(c);
    const dim3 grid(unsigned(cut.tiles * c.kv_heads), unsigned(cut.splits));
    const auto combine = [&](auto kernel) { kernel<<<dim3(grid.x, unsigned(cut.rows() / 16)), 256, 0, stream>>>(a, grid.y, scratch); };
    if constexpr (sizeof(T) == 2) {
        if constexpr (DP == 128) {
            if (cut.waves == 8) {  // (512 workgroups or more: never split)
                c.dim == DP ? launch_wide<DP, 8, true>(a, grid, scratch, stream) : launch_wide<DP, 8, false>(a, grid, scratch, stream);
                return;
            }
        }
        if (cut.waves) {
            c.dim == DP ? launch_wide<DP, 4, true>(a, grid, scratch, stream) : launch_wide<DP, 4, false>(a, grid, scratch, stream);
            if (grid.y > 1) {
                combine(paged_chunk_combine<T, DP, 128u, true>);
            }
            return;
        }
    }
    constexpr uint32_t keys = chroma::paged_whole_keys<T, DP>(), waves = chroma::paged_whole_waves<T, DP>();
    paged_chunk_tiles<T, DP, keys, waves><<<grid, 64 * waves, 0, stream>>>(a, grid.y, scratch);
    if (grid.y > 1) {
        combine(paged_chunk_combine<T, DP, 16u, false>);
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

__attribute__((visibility("default"))) size_t chroma_hip_paged_chunk_attention_workspace(const Call* call) {
    if (!call || mistake(*call)) {
        return 0;
    }
    return with_kernels(*call, [&](auto type, auto dim) { return scratch_bytes<decltype(type), decltype(dim)::value>(*call); });
}

__attribute__((visibility("default"))) int chroma_hip_paged_chunk_attention(const Call* call, void* workspace, size_t workspace_bytes,
                                                                            void* stream, char* error, size_t error_size) {
    if (!call) {
        return refuse("null call", error, error_size);
    }
    const Call& c = *call;
    if (const char* wrong = mistake(c)) {
        return refuse(wrong, error, error_size);
    }
    if (!c.q || !c.k_pages || !c.v_pages || !c.lengths || !c.starts || !c.out || (!c.table && c.longest)) {
        return refuse("null device pointer", error, error_size);
    }
    if ((reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.k_pages) | reinterpret_cast<uintptr_t>(c.v_pages) |
         reinterpret_cast<uintptr_t>(c.k_new) | reinterpret_cast<uintptr_t>(c.v_new) | reinterpret_cast<uintptr_t>(c.out)) & 15u) {
        return refuse("q, pages, new rows and out must start on 16 bytes", error, error_size);
    }
    const size_t need = chroma_hip_paged_chunk_attention_workspace(call);
    if (need && (!workspace || workspace_bytes < need)) {
        return refuse("workspace smaller than chroma_hip_paged_chunk_attention_workspace", error, error_size);
    }
    if (need && (reinterpret_cast<uintptr_t>(workspace) & 15u)) {
        return refuse("the workspace must start on 16 bytes", error, error_size);
    }
    using chroma_ranges::bytes_of;
    const uint64_t size = c.dtype == CHROMA_HIP_BFLOAT16 ? 2 : 4;
    const int64_t row = c.kv_heads * c.group * c.dim;
    const uint64_t new_bytes = bytes_of({{c.tokens, c.new_stride}, {c.kv_heads * c.dim, 1}}, size);
    const uint64_t page_bytes = bytes_of({{c.pages, c.page_stride}, {c.page_rows, c.row_stride}, {c.kv_heads, c.head_stride}, {c.dim, 1}}, size);
    const int64_t span = (c.longest + c.page_rows - 1) / c.page_rows;
    const chroma_ranges::Range ranges[] = {
        {c.out, bytes_of({{c.tokens, c.out_stride}, {row, 1}}, size), true}, {workspace, need, true},
        {c.q, bytes_of({{c.tokens, c.q_stride}, {row, 1}}, size), false}, {c.k_pages, page_bytes, false}, {c.v_pages, page_bytes, false},
        {c.k_new, new_bytes, false}, {c.v_new, new_bytes, false}, {c.sinks, uint64_t(c.kv_heads * c.group) * size, false},
        {c.table, span ? bytes_of({{c.sequences, c.table_stride}, {span, 1}}, 8) : 0, false},
        {c.starts, uint64_t(c.sequences + 1) * 8u, false}, {c.lengths, uint64_t(c.sequences) * 8u, false}};
    if (chroma_ranges::overlap(ranges)) {
        return refuse("out or the workspace overlaps another array", error, error_size);
    }
    with_kernels(c, [&](auto type, auto dim) {
        launch<decltype(type), decltype(dim)::value>(c, static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
        return 0;
    });
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? CHROMA_HIP_OK : refuse(hipGetErrorString(status), error, error_size);
}

}  // extern "C"
