// ``chroma_hip_paged_plan``: page tables, slots, positions and row starts of a step from its requests' lengths.
//
// Two running sums over the sequences (new tokens, then the pages that they begin) say where each one's tokens and pages lie.
// Every workgroup takes the sums itself, kSequences of them at a time, and finishes kItems tokens and new pages (there are no
// more new pages than tokens): an item finds its sequence by bisection of the sums in LDS. What bounds it is latency: the
// lengths, two scans, the bisection, a table or free entry, all dependent, in one launch that needs no scratch: 64 sequences of
// one token 5.0 us, 1024 of up to 80 tokens (2 MB written) 7.5.
#include "../../include/chroma_hip.h"

#include <hip/hip_runtime.h>

#include <chroma_hip/device.h>

#include "ranges.h"

#include <algorithm>
#include <cstdint>
#include <cstdio>

namespace {

using Call = chroma_hip_paged_plan_call;

constexpr uint32_t kThreads = 256, kPer = 4, kSequences = kThreads * kPer, kItems = kThreads;

// Inclusive sums of ``v`` over the workgroup's threads, in their order; ``all`` their total.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* scratch, uint64_t& all) {
    const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint64_t before = __shfl_up(static_cast<unsigned long long>(v), step, 64);
        v += lane >= uint32_t(step) ? before : 0u;
    }
    __syncthreads();  // scratch of the last call has been read
    if (lane == 63u) {
        scratch[wave] = v;
    }
    __syncthreads();
    uint64_t before = 0;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64u; ++w) {
        before += w < wave ? scratch[w] : 0u;
        all += scratch[w];
    }
    return v + before;
}

// grid: items / kItems
__global__ void __launch_bounds__(kThreads) plan_step(Call c) {
    // of this chunk's sequences: the token and the new page that each begins with (one entry more: where the chunk ends), its
    // rows and the pages that hold them
    __shared__ uint32_t token_at[kSequences + 1], page_at[kSequences + 1], length_of[kSequences], held_of[kSequences];
    __shared__ uint64_t scratch[kThreads / 64u];
    const uint32_t tokens = uint32_t(c.tokens), page_rows = uint32_t(c.page_rows), item = blockIdx.x * kItems + threadIdx.x;
    const uint64_t room = uint64_t(c.span) * page_rows;  // rows of a sequence
    const int64_t given = c.cursor ? *c.cursor : 0;
    const uint64_t cursor = given < 0 ? 0u : uint64_t(given);
    const auto entry = [&](uint64_t at) -> int64_t { return at < uint64_t(c.free_count) ? c.free_pages[at] : -1; };
    uint64_t counted = 0, taken = 0;  // tokens (all that are asked for) and new pages before the chunk
    for (uint32_t b0 = 0; b0 < uint32_t(c.sequences); b0 += kSequences) {
        const uint32_t here = min(kSequences, uint32_t(c.sequences) - b0);
        uint32_t length[kPer];
        uint64_t count[kPer], sum = 0, all;
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            const uint32_t i = threadIdx.x * kPer + k;
            const int64_t rows = i < here ? c.lengths[b0 + i] : 0, more = i < here ? c.counts[b0 + i] : 0;
            length[k] = rows < 0 ? 0u : uint64_t(rows) > room ? uint32_t(room) : uint32_t(rows);
            count[k] = more < 0 ? 0u : more > c.tokens ? tokens : uint64_t(more);
            sum += count[k];
        }
        uint64_t before = counted + block_scan(sum, scratch, all) - sum;
        counted += all;
        uint32_t held[kPer], wanted[kPer];
        sum = 0;
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            const uint32_t i = threadIdx.x * kPer + k;
            const uint32_t begin = uint32_t(min(before, uint64_t(tokens)));
            before += count[k];
            const uint32_t n = uint32_t(min(before, uint64_t(tokens))) - begin;
            const uint64_t rows = min(uint64_t(length[k]) + n, room);
            held[k] = (length[k] + page_rows - 1u) / page_rows;
            wanted[k] = uint32_t((rows + page_rows - 1u) / page_rows) - held[k];
            sum += wanted[k];
            if (i < here) {
                token_at[i] = begin;
                length_of[i] = length[k];
                held_of[i] = held[k];
                if (blockIdx.x == 0) {
                    c.starts[b0 + i] = begin;
                    if (c.new_lengths) {
                        c.new_lengths[b0 + i] = int64_t(rows);
                    }
                }
            }
        }
        before = block_scan(sum, scratch, all) - sum;
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            const uint32_t i = threadIdx.x * kPer + k;
            if (i < here) {
                page_at[i] = uint32_t(taken + before);
            }
            before += wanted[k];
        }
        if (threadIdx.x == 0) {
            token_at[here] = uint32_t(min(counted, uint64_t(tokens)));
            page_at[here] = uint32_t(taken + all);
        }
        taken += all;
        __syncthreads();
        // the last sequence that begins at the item or before it: the one that holds it, as empty ones begin where the next does
        const auto find = [&](const uint32_t* at) {
            uint32_t low = 0, high = here;
            while (high - low > 1u) {
                const uint32_t middle = (low + high) / 2u;
                (at[middle] <= item ? low : high) = middle;
            }
            return low;
        };
        if (item >= token_at[0] && item < token_at[here]) {
            const uint32_t i = find(token_at), b = b0 + i;
            const uint64_t position = uint64_t(length_of[i]) + (item - token_at[i]);
            int64_t page = -1;
            if (position < room) {
                const uint32_t at = uint32_t(position / page_rows);
                page = at < held_of[i] ? c.table[b * c.table_stride + at] : entry(cursor + page_at[i] + (at - held_of[i]));
            }
            c.slots[item] = page >= 0 && page < c.pages ? page * page_rows + int64_t(position % page_rows) : -1;
            if (c.positions) {
                c.positions[item] = int64_t(position);
            }
            if (c.owners) {
                c.owners[item] = b;
            }
        }
        if (item >= page_at[0] && item < page_at[here]) {
            const uint32_t i = find(page_at);
            c.table[(b0 + i) * c.table_stride + held_of[i] + (item - page_at[i])] = entry(cursor + item);
        }
        __syncthreads();  // the sums have been read
    }
    if (item < tokens && item >= counted) {
        c.slots[item] = -1;
        if (c.positions) {
            c.positions[item] = -1;
        }
        if (c.owners) {
            c.owners[item] = -1;
        }
    }
    if (item == 0) {
        c.starts[c.sequences] = int64_t(min(counted, uint64_t(tokens)));
        *c.taken = int64_t(cursor + taken);
    }
}

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "paged_plan: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

const char* mistake(const Call& c) {
    constexpr int64_t kMost = int64_t(1) << 31, kEntries = int64_t(1) << 40;
    if (c.sequences < 1 || c.sequences > 65535 || c.tokens < 1 || c.tokens > (int64_t(1) << 24)) {
        return "want 1 to 65535 sequences and 1 to 16777216 tokens";
    }
    if (c.pages < 1 || c.pages >= kMost || c.page_rows < 1 || c.page_rows >= kMost || c.span < 1 || c.span >= kMost ||
        c.span * c.page_rows >= kMost) {
        return "pages, page_rows or span out of range";
    }
    if (c.table_stride < c.span || c.table_stride > kEntries || c.free_count < 0 || c.free_count > kEntries) {
        return "a table row is shorter than the span, or an extent out of range";
    }
    if (!c.lengths || !c.counts || !c.table || !c.starts || !c.slots || !c.taken || (c.free_count && !c.free_pages)) {
        return "null device pointer";
    }
    const uint64_t n = uint64_t(c.sequences) * 8u, t = uint64_t(c.tokens) * 8u;
    const chroma_ranges::Range ranges[] = {
        {c.lengths, n, false}, {c.counts, n, false}, {c.free_pages, uint64_t(c.free_count) * 8u, false}, {c.cursor, 8u, false},
        {c.table, (uint64_t(c.sequences - 1) * uint64_t(c.table_stride) + uint64_t(c.span)) * 8u, true}, {c.starts, n + 8u, true},
        {c.slots, t, true}, {c.positions, t, true}, {c.owners, t, true}, {c.new_lengths, n, true}, {c.taken, 8u, true}};
    return chroma_ranges::overlap(ranges) ? "an array that is written overlaps another" : nullptr;
}

}  // namespace

extern "C" __attribute__((visibility("default"))) int chroma_hip_paged_plan(const Call* call, void* stream, char* error, size_t error_size) {
    if (!call) {
        return refuse("null call", error, error_size);
    }
    if (const char* wrong = mistake(*call)) {
        return refuse(wrong, error, error_size);
    }
    plan_step<<<unsigned((call->tokens + kItems - 1) / kItems), kThreads, 0, static_cast<hipStream_t>(stream)>>>(*call);
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? CHROMA_HIP_OK : refuse(hipGetErrorString(status), error, error_size);
}
