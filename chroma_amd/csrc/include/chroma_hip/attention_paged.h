// Attention of one new token per sequence over keys and values in pages:
//
//     o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m)),   s_j = scale * (q . k_j),
//
// j over the cached rows that the sequence's page table holds and its window leaves, and the new row. Scores, sums and
// products stay in float; the result is rounded once.
#pragma once

#include "attention_flash.h"

namespace chroma {

// Row j < length of sequence b lies at row j % page_rows of page table[b][j / page_rows]; the new row, if any, is
// position ``length``. Strides count elements.
template <class T> struct PagedOperands {
    const T* q;
    const T* k;
    const T* v;
    const T* k_new;  // null: no new row
    const T* v_new;
    const T* sinks;  // null: no sink
    const int64_t* table;
    const int64_t* lengths;
    T* out;
    uint64_t page_stride, row_stride, head_stride, q_stride, new_stride, out_stride, table_stride;
    uint64_t pages;
    uint32_t page_rows, longest, window, first;
    uint32_t kv_heads, group, dim;
    float scale;
};

// The rows a sequence's token sees: [0, head) and [low, end), the new row (position ``length``) among the latter.
struct PagedRange {
    uint32_t length, head, low, end;
};

template <class T> __device__ __forceinline__ PagedRange paged_range(const PagedOperands<T>& a, uint32_t b) {
    const int64_t given = a.lengths[b];
    PagedRange r;
    r.length = given < 0 ? 0u : given > int64_t(a.longest) ? a.longest : uint32_t(given);
    const uint32_t fresh = a.k_new ? 1u : 0u;
    r.end = r.length + fresh;
    // the token's position is end - 1; the cached rows after end - 1 - window are in its window (the new row always is)
    r.low = a.window && r.end > a.window ? r.end - a.window : 0u;
    r.head = a.first < r.low ? a.first : r.low;
    return r;
}

template <class T> __device__ __forceinline__ float paged_widen(T v) {
    if constexpr (sizeof(T) == 2) {
        return bf16_to_f32(v);
    } else {
        return v;
    }
}

// The kernel is the few-query one of attention_flash.h for one query and rows found through the table: a tile is 16 query
// heads of a KV head, a workgroup's 4 waves take key blocks in turn, and ``splits`` workgroups share a sequence's blocks,
// joined by ``attention_paged_combine``. A wave copies its block of K and V global -> LDS into buffers of its own (no
// barrier in the loop); lane l finds row l of the block once, and the lanes that copy it receive its place by a shuffle.
// DP is the head dimension in whole matrix-core operands; what lies past ``dim`` in a row is zero.
//
// Rows that are not seen keep their probability at exactly 0 and their values out of the products, so that they may hold
// anything. A bfloat16 probability meets V as two bfloat16 halves (2^-16 of it is lost): the products are a small part of
// the time, and one half alone (2^-9) would add as much error as the result's own rounding.
constexpr uint32_t kPagedWaves = 4;

template <class T, int DP> constexpr uint32_t paged_keys() {  // keys of a block: 16 KiB of K and V, a multiple of an operand
    constexpr uint32_t fits = 16384u / (2u * DP * sizeof(T)), least = sizeof(T) == 2 ? 32u : 16u;
    return fits > 64u ? 64u : fits < least ? least : fits;
}

// Floats of one (sequence, KV head, 16 query heads, split): per row the maximum and the sum, then the DP sums of p . v.
template <int DP> constexpr uint32_t paged_partial_floats() { return 16u * (DP + 2u); }

template <class T> __device__ __forceinline__ void paged_store4(T* to, const f32x4_t& v) {
    if constexpr (sizeof(T) == 2) {
        const uint32_t lo = f32_to_bf16(v[0]) | (uint32_t(f32_to_bf16(v[1])) << 16), hi = f32_to_bf16(v[2]) | (uint32_t(f32_to_bf16(v[3])) << 16);
        *reinterpret_cast<uint2*>(to) = uint2{lo, hi};
    } else {
        *reinterpret_cast<f32x4_t*>(to) = v;
    }
}

// grid: (KV heads, row tiles x splits, sequences), 256 threads
template <class T, int DP>
__device__ __forceinline__ void attention_paged(const PagedOperands<T>& a, uint32_t splits, float* __restrict__ partial) {
    constexpr bool BF16 = sizeof(T) == 2;
    constexpr uint32_t KEYS = paged_keys<T, DP>(), CHUNK = 16u / sizeof(T), PER_ROW = DP / CHUNK;
    constexpr uint32_t WAVE = 2u * KEYS * DP, OPAD = DP + 4u;
    constexpr int COPIES = KEYS * DP * sizeof(T) / 1024, PARTS = PER_ROW / 4u, TILES = KEYS / 16;
    constexpr uint32_t SWZ = PER_ROW % 8u == 0 ? 7u : 3u;  // chunk c of row r lies at c ^ ((r / 2) & SWZ)
    static_assert(PER_ROW % 4u == 0 && 64u % PER_ROW == 0 && 16u * (OPAD + 2u) * 4u <= WAVE * sizeof(T), "head dimension");
    __shared__ __attribute__((aligned(1024))) T lds[kPagedWaves * WAVE];
    const uint32_t lane = threadIdx.x % 64u, quad = lane / 16u, col = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t kv = blockIdx.x, tile = blockIdx.y / splits, split = blockIdx.y % splits, b = blockIdx.z;
    const uint32_t row0 = tile * 16u, chunks = a.dim / CHUNK;
    const float neg_inf = -__builtin_inff();
    T* ks = lds + wave * WAVE;
    T* vs = ks + KEYS * DP;
    const PagedRange range = paged_range(a, b);
    const T* q = a.q + b * a.q_stride + uint64_t(kv * a.group + (row0 + col < a.group ? row0 + col : a.group - 1u)) * a.dim;
    const T* k_new = a.k_new + b * a.new_stride + uint64_t(kv) * a.dim;
    const T* v_new = a.v_new + b * a.new_stride + uint64_t(kv) * a.dim;
    const T* k_pages = a.k + kv * a.head_stride;
    const T* v_pages = a.v + kv * a.head_stride;
    const int64_t* table = a.table + b * a.table_stride;
    uint4 qf[PARTS];
#pragma unroll
    for (int c = 0; c < PARTS; ++c) {
        qf[c] = uint4{0u, 0u, 0u, 0u};
        if (c * 4u + quad < chunks) {
            qf[c] = *reinterpret_cast<const uint4*>(q + (c * 4u + quad) * CHUNK);
        }
    }
    if (chunks < PER_ROW) {
        for (uint32_t c = lane; c < 2u * KEYS * PER_ROW; c += 64u) {
            *reinterpret_cast<uint4*>(ks + c * CHUNK) = uint4{0u, 0u, 0u, 0u};
        }
        __builtin_amdgcn_s_waitcnt(0);  // before copies into the same places
    }

    // Blocks: the first rows', then those from range.low on; this wave's are first, first + stride, ...
    const uint32_t head_blocks = (range.head + KEYS - 1u) / KEYS, blocks = head_blocks + (range.end - range.low + KEYS - 1u) / KEYS;
    const uint32_t stride = kPagedWaves * splits;
    auto block_begin = [&](uint32_t n) { return n < head_blocks ? n * KEYS : range.low + (n - head_blocks) * KEYS; };
    auto block_end = [&](uint32_t n) { return n < head_blocks ? range.head : range.end; };
    // The page of this lane's row of block n (-1: none).
    auto page_of = [&](uint32_t n) -> int64_t {
        const uint32_t j = block_begin(n) + lane;
        return lane < KEYS && j < block_end(n) && j < range.length ? table[j / a.page_rows] : -1;
    };
    unsigned long long seen = 0;
    auto copy = [&](uint32_t n, int64_t page) {
        const uint32_t begin = block_begin(n), j = begin + lane;
        const bool held = page >= 0 && uint64_t(page) < a.pages;
        const uint64_t place = held ? uint64_t(page) * a.page_stride + uint64_t(j % a.page_rows) * a.row_stride : 0u;
        seen = __ballot(held || (lane < KEYS && j >= range.length && j < block_end(n)));
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const uint32_t r = i * (64u / PER_ROW) + lane / PER_ROW, chunk = (lane % PER_ROW) ^ ((r / 2u) & SWZ);
            const uint64_t from = __shfl(place, r, kWave);
            const bool fresh = begin + r == range.length && range.end > range.length;
            const T* k = (fresh ? k_new : k_pages + from) + chunk * CHUNK;
            const T* v = (fresh ? v_new : v_pages + from) + chunk * CHUNK;
            if (chunk < chunks) {
                __builtin_amdgcn_global_load_lds((global_void*)k, (lds_void*)(ks + i * (1024u / sizeof(T))), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((global_void*)v, (lds_void*)(vs + i * (1024u / sizeof(T))), 16, 0, 0);
            }
        }
    };

    float peak = neg_inf, total = 0.0f;
    f32x4_t o[DP / 16];
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) {
        o[dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    uint32_t n = split * kPagedWaves + wave;
    if (n < blocks) {
        copy(n, page_of(n));
    }
    while (n < blocks) {
        const uint32_t next = n + stride;
        int64_t next_page = -1;
        if (next < blocks) {
            next_page = page_of(next);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(vmcnt_wait(0));
        __builtin_amdgcn_sched_barrier(0);
        if (seen != (KEYS == 64u ? ~0ull : (1ull << (KEYS % 64u)) - 1ull)) {  // 0 times an infinite value would be NaN
            for (uint32_t c = lane; c < KEYS * PER_ROW; c += 64u) {
                if (!((seen >> (c / PER_ROW)) & 1ull)) {
                    *reinterpret_cast<uint4*>(vs + c * CHUNK) = uint4{0u, 0u, 0u, 0u};
                }
            }
        }
        // scores of keys 16 t + 4 quad + r for this lane's query head
        float u[TILES][4], top = neg_inf;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < PARTS; ++c) {
                const uint32_t r = t * 16u + col;
                const uint4 kf = *reinterpret_cast<const uint4*>(ks + r * DP + ((c * 4u + quad) ^ ((r / 2u) & SWZ)) * CHUNK);
                if constexpr (BF16) {
                    kwave_mfma<T>(kf, qf[c], s);
                } else {
                    s += kwave_unit(kf, qf[c]);
                }
            }
            const uint32_t bits = uint32_t(seen >> (t * 16u + quad * 4u)) & 15u;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u[t][r] = (bits >> r) & 1u ? s[r] * a.scale : neg_inf;
                top = __builtin_fmaxf(top, u[t][r]);
            }
        }
        if (__ballot(top > peak + kFlashHeadroom || (peak == neg_inf && top != neg_inf)) != 0ull) {
            top = __builtin_fmaxf(top, __shfl_xor(top, 16, kWave));
            top = __builtin_fmaxf(top, __shfl_xor(top, 32, kWave));
            top = __builtin_fmaxf(top, peak);
            const float shrink = peak == neg_inf ? 0.0f : fast_exp(peak - top);
            total *= shrink;
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt) {
                o[dt] *= shrink;
            }
            peak = top;
        }
        const float base = peak == neg_inf ? 0.0f : peak;
        float part = 0.0f;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u[t][r] = fast_exp(u[t][r] - base);
                part += u[t][r];
            }
        }
        total += part;
        if constexpr (BF16) {
            // slots 0-3 and 4-7 of lane (d, quad) hold keys 32 h + 4 quad + r and 32 h + 16 + 4 quad + r (attention_flash.h)
#pragma unroll
            for (int h = 0; h < TILES / 2; ++h) {
                bf16x8_t high, low;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const float p = u[2 * h + x / 4][x % 4];
                    high[x] = __bf16(p);
                    low[x] = __bf16(p - float(high[x]));
                }
#pragma unroll
                for (int dt = 0; dt < DP / 16; ++dt) {
                    s16x4_t half[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t r = h * 32u + x * 16u + quad * 4u + col / 4u;
                        const uint32_t chunk = (dt * 2u + (col % 4u) / 2u) ^ ((r / 2u) & SWZ);
                        half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + r * DP + chunk * 8u + (col % 2u) * 4u));
                    }
                    const uint2 lo = __builtin_bit_cast(uint2, half[0]), hi = __builtin_bit_cast(uint2, half[1]);
                    const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, uint4{lo.x, lo.y, hi.x, hi.y});
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, high, o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, low, o[dt], 0, 0, 0);
                }
            }
        } else {
            // product (t, r) takes keys 16 t + 4 quad + r; 16 keys are summed before they join the row's
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
#pragma unroll
                for (int dt = 0; dt < DP / 16; ++dt) {
                    f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t key = t * 16u + quad * 4u + r;
                        const float v = vs[key * DP + ((dt * 4u + col / 4u) ^ ((key / 2u) & SWZ)) * 4u + col % 4u];
                        sum = __builtin_amdgcn_mfma_f32_16x16x4f32(v, u[t][r], sum, 0, 0, 0);
                    }
                    o[dt] += sum;
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (next < blocks) {  // both buffers have been read
            copy(next, next_page);
        }
        n = next;
    }

    // The waves' parts: rows of (DP + 4) floats in each wave's own buffers, then [row][max, sum].
    total += __shfl_xor(total, 16, kWave);
    total += __shfl_xor(total, 32, kWave);
    float* mine = reinterpret_cast<float*>(ks);
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) {
        *reinterpret_cast<f32x4_t*>(mine + col * OPAD + dt * 16u + quad * 4u) = o[dt];
    }
    if (quad == 0) {
        mine[16u * OPAD + 2u * col] = peak;
        mine[16u * OPAD + 2u * col + 1u] = total;
    }
    __syncthreads();
    const float* parts = reinterpret_cast<const float*>(lds);
    constexpr uint32_t PART = WAVE * sizeof(T) / 4u;
    for (uint32_t i = threadIdx.x; i < 16u * (DP / 4u); i += 64u * kPagedWaves) {
        const uint32_t r = i / (DP / 4u), d = i % (DP / 4u) * 4u;
        if (row0 + r >= a.group || d >= a.dim) {
            continue;
        }
        const uint32_t head = kv * a.group + row0 + r;
        const float sink = splits == 1u && a.sinks ? paged_widen<T>(a.sinks[head]) : neg_inf;
        FlashMerge merge{sink, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < kPagedWaves; ++w) {
            merge.top = __builtin_fmaxf(merge.top, parts[w * PART + 16u * OPAD + 2u * r]);
        }
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < kPagedWaves; ++w) {
            const float scale = merge.weight(parts[w * PART + 16u * OPAD + 2u * r]);
            merge.total += scale * parts[w * PART + 16u * OPAD + 2u * r + 1u];
            sum += scale * *reinterpret_cast<const f32x4_t*>(parts + w * PART + r * OPAD + d);
        }
        if (splits == 1u) {
            merge.total += merge.weight(sink);
            sum *= merge.total == 0.0f ? 0.0f : 1.0f / merge.total;
            paged_store4<T>(a.out + b * a.out_stride + uint64_t(head) * a.dim + d, sum);
        } else {
            float* to = partial + (uint64_t(b * gridDim.x + kv) * gridDim.y + blockIdx.y) * paged_partial_floats<DP>();
            *reinterpret_cast<f32x4_t*>(to + 32u + r * DP + d) = sum;
            if (d == 0) {
                to[2u * r] = merge.top;
                to[2u * r + 1u] = merge.total;
            }
        }
    }
}

// The splits of every row, in order, and the sink (grid: KV heads x row tiles x sequences, 256 threads).
template <class T, int DP>
__device__ __forceinline__ void attention_paged_combine(const PagedOperands<T>& a, uint32_t splits, const float* __restrict__ partial) {
    constexpr uint32_t PART = paged_partial_floats<DP>();
    const uint32_t kv = blockIdx.x, row0 = blockIdx.y * 16u, b = blockIdx.z;
    const float* parts = partial + (uint64_t(b * gridDim.x + kv) * gridDim.y + blockIdx.y) * splits * PART;
    for (uint32_t i = threadIdx.x; i < 16u * (DP / 4u); i += 256u) {
        const uint32_t r = i / (DP / 4u), d = i % (DP / 4u) * 4u;
        if (row0 + r >= a.group || d >= a.dim) {
            continue;
        }
        const uint32_t head = kv * a.group + row0 + r;
        const float sink = a.sinks ? paged_widen<T>(a.sinks[head]) : -__builtin_inff();
        FlashMerge merge{sink, 0.0f};
        for (uint32_t s = 0; s < splits; ++s) {
            merge.top = __builtin_fmaxf(merge.top, parts[s * PART + 2u * r]);
        }
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t s = 0; s < splits; ++s) {
            const float scale = merge.weight(parts[s * PART + 2u * r]);
            merge.total += scale * parts[s * PART + 2u * r + 1u];
            sum += scale * *reinterpret_cast<const f32x4_t*>(parts + s * PART + 32u + r * DP + d);
        }
        merge.total += merge.weight(sink);
        sum *= merge.total == 0.0f ? 0.0f : 1.0f / merge.total;
        paged_store4<T>(a.out + b * a.out_stride + uint64_t(head) * a.dim + d, sum);
    }
}

}  // namespace chroma
