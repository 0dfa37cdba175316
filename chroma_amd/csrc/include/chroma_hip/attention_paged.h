// Attention of one new token per sequence over keys and values in pages:
//
//     o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m)),   s_j = scale * (q . k_j),
//
// j over the cached rows that the sequence's page table holds and its window leaves, and the new row. Scores, sums and
// products stay in float; the result is rounded once.
#pragma once

#include "attention.h"

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

template <class T> __device__ __forceinline__ T paged_narrow(float v) {
    if constexpr (sizeof(T) == 2) {
        return f32_to_bf16(v);
    } else {
        return v;
    }
}

// One wave per (query head, KV head, sequence): a lane scores one key of 64, then the lanes take the head's dimensions.
template <class T> __device__ __forceinline__ void attention_paged(const PagedOperands<T>& a) {
    constexpr uint32_t MOST = 256;
    __shared__ float q[MOST];
    const uint32_t lane = threadIdx.x, g = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const float neg_inf = -__builtin_inff();
    const PagedRange range = paged_range(a, b);
    const uint32_t head = h * a.group + g;
    for (uint32_t d = lane; d < a.dim; d += kWave) {
        q[d] = paged_widen<T>(a.q[b * a.q_stride + uint64_t(head) * a.dim + d]);
    }
    __syncthreads();
    float peak = neg_inf, total = 0.0f, o[MOST / kWave] = {};
    const uint32_t count = range.head + (range.end - range.low);
    for (uint32_t n = 0; n < count; n += kWave) {
        const uint32_t i = n + lane, j = i < range.head ? i : range.low + (i - range.head);
        const T* k = nullptr;
        const T* v = nullptr;
        if (i < count) {
            if (j >= range.length) {
                k = a.k_new + b * a.new_stride + uint64_t(h) * a.dim;
                v = a.v_new + b * a.new_stride + uint64_t(h) * a.dim;
            } else {
                const int64_t page = a.table[b * a.table_stride + j / a.page_rows];
                if (page >= 0 && uint64_t(page) < a.pages) {
                    const uint64_t at = uint64_t(page) * a.page_stride + (j % a.page_rows) * a.row_stride + h * a.head_stride;
                    k = a.k + at;
                    v = a.v + at;
                }
            }
        }
        float score = neg_inf;
        if (k) {
            float sum = 0.0f;
            for (uint32_t d = 0; d < a.dim; ++d) {
                sum += q[d] * paged_widen<T>(k[d]);
            }
            score = sum * a.scale;
        }
        const float top = __builtin_fmaxf(peak, wave_max(score));
        const float base = top == neg_inf ? 0.0f : top;
        const float shrink = peak == neg_inf ? 0.0f : fast_exp(peak - base);
        const float p = k ? fast_exp(score - base) : 0.0f;
        total = total * shrink + wave_sum(p);
        for (uint32_t x = 0; x < MOST / kWave; ++x) {
            o[x] *= shrink;
        }
        peak = top;
        const unsigned long long seen = __ballot(k != nullptr);
        for (uint32_t from = 0; from < kWave; ++from) {
            if (!((seen >> from) & 1ull)) {
                continue;  // (a row that is not seen may hold anything)
            }
            const float weight = __shfl(p, from, kWave);
            const T* row = reinterpret_cast<const T*>(__shfl(reinterpret_cast<unsigned long long>(v), from, kWave));
            for (uint32_t x = 0; x < MOST / kWave; ++x) {
                if (lane + x * kWave < a.dim) {
                    o[x] += weight * paged_widen<T>(row[lane + x * kWave]);
                }
            }
        }
    }
    if (a.sinks) {
        const float sink = paged_widen<T>(a.sinks[head]), top = __builtin_fmaxf(peak, sink);
        const float base = top == neg_inf ? 0.0f : top;
        const float shrink = peak == neg_inf ? 0.0f : fast_exp(peak - base);
        total = total * shrink + (sink == neg_inf ? 0.0f : fast_exp(sink - base));
        for (uint32_t x = 0; x < MOST / kWave; ++x) {
            o[x] *= shrink;
        }
    }
    for (uint32_t x = 0; x < MOST / kWave; ++x) {
        if (lane + x * kWave < a.dim) {
            a.out[b * a.out_stride + uint64_t(head) * a.dim + lane + x * kWave] = paged_narrow<T>(total == 0.0f ? 0.0f : o[x] / total);
        }
    }
}

}  // namespace chroma
