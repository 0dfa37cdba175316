// Attention of one new token per sequence over keys and values in pages:
//
//     o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m)),   s_j = scale * (q . k_j),
//
// j over the cached rows that the sequence's page table holds and its window leaves, and the new row. Scores and sums stay
// in float and the result is rounded once; a bfloat16 weight meets V as two halves (below).
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
    uint32_t sequences, kv_heads, group, dim;
    float scale;
};

// The rows a sequence's token sees: [0, head) and [low, end), the new row (position ``length``) among the latter.
struct PagedRange {
    uint32_t length, head, low, end;
};

template <class T> __device__ __forceinline__ uint32_t paged_length(const PagedOperands<T>& a, uint32_t b) {
    const int64_t given = a.lengths[b];
    return given < 0 ? 0u : given > int64_t(a.longest) ? a.longest : uint32_t(given);
}

template <class T> __device__ __forceinline__ PagedRange paged_range(const PagedOperands<T>& a, uint32_t length) {
    PagedRange r;
    r.length = length;
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

// A wave takes blocks of a sequence's keys for 16 query heads of a KV head. It copies a block of K and of V global -> LDS into
// buffers of its own (no barrier); lane l finds row l of the block through the table, and the lanes that copy it receive its
// place by a shuffle. The products are those of attention_flash.h, a tile's 16 rows the query heads. Short sequences have a
// workgroup whose waves take the blocks in turn (``attention_paged_whole``, one launch). Otherwise the blocks of all
// sequences, in order, are cut into equal shares, so that long and short sequences load the chip alike
// (``attention_paged_shares``); where a share ends inside a sequence its (maximum, sum, p . v) go to scratch, and
// ``attention_paged_combine`` adds the sequence's parts in order. (Adding them in the wave that comes last, behind
// device-scope stores and flags, was slower: one sequence of 900 rows 19.6 us against 14.2 with the second launch, 32 up to 4096
// 50 against 38.) DP is the head dimension in whole matrix-core operands; what lies past ``dim`` in a row is zero.
//
// Rows that are not seen keep their probability at exactly 0 and their values out of the products, so that they may hold
// anything. A bfloat16 probability meets V as two bfloat16 halves (2^-16 of it is lost): the products are a small part of
// the time, and one half alone (2^-9) would add as much error as the result's own rounding.
constexpr uint32_t kPagedWaves = 4;  // of a workgroup on shares: they take adjacent KV heads, whose rows adjoin in memory

template <class T, int DP> constexpr uint32_t paged_keys() {  // keys of a block: 16 KiB of K and V, a multiple of an operand
    constexpr uint32_t fits = 16384u / (2u * DP * sizeof(T)), least = sizeof(T) == 2 ? 32u : 16u;
    return fits > 64u ? 64u : fits < least ? least : fits;
}

// In a workgroup that takes a whole sequence: blocks of half the size and 8 waves (two workgroups a compute unit; 4 waves
// of whole blocks take 8 mixed sequences up to 2000 rows in 19.5 us, these in 15.8, 8 of whole blocks in 14.3 but 128 up to 1000 in
// 38 against 31).
template <class T, int DP> constexpr uint32_t paged_whole_keys() {
    constexpr uint32_t keys = paged_keys<T, DP>(), least = sizeof(T) == 2 ? 32u : 16u;
    return keys / 2u < least ? least : keys / 2u;
}
template <class T, int DP> constexpr uint32_t paged_whole_waves() { return paged_whole_keys<T, DP>() * DP * sizeof(T) > 8192u ? 4u : 8u; }

// Key blocks of a sequence: the first rows', then those from range.low on; one (of nothing) where nothing is seen.
template <uint32_t KEYS> __device__ __forceinline__ uint32_t paged_blocks(const PagedRange& r) {
    const uint32_t n = (r.head + KEYS - 1u) / KEYS + (r.end - r.low + KEYS - 1u) / KEYS;
    return n ? n : 1u;
}

__device__ __forceinline__ uint32_t paged_scan(uint32_t v) {  // inclusive sums over the wave
    const uint32_t lane = threadIdx.x % kWave;
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) {
        const uint32_t before = __shfl_up(v, step, kWave);
        v += lane >= uint32_t(step) ? before : 0u;
    }
    return v;
}

// The sequences' lengths, the first 64 in registers, one to a lane (what is read once more waits once more).
template <uint32_t KEYS, class T> struct PagedLengths {
    const PagedOperands<T>& a;
    uint32_t own, own_blocks;
    __device__ __forceinline__ explicit PagedLengths(const PagedOperands<T>& a) : a(a) {
        const uint32_t lane = threadIdx.x % kWave;
        own = lane < a.sequences ? paged_length(a, lane) : 0u;
        own_blocks = lane < a.sequences ? paged_blocks<KEYS>(paged_range(a, own)) : 0u;
    }
    // blocks of this lane's sequence b0 + lane (0 past the last); b0 a multiple of 64
    __device__ __forceinline__ uint32_t blocks(uint32_t b0) const {
        const uint32_t b = b0 + threadIdx.x % kWave;
        return b0 == 0 ? own_blocks : b < a.sequences ? paged_blocks<KEYS>(paged_range(a, paged_length(a, b))) : 0u;
    }
    // of sequence b, the same in all lanes
    __device__ __forceinline__ PagedRange range(uint32_t b) const {
        return paged_range(a, b < uint32_t(kWave) ? uint32_t(__builtin_amdgcn_readlane(own, b)) : paged_length(a, b));
    }
};

// Share w < ranges holds blocks [begin(w), begin(w + 1)) of ``total``, one at least; ``of`` gives the share that holds a block.
struct PagedShares {
    uint64_t total, ranges;
    __device__ __forceinline__ PagedShares(uint32_t blocks, uint32_t most) : total(blocks), ranges(most < blocks ? most : blocks) {}
    __device__ __forceinline__ uint32_t begin(uint32_t w) const { return uint32_t(w * total / ranges); }
    __device__ __forceinline__ uint32_t of(uint32_t block) const { return uint32_t(((block + 1ull) * ranges - 1ull) / total); }
};

// Scratch: per (slot, query head) the DP sums of p . v, then the maximum and the sum. The part of sequence b in share w has
// slot w + b (one of the two grows from a part to the next).
template <int DP> struct PagedScratch {
    float* stats;
    float* sums;
    __device__ __forceinline__ PagedScratch(float* base, uint64_t slots, uint64_t heads) : stats(base + slots * heads * DP), sums(base) {}
};

template <class T> __device__ __forceinline__ void paged_store4(T* to, const f32x4_t& v) {
    if constexpr (sizeof(T) == 2) {
        const uint32_t lo = f32_to_bf16(v[0]) | (uint32_t(f32_to_bf16(v[1])) << 16), hi = f32_to_bf16(v[2]) | (uint32_t(f32_to_bf16(v[3])) << 16);
        *reinterpret_cast<uint2*>(to) = uint2{lo, hi};
    } else {
        *reinterpret_cast<f32x4_t*>(to) = v;
    }
}

// One wave's pass over key blocks of one sequence, 16 query heads of a KV head: (maximum, sum, p . v) of what they hold.
// ``ks`` and ``vs``: LDS of KEYS rows of DP values each. Lane (quad, col) ends up with values 16 dt + 4 quad .. + 3 of head
// ``col`` in o[dt], and that head's maximum and sum.
// STREAM: the copies leave no room in the caches to what they bring (it is read once).
template <class T, int DP, uint32_t KEYS, bool STREAM> struct PagedWave {
    static constexpr bool BF16 = sizeof(T) == 2;
    static constexpr uint32_t CHUNK = 16u / sizeof(T), PER_ROW = DP / CHUNK;
    static constexpr int COPIES = KEYS * DP * sizeof(T) / 1024, PARTS = PER_ROW / 4u, TILES = KEYS / 16;
    static constexpr uint32_t SWZ = PER_ROW % 8u == 0 ? 7u : 3u;  // chunk c of row r lies at c ^ ((r / 2) & SWZ)
    static constexpr uint32_t ELEMENTS = 2u * KEYS * DP;          // of LDS
    static constexpr int AUX = STREAM ? 2 : 0;                    // the copies' cache policy
    static_assert(PER_ROW % 4u == 0 && 64u % PER_ROW == 0 && KEYS <= 64u && KEYS % (BF16 ? 32u : 16u) == 0, "block");

    float peak, total;
    f32x4_t o[DP / 16];

    // Zeros behind the rows' ends, once, before the first copies.
    static __device__ __forceinline__ void prepare(const PagedOperands<T>& a, T* ks) {
        if (a.dim < uint32_t(DP)) {
            for (uint32_t c = threadIdx.x % 64u; c < 2u * KEYS * PER_ROW; c += 64u) {
                *reinterpret_cast<uint4*>(ks + c * CHUNK) = uint4{0u, 0u, 0u, 0u};
            }
            __builtin_amdgcn_s_waitcnt(0);
        }
    }

    // Blocks n, n + step, ... below stop of sequence b, KV head kv, query head ``head`` in this lane's column.
    __device__ __forceinline__ void run(const PagedOperands<T>& a, const PagedRange& range, uint32_t b, uint32_t kv, uint32_t head, uint32_t n,
                                        uint32_t stop, uint32_t step, T* ks, T* vs) {
        const uint32_t lane = threadIdx.x % 64u, quad = lane / 16u, col = lane % 16u, chunks = a.dim / CHUNK;
        const float neg_inf = -__builtin_inff();
        const T* k_pages = a.k + kv * a.head_stride;
        const T* v_pages = a.v + kv * a.head_stride;
        const T* q = a.q + b * a.q_stride + uint64_t(head) * a.dim;
        const T* k_new = a.k_new + b * a.new_stride + uint64_t(kv) * a.dim;
        const T* v_new = a.v_new + b * a.new_stride + uint64_t(kv) * a.dim;
        const int64_t* table = a.table + b * a.table_stride;
        const uint32_t head_blocks = (range.head + KEYS - 1u) / KEYS;
        auto block_begin = [&](uint32_t x) { return x < head_blocks ? x * KEYS : range.low + (x - head_blocks) * KEYS; };
        auto block_end = [&](uint32_t x) { return x < head_blocks ? range.head : range.end; };
        // The page of this lane's row of block x (-1: none).
        auto page_of = [&](uint32_t x) -> int64_t {
            const uint32_t j = block_begin(x) + lane;
            return lane < KEYS && j < block_end(x) && j < range.length ? table[j / a.page_rows] : -1;
        };
        unsigned long long seen = 0;
        auto copy = [&](uint32_t x, int64_t page) {
            const uint32_t first = block_begin(x), j = first + lane;
            const bool held = page >= 0 && uint64_t(page) < a.pages;
            const uint64_t place = held ? uint64_t(page) * a.page_stride + uint64_t(j % a.page_rows) * a.row_stride : 0u;
            seen = __ballot(held || (lane < KEYS && j >= range.length && j < block_end(x)));
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                const uint32_t r = i * (64u / PER_ROW) + lane / PER_ROW, chunk = (lane % PER_ROW) ^ ((r / 2u) & SWZ);
                const uint64_t from = __shfl(place, r, kWave);
                const bool fresh = first + r == range.length && range.end > range.length;
                const T* k = (fresh ? k_new : k_pages + from) + chunk * CHUNK;
                const T* v = (fresh ? v_new : v_pages + from) + chunk * CHUNK;
                if (chunk < chunks) {
                    __builtin_amdgcn_global_load_lds((global_void*)k, (lds_void*)(ks + i * (1024u / sizeof(T))), 16, 0, AUX);
                    __builtin_amdgcn_global_load_lds((global_void*)v, (lds_void*)(vs + i * (1024u / sizeof(T))), 16, 0, AUX);
                }
            }
        };
        if (n < stop) {
            copy(n, page_of(n));
        }
        uint4 qf[PARTS];
#pragma unroll
        for (int c = 0; c < PARTS; ++c) {
            qf[c] = uint4{0u, 0u, 0u, 0u};
            if (c * 4u + quad < chunks) {
                qf[c] = *reinterpret_cast<const uint4*>(q + (c * 4u + quad) * CHUNK);
            }
        }
        peak = neg_inf;
        total = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DP / 16; ++dt) {
            o[dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        while (n < stop) {
            const uint32_t next = n + step;
            int64_t next_page = -1;
            if (next < stop) {
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
            if (next < stop) {  // both buffers have been read
                copy(next, next_page);
            }
            n = next;
        }
        total += __shfl_xor(total, 16, kWave);
        total += __shfl_xor(total, 32, kWave);
    }

    // The finished row of this lane's head, the sink added, in place.
    __device__ __forceinline__ void finish(const PagedOperands<T>& a, uint32_t b, uint32_t head) {
        const uint32_t quad = threadIdx.x % 64u / 16u;
        const float sink = a.sinks ? paged_widen<T>(a.sinks[head]) : -__builtin_inff();
        const FlashMerge merge{__builtin_fmaxf(peak, sink), 0.0f};
        const float weight = merge.weight(peak), sum = weight * total + (a.sinks ? merge.weight(sink) : 0.0f);
        const float factor = sum == 0.0f ? 0.0f : weight / sum;
#pragma unroll
        for (int dt = 0; dt < DP / 16; ++dt) {
            if (dt * 16u + quad * 4u < a.dim) {
                paged_store4<T>(a.out + b * a.out_stride + uint64_t(head) * a.dim + dt * 16u + quad * 4u, o[dt] * factor);
            }
        }
    }
};

// One workgroup of WAVES waves for all blocks of a sequence and KV head: the waves take blocks in turn and meet in LDS.
// grid: (KV heads x row tiles, sequences)
template <class T, int DP, uint32_t KEYS, uint32_t WAVES> __device__ __forceinline__ void attention_paged_whole(const PagedOperands<T>& a) {
    using Wave = PagedWave<T, DP, KEYS, false>;
    constexpr uint32_t OPAD = DP + 4u, PART = Wave::ELEMENTS * sizeof(T) / 4u;  // floats of a wave's LDS
    static_assert(16u * (OPAD + 2u) <= PART, "a wave's sums fit its LDS");
    __shared__ __attribute__((aligned(1024))) T lds[WAVES * Wave::ELEMENTS];
    const uint32_t lane = threadIdx.x % 64u, quad = lane / 16u, col = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t tiles = (a.group + 15u) / 16u, kv = blockIdx.x / tiles, row0 = blockIdx.x % tiles * 16u, b = blockIdx.y;
    const uint32_t head = kv * a.group + (row0 + col < a.group ? row0 + col : a.group - 1u);
    T* ks = lds + wave * Wave::ELEMENTS;
    const PagedRange range = paged_range(a, paged_length(a, b));
    Wave x;
    Wave::prepare(a, ks);
    x.run(a, range, b, kv, head, wave, paged_blocks<KEYS>(range), WAVES, ks, ks + KEYS * DP);
    float* mine = reinterpret_cast<float*>(ks);
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) {
        *reinterpret_cast<f32x4_t*>(mine + col * OPAD + dt * 16u + quad * 4u) = x.o[dt];
    }
    if (quad == 0) {
        mine[16u * OPAD + 2u * col] = x.peak;
        mine[16u * OPAD + 2u * col + 1u] = x.total;
    }
    __syncthreads();
    const float* parts = reinterpret_cast<const float*>(lds);
    for (uint32_t i = threadIdx.x; i < 16u * (DP / 4u); i += 64u * WAVES) {
        const uint32_t r = i / (DP / 4u), d = i % (DP / 4u) * 4u;
        if (row0 + r >= a.group || d >= a.dim) {
            continue;
        }
        const uint32_t row = kv * a.group + row0 + r;
        const float sink = a.sinks ? paged_widen<T>(a.sinks[row]) : -__builtin_inff();
        FlashMerge merge{sink, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) {
            merge.top = __builtin_fmaxf(merge.top, parts[w * PART + 16u * OPAD + 2u * r]);
        }
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) {
            const float weight = merge.weight(parts[w * PART + 16u * OPAD + 2u * r]);
            merge.total += weight * parts[w * PART + 16u * OPAD + 2u * r + 1u];
            sum += weight * *reinterpret_cast<const f32x4_t*>(parts + w * PART + r * OPAD + d);
        }
        merge.total += a.sinks ? merge.weight(sink) : 0.0f;
        paged_store4<T>(a.out + b * a.out_stride + uint64_t(row) * a.dim + d, sum * (merge.total == 0.0f ? 0.0f : 1.0f / merge.total));
    }
}

// The blocks of all sequences in equal shares. STREAM where a head's row is whole 128-byte lines and one wave reads it (the
// other heads or row tiles of a line would fetch it again): 64 sequences of 8192 rows 206 -> 184 us (5.8 TB/s), six up to 131072
// with heads of 128 345 -> 305 (6.3 TB/s; heads of 32, two to a line, 32 -> 36 us for 32 of 16384).
// grid: ceil(ranges x KV heads x row tiles / kPagedWaves), 256 threads
template <class T, int DP, uint32_t KEYS, bool STREAM>
__device__ __forceinline__ void attention_paged_shares(const PagedOperands<T>& a, uint32_t ranges, float* __restrict__ scratch) {
    using Wave = PagedWave<T, DP, KEYS, STREAM>;
    __shared__ __attribute__((aligned(1024))) T lds[kPagedWaves * Wave::ELEMENTS];
    const uint32_t lane = threadIdx.x % 64u, quad = lane / 16u, col = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t tiles = (a.group + 15u) / 16u, heads = a.kv_heads * tiles, worker = blockIdx.x * kPagedWaves + wave;
    const uint32_t w = worker / heads, kv = worker % heads / tiles, row0 = worker % heads % tiles * 16u;
    T* ks = lds + wave * Wave::ELEMENTS;
    const PagedScratch<DP> parts(scratch, uint64_t(ranges) + a.sequences, uint64_t(a.kv_heads) * a.group);

    // This wave's share of the blocks, and the sequence b and its block n at which it begins.
    const PagedLengths<KEYS, T> lengths(a);
    uint32_t all = 0;
    for (uint32_t b0 = 0; b0 < a.sequences; b0 += kWave) {
        all += lengths.blocks(b0);
    }
    const uint32_t upto0 = paged_scan(all);
    const PagedShares shares(__builtin_amdgcn_readlane(upto0, kWave - 1), ranges);
    if (w >= shares.ranges) {
        return;
    }
    const uint32_t begin = shares.begin(w);
    uint32_t left = shares.begin(w + 1u) - begin, b = 0, n = 0;
    for (uint32_t before = 0, b0 = 0; b0 < a.sequences; b0 += kWave) {
        const uint32_t own = lengths.blocks(b0);
        const uint32_t upto = a.sequences <= uint32_t(kWave) ? upto0 : before + paged_scan(own);
        const unsigned long long past = __ballot(upto > begin);
        if (past) {
            const uint32_t at = __builtin_ctzll(past);
            b = b0 + at;
            n = begin - __builtin_amdgcn_readlane(upto - own, at);
            break;
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    Wave::prepare(a, ks);
    const uint32_t head = kv * a.group + (row0 + col < a.group ? row0 + col : a.group - 1u);
    for (; left; ++b, n = 0) {
        const PagedRange range = lengths.range(b);
        const uint32_t blocks = paged_blocks<KEYS>(range), count = blocks - n < left ? blocks - n : left;
        left -= count;
        Wave x;
        x.run(a, range, b, kv, head, n, n + count, 1u, ks, ks + KEYS * DP);
        if (row0 + col >= a.group) {
            continue;
        }
        if (count == blocks) {
            x.finish(a, b, head);
            continue;
        }
        const uint64_t at = uint64_t(w + b) * a.kv_heads * a.group + head;
#pragma unroll
        for (int dt = 0; dt < DP / 16; ++dt) {
            *reinterpret_cast<f32x4_t*>(parts.sums + at * DP + dt * 16u + quad * 4u) = x.o[dt];
        }
        if (quad == 0) {
            *reinterpret_cast<float2*>(parts.stats + 2u * at) = float2{x.peak, x.total};
        }
    }
}

// The parts of every sequence that lies in more than one share, and the sink. WAVES waves take a query head (grid:
// ceil(sequences x query heads x WAVES / 4), 256 threads): a lane holds 4 dimensions of every 64 / (DP / 4)-th part.
template <class T, int DP, uint32_t KEYS, uint32_t WAVES>
__device__ __forceinline__ void attention_paged_combine(const PagedOperands<T>& a, uint32_t ranges, float* __restrict__ scratch) {
    constexpr uint32_t ACROSS = DP / 4u, STEP = 64u / ACROSS * WAVES;
    __shared__ float sums[WAVES > 1 ? WAVES : 1][WAVES > 1 ? DP : 1], totals[WAVES > 1 ? WAVES : 1];
    const uint32_t lane = threadIdx.x % 64u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), heads = a.kv_heads * a.group;
    const uint32_t unit = WAVES > 1 ? blockIdx.x : blockIdx.x * 4u + wave, b = unit / heads, head = unit % heads;
    if (b >= a.sequences) {
        return;
    }
    const PagedScratch<DP> parts(scratch, uint64_t(ranges) + a.sequences, heads);
    const PagedLengths<KEYS, T> lengths(a);
    uint32_t all = 0, before = 0;
    for (uint32_t b0 = 0; b0 < a.sequences; b0 += kWave) {
        const uint32_t own = lengths.blocks(b0);
        all += own;
        before += b0 + lane < b ? own : 0u;
    }
    all = __builtin_amdgcn_readlane(paged_scan(all), kWave - 1);
    before = __builtin_amdgcn_readlane(paged_scan(before), kWave - 1);
    const PagedShares shares(all, ranges);
    const uint32_t first = shares.of(before), count = shares.of(before + paged_blocks<KEYS>(lengths.range(b)) - 1u) - first + 1u;
    if (count == 1u) {
        return;  // written by its wave
    }
    const uint64_t at0 = uint64_t(first + b) * heads + head;
    const float sink = a.sinks ? paged_widen<T>(a.sinks[head]) : -__builtin_inff();
    float top = sink;
    for (uint32_t s = lane; s < count; s += kWave) {
        top = __builtin_fmaxf(top, parts.stats[2u * (at0 + uint64_t(s) * heads)]);
    }
    top = wave_max(top);
    const FlashMerge merge{top, 0.0f};
    const uint32_t d = lane % ACROSS * 4u, group = lane / ACROSS + (WAVES > 1 ? wave * (64u / ACROSS) : 0u);
    f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float total = 0.0f;
#pragma unroll 4
    for (uint32_t s = group; s < count; s += STEP) {
        const uint64_t at = at0 + uint64_t(s) * heads;
        const float2 stat = *reinterpret_cast<const float2*>(parts.stats + 2u * at);
        const f32x4_t o = *reinterpret_cast<const f32x4_t*>(parts.sums + at * DP + d);  // (past dim: what lies there, never stored)
        const float weight = merge.weight(stat.x);
        total += weight * stat.y;
        sum += weight * o;
    }
#pragma unroll
    for (uint32_t step = ACROSS; step < 64u; step *= 2u) {
        total += __shfl_xor(total, step, kWave);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum[i] += __shfl_xor(sum[i], step, kWave);
        }
    }
    if constexpr (WAVES > 1) {
        if (lane < ACROSS) {
            *reinterpret_cast<f32x4_t*>(&sums[wave][d]) = sum;
            totals[wave] = total;
        }
        __syncthreads();
        if (wave) {
            return;
        }
#pragma unroll
        for (uint32_t x = 1; x < WAVES; ++x) {
            sum += *reinterpret_cast<const f32x4_t*>(&sums[x][d]);
            total += totals[x];
        }
    }
    total += a.sinks ? merge.weight(sink) : 0.0f;
    if (lane < ACROSS && d < a.dim) {
        paged_store4<T>(a.out + b * a.out_stride + uint64_t(head) * a.dim + d, sum * (total == 0.0f ? 0.0f : 1.0f / total));
    }
}

}  // namespace chroma
