// Attention of a chunk of new tokens of every sequence over keys and values in pages (attention_paged.h for one token each):
//
//     o_i = sum_j exp(s_ij - m) v_j / (sum_j exp(s_ij - m) + exp(sink - m)),   s_ij = scale * (q_i . k_j),
//
// j over the rows that token i of the sequence sees: j <= p_i (its own row included), and with a window those after
// p_i - window and the first ones. Scores and sums stay in float and the result is rounded once; a bfloat16 weight meets V
// rounded to bfloat16.
//
// A tile is 16 (token, head of the group) rows of a sequence and KV head, token by token: one token of 8 heads fills half of
// one, 16 tokens 8 of them. The tiles of all sequences are counted from ``starts`` on the device.
#pragma once

#include "attention_paged.h"

namespace chroma {

// Token i of sequence b is row starts[b] + i of q, out and the new rows; its position is the cached rows + i where new rows
// are given beside the cache, and otherwise the last starts[b + 1] - starts[b] of the cached rows are the new ones.
template <class T> struct ChunkOperands : PagedOperands<T> {
    const int64_t* starts;
    uint32_t tokens;
};

// Tokens of a sequence: rows [begin, end) of q.
struct ChunkRows {
    uint32_t begin, end;
};

template <class T> __device__ __forceinline__ ChunkRows chunk_rows(const ChunkOperands<T>& a, uint32_t b) {
    const auto within = [&](int64_t v, uint32_t low) { return v < int64_t(low) ? low : v > int64_t(a.tokens) ? a.tokens : uint32_t(v); };
    ChunkRows r;
    r.begin = within(a.starts[b], 0u);
    r.end = within(a.starts[b + 1], r.begin);
    return r;
}

// ROWS rows from ``row`` on of a sequence's tokens and a KV head, and the keys that some of them see: [0, head) and [low, end).
struct ChunkTile {
    uint32_t b, row, rows;            // rows: of the sequence (tokens x group)
    uint32_t begin, length;           // its first row of q, its cached rows
    int32_t base;                     // position of its first token
    int32_t first_position, last_position;  // of the tile's tokens
    uint32_t head, low, end;

    // Whether position p sees row j.
    template <class T> __device__ __forceinline__ bool sees(const ChunkOperands<T>& a, int32_t p, uint32_t j) const {
        return int32_t(j) <= p && (!a.window || int64_t(j) + a.window > int64_t(p) || j < a.first);
    }
    template <uint32_t KEYS> __device__ __forceinline__ uint32_t head_blocks() const { return (head + KEYS - 1u) / KEYS; }
    template <uint32_t KEYS> __device__ __forceinline__ uint32_t blocks() const { return head_blocks<KEYS>() + (end - low + KEYS - 1u) / KEYS; }
    template <uint32_t KEYS> __device__ __forceinline__ uint32_t block_begin(uint32_t x) const {
        return x < head_blocks<KEYS>() ? x * KEYS : low + (x - head_blocks<KEYS>()) * KEYS;
    }
    template <uint32_t KEYS> __device__ __forceinline__ uint32_t block_end(uint32_t x) const {  // of what the tile may see of it
        const uint32_t stop = x < head_blocks<KEYS>() ? head : end, last = block_begin<KEYS>(x) + KEYS;
        return last < stop ? last : stop;
    }
};

// Tile ``index`` of the call in the sequences' order, the same in all lanes of a wave; false past the last.
template <uint32_t ROWS, class T> __device__ __forceinline__ bool chunk_tile(const ChunkOperands<T>& a, uint32_t index, ChunkTile& tile) {
    const uint32_t lane = threadIdx.x % kWave;
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.sequences; b0 += kWave) {
        ChunkRows rows{0u, 0u};
        uint32_t own = 0;
        if (b0 + lane < a.sequences) {
            rows = chunk_rows(a, b0 + lane);
            own = ((rows.end - rows.begin) * a.group + ROWS - 1u) / ROWS;
        }
        const uint32_t upto = before + paged_scan(own);
        const unsigned long long past = __ballot(upto > index);
        if (past) {
            const uint32_t at = __builtin_ctzll(past);
            tile.b = b0 + at;
            tile.begin = __builtin_amdgcn_readlane(rows.begin, at);
            const uint32_t count = __builtin_amdgcn_readlane(rows.end, at) - tile.begin;
            tile.rows = count * a.group;
            tile.row = (index - __builtin_amdgcn_readlane(upto - own, at)) * ROWS;
            tile.length = paged_length(a, tile.b);
            tile.base = int32_t(tile.length) - (a.k_new ? 0 : int32_t(count));
            const uint32_t last = (tile.row + ROWS < tile.rows ? tile.row + ROWS : tile.rows) - 1u;
            tile.first_position = tile.base + int32_t(tile.row / a.group);
            tile.last_position = tile.base + int32_t(last / a.group);
            tile.end = tile.last_position < 0 ? 0u : uint32_t(tile.last_position) + 1u;
            const int64_t low = int64_t(tile.first_position) - int64_t(a.window) + 1;
            tile.low = a.window && low > 0 ? (low < int64_t(tile.end) ? uint32_t(low) : tile.end) : 0u;
            tile.head = a.first < tile.low ? a.first : tile.low;
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return false;
}

template <class T> __device__ __forceinline__ bool chunk_not_finite(T v) {
    if constexpr (sizeof(T) == 2) {
        return (v & 0x7f80u) == 0x7f80u;
    } else {
        return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
    }
}

// One wave's pass over key blocks of one tile of 16 rows: PagedWave's products (attention_paged.h), with a limit for each
// row. Lane (quad, col) ends up with values 16 dt + 4 quad .. + 3 of row ``col`` in o[dt], and that row's maximum and sum.
//
// Where a row of V is hidden from some rows of the tile and not from others, its weight for the former is 0, and 0 times an
// infinity or NaN would be NaN: such values join the rows that see them by themselves and leave the product.
template <class T, int DP, uint32_t KEYS> struct ChunkWave {
    static constexpr bool BF16 = sizeof(T) == 2;
    static constexpr uint32_t CHUNK = 16u / sizeof(T), PER_ROW = DP / CHUNK;
    static constexpr int COPIES = KEYS * DP * sizeof(T) / 1024, PARTS = PER_ROW / 4u, TILES = KEYS / 16;
    static constexpr uint32_t SWZ = PER_ROW % 8u == 0 ? 7u : 3u;  // chunk c of row r lies at c ^ ((r / 2) & SWZ)
    static constexpr uint32_t ELEMENTS = 2u * KEYS * DP;          // of LDS
    static_assert(PER_ROW % 4u == 0 && 64u % PER_ROW == 0 && KEYS <= 64u && KEYS % (BF16 ? 32u : 16u) == 0, "block");

    float peak, total;
    f32x4_t o[DP / 16];

    // Zeros behind the rows' ends, once, before the first copies.
    static __device__ __forceinline__ void prepare(const ChunkOperands<T>& a, T* ks) {
        if (a.dim < uint32_t(DP)) {
            for (uint32_t c = threadIdx.x % 64u; c < 2u * KEYS * PER_ROW; c += 64u) {
                *reinterpret_cast<uint4*>(ks + c * CHUNK) = uint4{0u, 0u, 0u, 0u};
            }
            __builtin_amdgcn_s_waitcnt(0);
        }
    }

    // Blocks n, n + step, ... of the tile, KV head kv.
    __device__ __forceinline__ void run(const ChunkOperands<T>& a, const ChunkTile& tile, uint32_t kv, uint32_t n, uint32_t step, T* ks, T* vs) {
        const uint32_t lane = threadIdx.x % 64u, quad = lane / 16u, col = lane % 16u, chunks = a.dim / CHUNK, stop = tile.template blocks<KEYS>();
        const float neg_inf = -__builtin_inff();
        const uint32_t row = tile.row + col < tile.rows ? tile.row + col : tile.rows - 1u, token = row / a.group;
        const int32_t position = tile.base + int32_t(token);
        const T* k_pages = a.k + kv * a.head_stride;
        const T* v_pages = a.v + kv * a.head_stride;
        const T* q = a.q + (tile.begin + token) * a.q_stride + (uint64_t(kv) * a.group + row % a.group) * a.dim;
        const T* k_new = a.k_new + uint64_t(kv) * a.dim;
        const T* v_new = a.v_new + uint64_t(kv) * a.dim;
        const int64_t* table = a.table + tile.b * a.table_stride;
        // The page of this lane's row of block x (-1: none).
        auto page_of = [&](uint32_t x) -> int64_t {
            const uint32_t j = tile.template block_begin<KEYS>(x) + lane;
            return j < tile.template block_end<KEYS>(x) && j < tile.length ? table[j / a.page_rows] : -1;
        };
        unsigned long long seen = 0;
        auto copy = [&](uint32_t x, int64_t page) {
            const uint32_t j = tile.template block_begin<KEYS>(x) + lane;
            const bool held = page >= 0 && uint64_t(page) < a.pages;
            const bool is_new = j >= tile.length && j < tile.template block_end<KEYS>(x);
            const uint64_t place = held ? uint64_t(page) * a.page_stride + uint64_t(j % a.page_rows) * a.row_stride
                                 : is_new ? uint64_t(tile.begin + (j - tile.length)) * a.new_stride : 0u;
            seen = __ballot(held || is_new);
            const unsigned long long fresh = __ballot(is_new);
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                const uint32_t r = i * (64u / PER_ROW) + lane / PER_ROW, chunk = (lane % PER_ROW) ^ ((r / 2u) & SWZ);
                const uint64_t from = __shfl(place, r, kWave);
                const bool beside = (fresh >> r) & 1ull;
                const T* k = (beside ? k_new : k_pages) + from + chunk * CHUNK;
                const T* v = (beside ? v_new : v_pages) + from + chunk * CHUNK;
                if (chunk < chunks) {
                    __builtin_amdgcn_global_load_lds((global_void*)k, (lds_void*)(ks + i * (1024u / sizeof(T))), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((global_void*)v, (lds_void*)(vs + i * (1024u / sizeof(T))), 16, 0, 0);
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
            const uint32_t next = n + step, begin = tile.template block_begin<KEYS>(n);
            int64_t next_page = -1;
            if (next < stop) {
                next_page = page_of(next);
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(vmcnt_wait(0));
            __builtin_amdgcn_sched_barrier(0);
            if (seen != (KEYS == 64u ? ~0ull : (1ull << (KEYS % 64u)) - 1ull)) {  // what no row sees may hold anything
                for (uint32_t c = lane; c < KEYS * PER_ROW; c += 64u) {
                    if (!((seen >> (c / PER_ROW)) & 1ull)) {
                        *reinterpret_cast<uint4*>(vs + c * CHUNK) = uint4{0u, 0u, 0u, 0u};
                    }
                }
            }
            // every row of the tile sees every key of the block (but those that nothing sees)
            const bool whole = int32_t(begin + KEYS - 1u) <= tile.first_position &&
                               (!a.window || int64_t(begin) + a.window > int64_t(tile.last_position) || begin + KEYS <= a.first);
            if (!whole) {
                bool odd = false;
                for (uint32_t c = lane; c < KEYS * DP; c += 64u) {
                    odd |= chunk_not_finite<T>(vs[c]);
                }
                if (__ballot(odd) != 0ull) {
                    for (uint32_t r = 0; r < KEYS; ++r) {
                        const bool sees = ((seen >> r) & 1ull) && tile.sees(a, position, begin + r);
#pragma unroll
                        for (int dt = 0; dt < DP / 16; ++dt) {
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) {
                                const uint32_t d = dt * 16u + quad * 4u + e;
                                const T v = vs[r * DP + ((d / CHUNK) ^ ((r / 2u) & SWZ)) * CHUNK + d % CHUNK];
                                o[dt][e] += sees && chunk_not_finite<T>(v) ? paged_widen<T>(v) : 0.0f;
                            }
                        }
                    }
                    for (uint32_t c = lane; c < KEYS * DP; c += 64u) {
                        if (chunk_not_finite<T>(vs[c])) {
                            vs[c] = T(0);
                        }
                    }
                }
            }
            // scores of keys 16 t + 4 quad + r for this lane's row
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
                    const bool sees = ((bits >> r) & 1u) && (whole || tile.sees(a, position, begin + t * 16u + quad * 4u + r));
                    u[t][r] = sees ? s[r] * a.scale : neg_inf;
                    top = __builtin_fmaxf(top, u[t][r]);
                }
            }
            if (__ballot(top > peak + kFlashHeadroom || (peak == neg_inf && top != neg_inf)) != 0ull) {
                top = __builtin_fmaxf(top, __shfl_xor(top, 16, kWave));
                top = __builtin_fmaxf(top, __shfl_xor(top, 32, kWave));
                top = __builtin_fmaxf(top, peak);
                const float shrink = peak == neg_inf ? 0.0f : fast_exp(peak - top);
                if (peak != neg_inf) {  // (what has no maximum yet has no sums but values that are not finite)
                    total *= shrink;
#pragma unroll
                    for (int dt = 0; dt < DP / 16; ++dt) {
                        o[dt] *= shrink;
                    }
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
                    bf16x8_t weights;
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        weights[x] = __bf16(u[2 * h + x / 4][x % 4]);
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
                        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, weights, o[dt], 0, 0, 0);
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
};

// A row's result from parts of (maximum, sum, p . v); where a sum is 0 the row saw nothing.
template <class T>
__device__ __forceinline__ void chunk_store(const ChunkOperands<T>& a, const ChunkTile& tile, uint32_t kv, uint32_t r, uint32_t d, f32x4_t sum,
                                            float total) {
    const uint32_t row = tile.row + r;
    paged_store4<T>(a.out + (tile.begin + row / a.group) * a.out_stride + (uint64_t(kv) * a.group + row % a.group) * a.dim + d,
                    sum * (total == 0.0f ? 0.0f : 1.0f / total));
}

// Floats of one (tile, KV head, split): 16 rows of DP sums, then each row's maximum and sum.
template <int DP> constexpr uint32_t chunk_partial_floats() { return 16u * (DP + 2u); }

// A workgroup of WAVES waves takes every ``splits``-th of a tile's blocks; its waves take blocks in turn and meet in LDS.
// grid: (tiles x KV heads, splits)
template <class T, int DP, uint32_t KEYS, uint32_t WAVES>
__device__ __forceinline__ void attention_chunk_tiles(const ChunkOperands<T>& a, uint32_t splits, float* __restrict__ partial) {
    using Wave = ChunkWave<T, DP, KEYS>;
    constexpr uint32_t OPAD = DP + 4u, PART = Wave::ELEMENTS * sizeof(T) / 4u;  // floats of a wave's LDS
    static_assert(16u * (OPAD + 2u) <= PART, "a wave's sums fit its LDS");
    __shared__ __attribute__((aligned(1024))) T lds[WAVES * Wave::ELEMENTS];
    const uint32_t lane = threadIdx.x % 64u, quad = lane / 16u, col = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t kv = blockIdx.x % a.kv_heads, split = blockIdx.y;
    ChunkTile tile;
    if (!chunk_tile<16u>(a, blockIdx.x / a.kv_heads, tile)) {
        return;
    }
    T* ks = lds + wave * Wave::ELEMENTS;
    Wave x;
    Wave::prepare(a, ks);
    x.run(a, tile, kv, split * WAVES + wave, WAVES * splits, ks, ks + KEYS * DP);
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
        if (tile.row + r >= tile.rows || d >= a.dim) {
            continue;
        }
        const bool sinks = a.sinks && splits == 1u;
        const float sink = sinks ? paged_widen<T>(a.sinks[kv * a.group + (tile.row + r) % a.group]) : -__builtin_inff();
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
        if (splits == 1u) {
            chunk_store(a, tile, kv, r, d, sum, merge.total + (sinks ? merge.weight(sink) : 0.0f));
        } else {
            float* to = partial + (uint64_t(blockIdx.x) * splits + split) * chunk_partial_floats<DP>();
            *reinterpret_cast<f32x4_t*>(to + r * DP + d) = sum;
            if (d == 0) {
                to[16u * DP + 2u * r] = merge.top;
                to[16u * DP + 2u * r + 1u] = merge.total;
            }
        }
    }
}

// The splits of a tile, in order, and the sink. grid: tiles x KV heads, 256 threads
template <class T, int DP>
__device__ __forceinline__ void attention_chunk_combine(const ChunkOperands<T>& a, uint32_t splits, const float* __restrict__ partial) {
    const uint32_t kv = blockIdx.x % a.kv_heads;
    ChunkTile tile;
    if (!chunk_tile<16u>(a, blockIdx.x / a.kv_heads, tile)) {
        return;
    }
    const float* parts = partial + uint64_t(blockIdx.x) * splits * chunk_partial_floats<DP>();
    for (uint32_t i = threadIdx.x; i < 16u * (DP / 4u); i += 256u) {
        const uint32_t r = i / (DP / 4u), d = i % (DP / 4u) * 4u;
        if (tile.row + r >= tile.rows || d >= a.dim) {
            continue;
        }
        const float sink = a.sinks ? paged_widen<T>(a.sinks[kv * a.group + (tile.row + r) % a.group]) : -__builtin_inff();
        FlashMerge merge{sink, 0.0f};
        for (uint32_t s = 0; s < splits; ++s) {
            merge.top = __builtin_fmaxf(merge.top, parts[s * chunk_partial_floats<DP>() + 16u * DP + 2u * r]);
        }
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t s = 0; s < splits; ++s) {
            const float* part = parts + s * chunk_partial_floats<DP>();
            const float weight = merge.weight(part[16u * DP + 2u * r]);
            merge.total += weight * part[16u * DP + 2u * r + 1u];
            sum += weight * *reinterpret_cast<const f32x4_t*>(part + r * DP + d);
        }
        chunk_store(a, tile, kv, r, d, sum, merge.total + (a.sinks ? merge.weight(sink) : 0.0f));
    }
}

}  // namespace chroma
