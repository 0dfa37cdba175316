// Attention of a chunk of new tokens of every sequence over keys and values in pages (attention_paged.h for one token each):
//
//     o_i = sum_j exp(s_ij - m) v_j / (sum_j exp(s_ij - m) + exp(sink - m)),   s_ij = scale * (q_i . k_j),
//
// j over the rows that token i of the sequence sees: j <= p_i (its own row included), and with a window those after
// p_i - window and the first ones. Scores and sums stay in float and the result is rounded once.
//
// A bfloat16 weight meets V in tiles of 16 rows as two bfloat16 halves (2^-16 of it is lost), as attention_paged.h has it: the
// copies bound those, and the second product costs little (4 sequences of 16 tokens over 4000 rows, heads of 32, 19.3 -> 20.4 us,
// 32 of 4 over 4096, heads of 64, 59.5 -> 60.2, 16 tokens over 900 rows 12.5 either way). In the larger tiles, which the products
// and the weights themselves bound, it is rounded once (within 2^-8 of it): that adds as much error as the result's own rounding,
// 0.0023 of a result's size against 64 bits instead of 0.0017, and two halves would take a quarter longer (2 x 2048 tokens over
// 30000 rows 2241 -> 2871 us, 2048 of heads of 64 over 30000 1465 -> 1844, 4 x 512 over 4096 217 -> 270).
//
// A tile is 16 (token, head of the group) rows of a sequence and KV head, token by token: one token of 8 heads fills half of
// one, 16 tokens 8 of them. The tiles of all sequences are counted from ``starts`` on the device. A wave copies a block of keys
// and values global -> LDS through the page table and goes over it once, with a running maximum and sum; the waves of a
// workgroup take blocks in turn and are joined in LDS. Small calls are bound by that chain of dependent requests (starts, lengths,
// table, rows): 16 tokens over 900 rows, 8 KV heads of 8 heads of 64, 12.8 us; 32 sequences of one over 4096 56 us (4.8 TB/s; 48 where
// they are called again over the same cache, which the last cache then holds in part).
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

// The tile's extents, from its sequence's rows and their number.
template <uint32_t ROWS, class T>
__device__ __forceinline__ void chunk_extents(const ChunkOperands<T>& a, uint32_t b, ChunkRows rows, uint32_t held, uint32_t place, ChunkTile& tile) {
    const uint32_t count = rows.end - rows.begin;
    tile.b = b;
    tile.begin = rows.begin;
    tile.rows = count * a.group;
    tile.row = place * ROWS;
    tile.length = held;
    tile.base = int32_t(tile.length) - (a.k_new ? 0 : int32_t(count));
    const uint32_t last = (tile.row + ROWS < tile.rows ? tile.row + ROWS : tile.rows) - 1u;
    tile.first_position = tile.base + int32_t(tile.row / a.group);
    tile.last_position = tile.base + int32_t(last / a.group);
    tile.end = tile.last_position < 0 ? 0u : uint32_t(tile.last_position) + 1u;
    const int64_t low = int64_t(tile.first_position) - int64_t(a.window) + 1;
    tile.low = a.window && low > 0 ? (low < int64_t(tile.end) ? uint32_t(low) : tile.end) : 0u;
    tile.head = a.first < tile.low ? a.first : tile.low;
}

// Tile ``index`` of the call, the same in all lanes of a wave; false past the last. The sequences come in their order;
// LONGEST: up to 64 of them by the rows that they hold, and a sequence's last tile first, so that what takes longest starts
// first (workgroups start in the order of their indices). Above 512 they are counted eight to a lane, as each count waits for its
// loads: 1024 sequences of 8 tokens after 100 rows 195 -> 155 us (200 of 4, counted so, 49 -> 56).
template <uint32_t ROWS, bool LONGEST, class T> __device__ __forceinline__ bool chunk_tile(const ChunkOperands<T>& a, uint32_t index, ChunkTile& tile) {
    const uint32_t lane = threadIdx.x % kWave;
    const auto tiles_of = [&](ChunkRows rows) { return ((rows.end - rows.begin) * a.group + ROWS - 1u) / ROWS; };
    uint32_t before = 0;
    if (a.sequences <= 512u) {
        for (uint32_t b0 = 0; b0 < a.sequences; b0 += kWave) {
            ChunkRows rows{0u, 0u};
            uint32_t own = 0, order = lane, held = 0;
            if (b0 + lane < a.sequences) {
                rows = chunk_rows(a, b0 + lane);
                held = paged_length(a, b0 + lane);  // (under way together)
                own = tiles_of(rows);
            }
            if (LONGEST && a.sequences <= uint32_t(kWave)) {
                uint32_t rank = 0;
                for (uint32_t i = 0; i < a.sequences; ++i) {
                    const uint32_t other = __builtin_amdgcn_readlane(held, i);
                    rank += other > held || (other == held && i < lane) ? 1u : 0u;
                }
                rank = lane < a.sequences ? rank : lane;
                order = __builtin_amdgcn_ds_permute(int(rank * 4u), int(lane));  // the sequence of this lane's rank
                own = __shfl(own, order, kWave);
            }
            const uint32_t upto = before + paged_scan(own);
            const unsigned long long past = __ballot(upto > index);
            if (past) {
                const uint32_t at = __builtin_ctzll(past), b = __builtin_amdgcn_readlane(order, at);
                const uint32_t place = index - __builtin_amdgcn_readlane(upto - own, at);
                const ChunkRows found{uint32_t(__builtin_amdgcn_readlane(rows.begin, b)), uint32_t(__builtin_amdgcn_readlane(rows.end, b))};
                chunk_extents<ROWS>(a, b0 + b, found, __builtin_amdgcn_readlane(held, b),
                                    LONGEST ? __builtin_amdgcn_readlane(own, at) - 1u - place : place, tile);
                return true;
            }
            before = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        return false;
    }
    constexpr uint32_t EACH = 8u;
    for (uint32_t b0 = 0; b0 < a.sequences; b0 += EACH * kWave) {
        uint32_t own[EACH], sum = 0;
#pragma unroll
        for (uint32_t k = 0; k < EACH; ++k) {  // (clamped, so that all loads are under way together)
            const uint32_t b = b0 + lane * EACH + k, count = tiles_of(chunk_rows(a, b < a.sequences ? b : a.sequences - 1u));
            own[k] = b < a.sequences ? count : 0u;
            sum += own[k];
        }
        const uint32_t upto = before + paged_scan(sum);
        const unsigned long long past = __ballot(upto > index);
        if (past) {
            const uint32_t at = __builtin_ctzll(past);
            uint32_t place = index - __builtin_amdgcn_readlane(upto - sum, at), b = b0 + at * EACH;
            bool found = false;
#pragma unroll
            for (uint32_t k = 0; k < EACH; ++k) {
                const uint32_t count = __builtin_amdgcn_readlane(own[k], at);
                found = found || place < count;
                place -= found ? 0u : count;
                b += found ? 0u : 1u;
            }
            chunk_extents<ROWS>(a, b, chunk_rows(a, b), paged_length(a, b), LONGEST ? tiles_of(chunk_rows(a, b)) - 1u - place : place, tile);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return false;
}

// The rows that a token sees: ``span`` + 1 from ``low`` on, and those below ``head``.
struct ChunkSight {
    uint32_t low, span, head;
    template <class T> __device__ __forceinline__ ChunkSight(const ChunkOperands<T>& a, int32_t position) {
        const int64_t begin = int64_t(position) - int64_t(a.window) + 1;
        low = position < 0 ? ~0u : a.window && begin > 0 ? uint32_t(begin) : 0u;
        span = position < 0 ? 0u : uint32_t(position) - low;
        head = position < 0 ? 0u : a.first <= uint32_t(position) ? a.first : uint32_t(position) + 1u;
    }
    __device__ __forceinline__ bool operator()(uint32_t j) const { return j - low <= span || j < head; }
    // Bit r: whether it sees row begin + r, r < 64.
    __device__ __forceinline__ unsigned long long bits(uint32_t begin) const {
        const auto below = [&](uint32_t end) {  // rows before ``end``
            const int32_t n = int32_t(end) - int32_t(begin);
            return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull;
        };
        return (below(low + span + 1u) & ~below(low)) | below(head);  // (low + span + 1 is 0 where it sees none)
    }
};

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
// infinity or NaN would be NaN: such values join the rows that see them by themselves and leave the product. In bfloat16, where an
// infinity times halves of two signs would be NaN too, in a second pass where a sum comes out not finite; in float in every block
// that is not seen whole (a second pass takes registers: with heads of 64 a wave less of a SIMD, 2048 tokens over 4096 rows 2.4 -> 3.0 ms).
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
        const ChunkSight sight(a, tile.base + int32_t(token));
        const T* k_pages = a.k + kv * a.head_stride;
        const T* v_pages = a.v + kv * a.head_stride;
        const T* q = a.q + (tile.begin + token) * a.q_stride + (uint64_t(kv) * a.group + row % a.group) * a.dim;
        const T* k_new = a.k_new ? a.k_new + uint64_t(kv) * a.dim : k_pages;  // (never followed without new rows)
        const T* v_new = a.v_new ? a.v_new + uint64_t(kv) * a.dim : v_pages;
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
        // The pass over the blocks, and in bfloat16 a second one where a sum is not finite (``careful``).
        const uint32_t from = n;
        for (bool careful = false;; careful = true) {
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
                const auto join = [&] {  // values that are not finite
                    for (uint32_t r = 0; r < KEYS; ++r) {
                        const bool sees = ((seen >> r) & 1ull) && sight(begin + r);
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
                };
                if (BF16 && careful) {
                    join();
                }
                // every row of the tile sees every key of the block (but those that nothing sees)
                const bool whole = int32_t(begin + KEYS - 1u) <= tile.first_position &&
                                   (!a.window || int64_t(begin) + a.window > int64_t(tile.last_position) || begin + KEYS <= a.first);
                if (!BF16 && !whole) {
                    bool odd = false;
                    for (uint32_t c = lane; c < KEYS * DP; c += 64u) {
                        odd |= chunk_not_finite<T>(vs[c]);
                    }
                    if (__ballot(odd) != 0ull) {
                        join();
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
                        const bool sees = ((bits >> r) & 1u) && (whole || sight(begin + t * 16u + quad * 4u + r));
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
            bool odd = false;
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    odd |= !(__builtin_fabsf(o[dt][e]) < __builtin_inff());
                }
            }
            if (!BF16 || careful || __ballot(odd) == 0ull) {
                break;
            }
            n = from;  // (it has blocks: a wave without any has sums of 0)
            copy(n, page_of(n));
        }
        total += __shfl_xor(total, 16, kWave);
        total += __shfl_xor(total, 32, kWave);
    }
};

// Four values of a result, rounded by the conversion instruction.
template <class T> __device__ __forceinline__ void chunk_store4(T* to, f32x4_t v) {
    if constexpr (sizeof(T) == 2) {
        const bf16x2_t lo = __builtin_convertvector(f32x2_t{v[0], v[1]}, bf16x2_t), hi = __builtin_convertvector(f32x2_t{v[2], v[3]}, bf16x2_t);
        *reinterpret_cast<uint2*>(to) = uint2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    } else {
        *reinterpret_cast<f32x4_t*>(to) = v;
    }
}

// A row's result from parts of (maximum, sum, p . v); where a sum is 0 the row saw nothing.
template <class T>
__device__ __forceinline__ void chunk_store(const ChunkOperands<T>& a, const ChunkTile& tile, uint32_t kv, uint32_t r, uint32_t d, f32x4_t sum,
                                            float total) {
    const uint32_t row = tile.row + r;
    chunk_store4<T>(a.out + (tile.begin + row / a.group) * a.out_stride + (uint64_t(kv) * a.group + row % a.group) * a.dim + d,
                    sum * (total == 0.0f ? 0.0f : 1.0f / total));
}

// Floats of one (tile, KV head, split): ROWS rows of DP sums, then each row's maximum and sum.
template <int DP, uint32_t ROWS> constexpr uint32_t chunk_partial_floats() { return ROWS * (DP + 2u); }

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
    if (!chunk_tile<16u, false>(a, blockIdx.x / a.kv_heads, tile)) {
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
            float* to = partial + (uint64_t(blockIdx.x) * splits + split) * chunk_partial_floats<DP, 16u>();
            *reinterpret_cast<f32x4_t*>(to + r * DP + d) = sum;
            if (d == 0) {
                to[16u * DP + 2u * r] = merge.top;
                to[16u * DP + 2u * r + 1u] = merge.total;
            }
        }
    }
}

// FlashMerge with the maxima in units of log2 or not.
constexpr float kLog2e = 1.44269504088896341f;
template <bool LOG2> struct ChunkMerge {
    float top, total;
    __device__ __forceinline__ float weight(float peak) const {
        return peak == -__builtin_inff() ? 0.0f : LOG2 ? __builtin_amdgcn_exp2f(peak - top) : fast_exp(peak - top);
    }
};

// The splits of a tile of ROWS rows, in order, and the sink; LOG2: the maxima are of scores in units of log2.
// grid: (tiles x KV heads, ROWS / 16), 256 threads
template <class T, int DP, uint32_t ROWS, bool LOG2>
__device__ __forceinline__ void attention_chunk_combine(const ChunkOperands<T>& a, uint32_t splits, const float* __restrict__ partial) {
    constexpr uint32_t PART = chunk_partial_floats<DP, ROWS>();
    const uint32_t kv = blockIdx.x % a.kv_heads;
    ChunkTile tile;
    if (!chunk_tile<ROWS, LOG2>(a, blockIdx.x / a.kv_heads, tile)) {
        return;
    }
    const float* parts = partial + uint64_t(blockIdx.x) * splits * PART;
    for (uint32_t i = threadIdx.x; i < 16u * (DP / 4u); i += 256u) {
        const uint32_t r = blockIdx.y * 16u + i / (DP / 4u), d = i % (DP / 4u) * 4u;
        if (tile.row + r >= tile.rows || d >= a.dim) {
            continue;
        }
        const float sink = a.sinks ? paged_widen<T>(a.sinks[kv * a.group + (tile.row + r) % a.group]) * (LOG2 ? kLog2e : 1.0f) : -__builtin_inff();
        ChunkMerge<LOG2> merge{sink, 0.0f};
        for (uint32_t s = 0; s < splits; ++s) {
            merge.top = __builtin_fmaxf(merge.top, parts[uint64_t(s) * PART + ROWS * DP + 2u * r]);
        }
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (uint32_t s = 0; s < splits; ++s) {
            const float* part = parts + uint64_t(s) * PART;
            const float weight = merge.weight(part[ROWS * DP + 2u * r]);
            merge.total += weight * part[ROWS * DP + 2u * r + 1u];
            sum += weight * *reinterpret_cast<const f32x4_t*>(part + r * DP + d);
        }
        chunk_store(a, tile, kv, r, d, sum, merge.total + (a.sinks ? merge.weight(sink) : 0.0f));
    }
}

// ---------------------------------------------------------------------------------------------
// Long chunks of bfloat16: a tile is 32 rows a wave, and a workgroup's four or eight waves share blocks of K and V in LDS (two
// buffers of each, one barrier a block). Scores are K Q^T, so that a lane holds 16 of 32 keys of one row, and its
// weights are the second product's operand as they are: key slot (h, i) of 16 stands for key 8 (i / 4) + 4 h + i % 4 on both
// sides (V's comes from transposing reads).
//
// Scores are kept in units of log2: t = s * (scale log2 e), p = 2^(t - m). A lane's maximum is raised only past a headroom, so
// that most blocks change no sums.
//
// What bounds it is vector work: a score costs a product, a maximum, a power at a quarter of the rate, an addition and half a
// conversion, 30 cycles a wave's 64 of them against 16 (heads of 64) or 32 (heads of 128) of the matrix cores. 2 x 2048 tokens
// over 30000 rows with heads of 128 take 2.12-2.25 ms (925-980 TFLOP/s; the matrix cores 41% and the vector units 45% busy, no bank
// conflicts), 2048 over 30000 with heads of 64 1.46-1.54 ms (675-710 TFLOP/s; 31% and 64%). Without the copies the former would take a quarter
// less; copies further ahead, barriers for the scheduler and wave priorities moved it by 4% either way.

typedef float f32x16_t __attribute__((ext_vector_type(16)));

static __device__ const uint4 chunk_zeros[32] = {};  // a row of V for keys that nothing sees

template <int DP> constexpr uint32_t chunk_wide_keys() { return DP > 128 ? 32u : 64u; }

// FULL: the head dimension is DP.
// grid: (tiles x KV heads, splits), WAVES waves
template <int DP, uint32_t KEYS, uint32_t WAVES, bool FULL>
__device__ __forceinline__ void attention_chunk_wide(const ChunkOperands<uint16_t>& a, uint32_t splits, float* __restrict__ partial) {
    constexpr uint32_t PER_ROW = DP / 8u, BLOCK = KEYS * DP;          // 16-byte chunks of a row; elements of K or V of a block
    constexpr uint32_t ROWS = 32u * WAVES;
    constexpr int COPIES = BLOCK / 512 / WAVES;                 // 1 KiB pieces of K, and of V, that a wave copies
    constexpr int STEPS = DP / 16, TILES = KEYS / 32, DEEP = DP / 32;
    constexpr unsigned long long EVERY = KEYS == 64u ? ~0ull : (1ull << (KEYS % 64u)) - 1ull;
    static_assert(COPIES >= 1 && BLOCK % (512 * WAVES) == 0, "whole pieces for every wave");
    // Chunk c of K's row r lies at c ^ swizzle: 16 rows of one chunk, that one read's pass takes, fill the banks once; so do four
    // rows of V's 64 bytes.
    const auto k_swizzle = [](uint32_t r) { return PER_ROW >= 16u ? r & 15u : PER_ROW == 8u ? (r / 2u) & 7u : (r / 4u) & 3u; };
    const auto v_swizzle = [](uint32_t r) { return PER_ROW >= 16u ? (r & 3u) * 4u : PER_ROW == 8u ? ((r / 2u) & 1u) * 4u : 0u; };
    __shared__ __attribute__((aligned(1024))) uint16_t lds[4u * BLOCK];
    const uint32_t lane = threadIdx.x % 64u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), half = lane / 32u, col = lane % 32u;
    const uint32_t kv = blockIdx.x % a.kv_heads, split = blockIdx.y, chunks = FULL ? PER_ROW : a.dim / 8u;
    const float neg_inf = -__builtin_inff();
    ChunkTile tile;
    if (!chunk_tile<ROWS, true>(a, blockIdx.x / a.kv_heads, tile)) {
        return;
    }
    // this wave's rows (none: it only copies) and this lane's
    const uint32_t row0 = tile.row + wave * 32u, last_row = (row0 + 32u < tile.rows ? row0 + 32u : tile.rows) - 1u;
    const bool idle = row0 >= tile.rows;
    const uint32_t row = row0 + col < tile.rows ? row0 + col : tile.rows - 1u, token = row / a.group;
    const ChunkSight sight(a, tile.base + int32_t(token));
    const int32_t first_position = tile.base + int32_t((idle ? last_row : row0) / a.group), last_position = tile.base + int32_t(last_row / a.group);
    const uint64_t k_pages = uint64_t(a.k + kv * a.head_stride), v_pages = uint64_t(a.v + kv * a.head_stride);  // addresses
    const uint64_t k_new = uint64_t(a.k_new + uint64_t(kv) * a.dim), v_new = uint64_t(a.v_new + uint64_t(kv) * a.dim);
    const int64_t* table = a.table + tile.b * a.table_stride;
    // (the first rows and the window's follow one another: place v is that of row v, or behind the first rows of row v - head + low)
    const uint32_t places = tile.head + (tile.end - tile.low), stop = (places + KEYS - 1u) / KEYS, page_rows = a.page_rows, inverse = 0xffffffffu / page_rows;
    // j / page_rows: the rounded reciprocal is right or one too small
    const auto page_index = [&](uint32_t j) {
        const uint32_t q = __umulhi(j, inverse);
        return q + (j - q * page_rows >= page_rows ? 1u : 0u);
    };
    const auto row_at = [&](uint32_t v) { return v < tile.head ? v : v - tile.head + tile.low; };
    auto page_of = [&](uint32_t x) -> int64_t {  // of this lane's row of block x (-1: none)
        const uint32_t v = x * KEYS + lane, j = row_at(v);
        return lane < KEYS && v < places && j < tile.length ? table[page_index(j)] : -1;
    };
    if constexpr (!FULL) {  // zeros behind the rows' ends
        for (uint32_t c = threadIdx.x; c < 4u * BLOCK / 8u; c += 64u * WAVES) {
            *reinterpret_cast<uint4*>(lds + c * 8u) = uint4{0u, 0u, 0u, 0u};
        }
        __syncthreads();
    }
    // Copies block x into buffer ``to``; returns which of its rows there are.
    auto copy = [&](uint32_t x, uint32_t to, int64_t page) -> unsigned long long {
        const uint32_t v = x * KEYS + lane, j = row_at(v);
        const bool held = page >= 0 && uint64_t(page) < a.pages;
        const bool is_new = lane < KEYS && v < places && j >= tile.length;
        const uint64_t place = 2u * (held ? uint64_t(page) * a.page_stride + uint64_t(j - page_index(j) * page_rows) * a.row_stride
                                     : is_new ? uint64_t(tile.begin + (j - tile.length)) * a.new_stride : 0u);
        const unsigned long long here = __ballot(held || is_new), fresh = __ballot(is_new);
        uint16_t* ks = lds + to * 2u * BLOCK;
        uint16_t* vs = ks + BLOCK;
        const auto pieces = [&](auto addresses) {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                const uint32_t piece = wave * COPIES + i, r = piece * (64u / PER_ROW) + lane / PER_ROW;
                const uint32_t k_chunk = (lane % PER_ROW) ^ k_swizzle(r), v_chunk = (lane % PER_ROW) ^ v_swizzle(r);
                uint64_t k, v;
                addresses(r, __shfl(place, r, kWave), k, v);
                if (k_chunk < chunks) {
                    __builtin_amdgcn_global_load_lds((global_void*)(k + k_chunk * 16u), (lds_void*)(ks + piece * 512u), 16, 0, 0);
                }
                if (v_chunk < chunks) {
                    __builtin_amdgcn_global_load_lds((global_void*)(v + v_chunk * 16u), (lds_void*)(vs + piece * 512u), 16, 0, 0);
                }
            }
        };
        if (here == EVERY && fresh == 0ull) {
            pieces([&](uint32_t, uint64_t from, uint64_t& k, uint64_t& v) { k = k_pages + from, v = v_pages + from; });
        } else {
            pieces([&](uint32_t r, uint64_t from, uint64_t& k, uint64_t& v) {
                const bool beside = (fresh >> r) & 1ull, there = (here >> r) & 1ull;
                k = (beside ? k_new : k_pages) + from;
                v = there ? (beside ? v_new : v_pages) + from : uint64_t(chunk_zeros);
            });
        }
        return here;
    };

    // Scores are taken with |scale|, a negative one's sign in Q, and one of 0 as a Q of zeros.
    const float factor = a.scale == 0.0f ? 1.0f : __builtin_fabsf(a.scale) * kLog2e;
    const uint32_t keep = a.scale == 0.0f ? 0u : ~0u, flip = a.scale < 0.0f ? 0x80008000u : 0u;
    uint4 qf[STEPS];
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
        qf[c] = uint4{0u, 0u, 0u, 0u};
        if (c * 2u + half < chunks) {
            qf[c] = *reinterpret_cast<const uint4*>(a.q + (tile.begin + token) * a.q_stride + (uint64_t(kv) * a.group + row % a.group) * a.dim + (c * 2u + half) * 8u);
            qf[c] = uint4{(qf[c].x ^ flip) & keep, (qf[c].y ^ flip) & keep, (qf[c].z ^ flip) & keep, (qf[c].w ^ flip) & keep};
        }
    }
    float peak, total;
    f32x16_t o[DEEP];
    // The pass over the blocks, and a second one where a result is not finite (``careful``), in which the values that are not
    // finite leave V's block and join the rows that see them by themselves (ChunkWave).
    for (bool careful = false;; careful = true) {
        peak = neg_inf;
        total = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DEEP; ++dt) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                o[dt][e] = 0.0f;
            }
        }
        uint32_t n = split, buffer = 0;
        unsigned long long seen = 0;
        int64_t ahead = -1;
        if (n < stop) {
            seen = copy(n, 0u, page_of(n));
            ahead = n + splits < stop ? page_of(n + splits) : -1;
        }
        for (; n < stop; n += splits, buffer ^= 1u) {
            const uint32_t place = n * KEYS, begin = place - tile.head + tile.low, next = n + splits;
            const uint32_t firsts = place < tile.head ? tile.head - place : 0u;  // first rows that it begins with
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(vmcnt_wait(0));
            __builtin_amdgcn_s_barrier();  // block n has landed, and every wave is done with the other buffer
            __builtin_amdgcn_sched_barrier(0);
            const unsigned long long here = seen;
            if (next < stop) {
                seen = copy(next, buffer ^ 1u, ahead);
                ahead = next + splits < stop ? page_of(next + splits) : -1;
            }
            __builtin_amdgcn_sched_barrier(0);
            const uint16_t* ks = lds + buffer * 2u * BLOCK;
            uint16_t* vs = lds + buffer * 2u * BLOCK + BLOCK;
            if (careful) {
                for (uint32_t r = 0; r < KEYS; ++r) {
                    const bool sees = ((here >> r) & 1ull) && sight(row_at(place + r));
#pragma unroll
                    for (int dt = 0; dt < DEEP; ++dt) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint32_t d = dt * 32u + 8u * (e / 4) + 4u * half + e % 4;
                            const uint16_t v = vs[r * DP + ((d / 8u) ^ v_swizzle(r)) * 8u + d % 8u];
                            o[dt][e] += sees && chunk_not_finite<uint16_t>(v) ? bf16_to_f32(v) : 0.0f;
                        }
                    }
                }
                __syncthreads();  // every wave has read them
                for (uint32_t c = threadIdx.x; c < BLOCK; c += 64u * WAVES) {
                    if (chunk_not_finite<uint16_t>(vs[c])) {
                        vs[c] = 0;
                    }
                }
                __syncthreads();
            }
            // what none of this wave's rows sees is skipped
            if (idle || (!firsts && (int32_t(begin) > last_position ||
                                     (a.window && int64_t(begin) + KEYS - 1 + a.window <= int64_t(first_position) && begin >= a.first)))) {
                continue;
            }
            f32x16_t s[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[t][e] = 0.0f;
                }
            }
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const uint32_t r = t * 32u + col;
                    const uint4 kf = *reinterpret_cast<const uint4*>(ks + r * DP + ((c * 2u + half) ^ k_swizzle(r)) * 8u);
                    s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, kf), __builtin_bit_cast(bf16x8_t, qf[c]), s[t], 0, 0, 0);
                }
            }
            // rows that some of the wave's tokens do not see (the chunk's own, the window's first), and rows that are not there
            const bool some = firsts < KEYS && (int32_t(begin + KEYS - 1u) > first_position ||
                                                (a.window && int64_t(begin) + a.window <= int64_t(last_position) && begin + KEYS > a.first));
            if (some || here != EVERY) {
                const unsigned long long others = firsts < 64u ? ~0ull << firsts : 0ull;  // (all see the first rows)
                const unsigned long long visible = some ? here & (sight.bits(begin) | ~others) : here;
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const uint32_t bits = uint32_t(visible >> (32 * t)) >> (4u * half);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {  // a bit spread over a word chooses the score's bits or those of -inf
                        const uint32_t mask = uint32_t(__builtin_amdgcn_sbfe(int(bits), 8 * (e / 4) + e % 4, 1));
                        s[t][e] = __uint_as_float((__float_as_uint(s[t][e]) & mask) | (0xff800000u & ~mask));
                    }
                }
            }
            float tops[4] = {neg_inf, neg_inf, neg_inf, neg_inf};
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    tops[e % 4] = __builtin_fmaxf(tops[e % 4], s[t][e]);
                }
            }
            float top = __builtin_fmaxf(__builtin_fmaxf(tops[0], tops[1]), __builtin_fmaxf(tops[2], tops[3]));
            top *= factor;
            if (__ballot(top > peak + kFlashHeadroom || (peak == neg_inf && top != neg_inf)) != 0ull) {
                const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                top = __builtin_fmaxf(__builtin_fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1])), peak);
                const float shrink = peak == neg_inf ? 1.0f : __builtin_amdgcn_exp2f(peak - top);
                total *= shrink;
#pragma unroll
                for (int dt = 0; dt < DEEP; ++dt) {
                    o[dt] *= shrink;
                }
                peak = top;
            }
            const float base = peak == neg_inf ? 0.0f : -peak;
            float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < 2 * TILES; ++g) {
                bf16x8_t weights;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g / 2][g % 2 * 8 + e], factor, base));
                    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g / 2][g % 2 * 8 + e + 1], factor, base));
                    sums[e % 4] += x;
                    sums[e % 4 + 1] += y;
                    const bf16x2_t pair = __builtin_convertvector(f32x2_t{x, y}, bf16x2_t);
                    weights[e] = pair[0];
                    weights[e + 1] = pair[1];
                }
#pragma unroll
                for (int dt = 0; dt < DEEP; ++dt) {
                    s16x4_t four[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t r = g * 16u + x * 8u + half * 4u + (lane % 16u) / 4u;
                        const uint32_t chunk = (dt * 4u + (lane / 16u) % 2u * 2u + (lane % 4u) / 2u) ^ v_swizzle(r);
                        four[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vs + r * DP + chunk * 8u + (lane % 2u) * 4u));
                    }
                    const uint2 lo = __builtin_bit_cast(uint2, four[0]), hi = __builtin_bit_cast(uint2, four[1]);
                    const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, uint4{lo.x, lo.y, hi.x, hi.y});
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, weights, o[dt], 0, 0, 0);
                }
            }
            total += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        }
        bool odd = false;
#pragma unroll
        for (int dt = 0; dt < DEEP; ++dt) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                odd |= !(__builtin_fabsf(o[dt][e]) < __builtin_inff());
            }
        }
        // (asked in the same LDS array: beside a second one every read above would wait for all copies)
        uint32_t* flags = reinterpret_cast<uint32_t*>(lds);
        __syncthreads();
        if (lane == 0u) {
            flags[wave] = 0u;
        }
        if (odd) {
            flags[wave] = 1u;
        }
        __syncthreads();
        uint32_t any = 0;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) {
            any |= flags[w];
        }
        __syncthreads();
        if (careful || !any) {
            break;
        }
    }
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(total), __float_as_uint(total), false, false);
    total = __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
    if (row0 + col >= tile.rows) {
        return;
    }
    if (splits == 1u) {
        const float sink = a.sinks ? bf16_to_f32(a.sinks[kv * a.group + row % a.group]) * kLog2e : neg_inf;
        const ChunkMerge<true> merge{__builtin_fmaxf(peak, sink), 0.0f};
        const float weight = merge.weight(peak), sum = weight * total + (a.sinks ? merge.weight(sink) : 0.0f), scaled = sum == 0.0f ? 0.0f : weight / sum;
        uint16_t* to = a.out + (tile.begin + token) * a.out_stride + (uint64_t(kv) * a.group + row % a.group) * a.dim;
#pragma unroll
        for (int dt = 0; dt < DEEP; ++dt) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t d = dt * 32u + 2u * e + 4u * half;
                if (FULL || d < a.dim) {
                    chunk_store4<uint16_t>(to + d, f32x4_t{o[dt][e], o[dt][e + 1], o[dt][e + 2], o[dt][e + 3]} * scaled);
                }
            }
        }
    } else {
        const uint32_t r = wave * 32u + col;
        float* to = partial + (uint64_t(blockIdx.x) * splits + split) * chunk_partial_floats<DP, ROWS>();
#pragma unroll
        for (int dt = 0; dt < DEEP; ++dt) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                *reinterpret_cast<f32x4_t*>(to + r * DP + dt * 32u + 2u * e + 4u * half) = f32x4_t{o[dt][e], o[dt][e + 1], o[dt][e + 2], o[dt][e + 3]};
            }
        }
        if (half == 0u) {
            to[ROWS * DP + 2u * r] = peak;
            to[ROWS * DP + 2u * r + 1u] = total;
        }
    }
}

}  // namespace chroma
