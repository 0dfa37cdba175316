// ``chroma_hip_rows_adjust``: penalties for a row's repeated tokens, biases and a token mask on logits, in one pass.
//
// A workgroup takes a span of one row's ids: it requests the span's logits, biases and mask words, counts the span's tokens
// of the row's history in LDS (integer atomics: their order does not matter) while those are under way, then changes and
// writes the logits. Every workgroup of a row reads its whole history, so long spans read less and short ones spread a few
// rows over the chip. What bounds it: many rows the memory (256 rows of 201088 float logits with masks, 412 MB,
// 76 us, 5.5 TB/s), few rows the chain of requests (one row with a history of 700: 4 us).
#include "adjust.h"

#include <hip/hip_runtime.h>

#include <chroma_hip/device.h>

#include <cstdio>

namespace {

// 16 bytes of logits as 4 words: float values, or pairs of bfloat16 ones.
template <class T> struct Vector;

template <> struct Vector<float> {
    uint32_t w[4];
    __device__ __forceinline__ float get(int e) const { return __uint_as_float(w[e]); }
    __device__ __forceinline__ void set(int e, float v) { w[e] = __float_as_uint(v); }
    // -inf where bit e of ``allowed`` is 0
    __device__ __forceinline__ void keep(uint32_t allowed) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t all = uint32_t(int32_t(allowed << (31 - e)) >> 31);
            w[e] = (w[e] & all) | (0xff800000u & ~all);
        }
    }
};

template <> struct Vector<uint16_t> {
    uint32_t w[4];
    __device__ __forceinline__ float get(int e) const { return __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16); }
    __device__ __forceinline__ void set(int e, float v) {
        const uint32_t bits = chroma::f32_to_bf16(v);
        w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | bits << 16 : (w[e / 2] & 0xffff0000u) | bits;
    }
    __device__ __forceinline__ void keep(uint32_t allowed) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t low = uint32_t(int32_t(allowed << (31 - e)) >> 31), high = uint32_t(int32_t(allowed << (30 - e)) >> 31);
            const uint32_t all = (low & 0xffffu) | (high & 0xffff0000u);
            w[e / 2] = (w[e / 2] & all) | (0xff80ff80u & ~all);
        }
    }
};

// Both values to bfloat16 as f32_to_bf16 rounds them (v_cvt_pk_bf16_f32 keeps a NaN's payload).
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
    const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(chroma::f32x2_t{x, y}, chroma::bf16x2_t));
    return (__builtin_isnan(x) ? 0x7fc0u : w & 0xffffu) | (__builtin_isnan(y) ? 0x7fc00000u : w & 0xffff0000u);
}

// N values that start on their own size (global loads and stores of 16 bytes need no more).
template <class V, int N> struct __attribute__((packed, aligned(sizeof(V)))) Values {
    V v[N];
};

// A span is THREADS x PER vectors of 16 bytes of logits, a multiple of 32 ids.
template <class T, int THREADS, int PER> constexpr uint32_t span_ids() { return THREADS * PER * (16 / sizeof(T)); }

// What happens to one logit (``n`` occurrences in the history), before it is rounded.
struct Penalties {
    float repetition, presence, frequency;
    __device__ __forceinline__ float operator()(float value, uint32_t n) const {
        value = value > 0.0f ? value / repetition : value * repetition;
        return value - (presence + frequency * float(n));
    }
};

template <class T, int THREADS, int PER> __global__ void __launch_bounds__(THREADS) rows_adjust(chroma_hip_adjust_call c) {
    constexpr int N = 16 / sizeof(T);
    constexpr uint32_t SPAN = span_ids<T, THREADS, PER>();
    using Logits = Values<T, N>;
    using Words = Vector<T>;
    using Floats = Values<float, N>;
    __shared__ __attribute__((aligned(16))) uint32_t counts[SPAN];
    const uint64_t r = blockIdx.y;
    const uint32_t begin = blockIdx.x * SPAN, ids = min(SPAN, uint32_t(c.width) - begin), vectors = ids / N;
    const T* x = static_cast<const T*>(c.x) + r * c.x_stride + begin;
    T* y = static_cast<T*>(c.y) + r * c.y_stride + begin;
    const float* bias = c.bias ? c.bias + r * c.bias_stride + begin : nullptr;
    const uint32_t* mask = c.mask ? c.mask + r * c.mask_stride + begin / 32u : nullptr;
    const bool in_place = x == y, sparse = in_place && !bias && !mask;  // (sparse: only the history's logits are read)
    const Penalties penalties{c.repetition ? c.repetition[r] : 1.0f, c.presence ? c.presence[r] : 0.0f, c.frequency ? c.frequency[r] : 0.0f};
    // Whole vectors threadIdx.x + k THREADS of the span, every load unconditional with its index clamped (a guarded load
    // ends its branch with a wait for all loads in flight). What is left of a row's end, fewer than N, comes last.
    const auto place = [&](int k) { return min(k * THREADS + threadIdx.x, vectors - 1u) * N; };
    Words logits[PER];
    Floats biases[PER];
    uint32_t words[PER];
    // The first ids of the history are requested before its length is known.
    constexpr int BATCH = 4;
    int64_t id[BATCH] = {-1, -1, -1, -1};
    const int64_t* history = c.history + r * c.history_stride;
    if (c.history && c.history_width) {
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            id[k] = history[min(int64_t(k * THREADS + threadIdx.x), c.history_width - 1)];
        }
    }
    if (vectors && !sparse) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            logits[k] = __builtin_bit_cast(Words, *reinterpret_cast<const Logits*>(x + place(k)));
        }
    }
    if (vectors && mask) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            words[k] = mask[place(k) / 32u];
        }
    }
    if (vectors && bias) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            biases[k] = *reinterpret_cast<const Floats*>(bias + place(k));
        }
    }
    if (c.history) {
#pragma unroll
        for (uint32_t i = threadIdx.x * 4u; i < SPAN; i += THREADS * 4u) {
            *reinterpret_cast<uint4*>(counts + i) = uint4{0u, 0u, 0u, 0u};
        }
        const int64_t given = c.history_lengths ? c.history_lengths[r] : c.history_width;
        const int64_t length = given < 0 ? 0 : given > c.history_width ? c.history_width : given;
        __syncthreads();
        for (int64_t i0 = 0;;) {
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const uint64_t at = uint64_t(id[k]) - begin;
                if (at < ids && i0 + k * THREADS + threadIdx.x < length) {
                    atomicAdd(&counts[at], 1u);
                }
            }
            i0 += THREADS * BATCH;
            if (i0 >= length) {
                break;
            }
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                id[k] = history[min(i0 + k * THREADS + threadIdx.x, length - 1)];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t i = (k * THREADS + threadIdx.x) * N;
        if (i >= vectors * N) {
            break;
        }
        uint32_t n[N], counted = 0;
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const uint4 four = c.history ? *reinterpret_cast<const uint4*>(counts + i + e) : uint4{0u, 0u, 0u, 0u};
            n[e] = four.x, n[e + 1] = four.y, n[e + 2] = four.z, n[e + 3] = four.w;
            counted |= four.x | four.y | four.z | four.w;
        }
        const uint32_t every = (1u << N) - 1u, allowed = mask ? words[k] >> (i % 32u) & every : every;
        if (in_place && !counted && !bias && allowed == every) {
            continue;
        }
        Words w = logits[k];
        if (sparse) {
            w = __builtin_bit_cast(Words, *reinterpret_cast<const Logits*>(x + i));
        }
        if (counted) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (n[e]) {
                    const float value = penalties(w.get(e), n[e]);
                    w.set(e, bias ? value + biases[k].v[e] : value);
                    biases[k].v[e] = -0.0f;  // added
                }
            }
        }
        if (bias) {
            if constexpr (N == 8) {
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    w.w[e / 2] = bf16_pair(w.get(e) + biases[k].v[e], w.get(e + 1) + biases[k].v[e + 1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    w.set(e, w.get(e) + biases[k].v[e]);
                }
            }
        }
        w.keep(allowed);
        *reinterpret_cast<Logits*>(y + i) = __builtin_bit_cast(Logits, w);
    }
    if (const uint32_t i = vectors * N + threadIdx.x; i < ids) {
        Words w;
        w.w[0] = x[i];
        if constexpr (N == 4) {
            w.set(0, x[i]);
        }
        const uint32_t n = c.history ? counts[i] : 0u;
        if (n || bias) {
            const float value = n ? penalties(w.get(0), n) : w.get(0);
            w.set(0, bias ? value + bias[i] : value);
        }
        const bool allowed = !mask || (mask[i / 32u] >> (i % 32u) & 1u);
        T result;
        if constexpr (N == 4) {
            result = allowed ? w.get(0) : -__builtin_inff();
        } else {
            result = allowed ? T(w.w[0]) : T(0xff80u);
        }
        if (!in_place || n || bias || !allowed) {
            y[i] = result;
        }
    }
}

template <class T, int THREADS, int PER> void launch(const chroma_hip_adjust_call& c, hipStream_t stream) {
    constexpr int64_t span = span_ids<T, THREADS, PER>();
    rows_adjust<T, THREADS, PER><<<dim3(unsigned((c.width + span - 1) / span), unsigned(c.rows)), THREADS, 0, stream>>>(c);
}

// Spans of 8192 ids once they leave three workgroups for every compute unit, else of 4096: 64 rows of 201088 bfloat16
// logits, histories of 4096, a bias and masks 17.6 us (1024 / 16384 ids with 1024 threads: 35 / 20.2), 32 rows with
// histories of 8192 and neither 13.3 against 13.1, 4 rows 6.9 against 5.3 (1024 ids: 8.9).
template <class T> void launch(const chroma_hip_adjust_call& c, hipStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (c.rows * ((c.width + 8191) / 8192) >= 768) {
        launch<T, 512, 16 / V>(c, stream);
    } else {
        launch<T, 512, 8 / V>(c, stream);
    }
}

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "rows_adjust: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

}  // namespace

namespace chroma_adjust {

int launch_rows_adjust(const chroma_hip_adjust_call& c, hipStream_t stream, char* error, size_t error_size) {
    if (const char* wrong = mistake(c)) {
        return refuse(wrong, error, error_size);
    }
    if (c.dtype == CHROMA_HIP_FLOAT32) {
        launch<float>(c, stream);
    } else {
        launch<uint16_t>(c, stream);
    }
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? CHROMA_HIP_OK : refuse(hipGetErrorString(status), error, error_size);
}

}  // namespace chroma_adjust

extern "C" __attribute__((visibility("default"))) int chroma_hip_rows_adjust(const chroma_hip_adjust_call* call, void* stream, char* error,
                                                                             size_t error_size) {
    if (!call) {
        return refuse("null call", error, error_size);
    }
    return chroma_adjust::launch_rows_adjust(*call, static_cast<hipStream_t>(stream), error, error_size);
}
