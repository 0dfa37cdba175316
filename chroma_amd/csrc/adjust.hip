// ``chroma_hip_rows_adjust``: penalties for a row's repeated tokens, biases and a token mask on logits, in one pass.
//
// A workgroup takes a span of one row's ids: it counts the span's tokens of the row's history in LDS (integer atomics:
// their order does not matter), then reads, changes and writes the span's logits.
#include "adjust.h"

#include <hip/hip_runtime.h>

#include <chroma_hip/device.h>

#include <cstdio>

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kSpan = 4096;  // ids of a workgroup; a multiple of 32, so its mask words are its own

template <class T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<uint16_t>(uint16_t v) { return chroma::bf16_to_f32(v); }
template <class T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t narrow<uint16_t>(float v) { return chroma::f32_to_bf16(v); }

template <class T> __global__ void __launch_bounds__(kThreads) rows_adjust(chroma_hip_adjust_call c) {
    __shared__ uint32_t counts[kSpan];
    const uint64_t r = blockIdx.y;
    const uint32_t begin = blockIdx.x * kSpan, ids = min(kSpan, uint32_t(c.width) - begin);
    for (uint32_t i = threadIdx.x; i < kSpan; i += kThreads) {
        counts[i] = 0;
    }
    __syncthreads();
    if (c.history) {
        const int64_t given = c.history_lengths ? c.history_lengths[r] : c.history_width;
        const int64_t length = given < 0 ? 0 : given > c.history_width ? c.history_width : given;
        for (int64_t i = threadIdx.x; i < length; i += kThreads) {
            const uint64_t at = uint64_t(c.history[r * c.history_stride + i]) - begin;
            if (at < ids) {
                atomicAdd(&counts[at], 1u);
            }
        }
    }
    __syncthreads();
    const float repetition = c.repetition ? c.repetition[r] : 1.0f;
    const float presence = c.presence ? c.presence[r] : 0.0f, frequency = c.frequency ? c.frequency[r] : 0.0f;
    const T* x = static_cast<const T*>(c.x) + r * c.x_stride + begin;
    T* y = static_cast<T*>(c.y) + r * c.y_stride + begin;
    for (uint32_t i = threadIdx.x; i < ids; i += kThreads) {
        float value = widen<T>(x[i]);
        if (const uint32_t n = counts[i]) {
            value = value > 0.0f ? value / repetition : value * repetition;
            value -= presence + frequency * float(n);
        }
        if (c.bias) {
            value += c.bias[r * c.bias_stride + begin + i];
        }
        if (c.mask && !((c.mask[r * c.mask_stride + (begin + i) / 32u] >> (i % 32u)) & 1u)) {
            value = -__builtin_inff();
        }
        y[i] = narrow<T>(value);
    }
}

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "rows_adjust: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

const char* mistake(const chroma_hip_adjust_call& c) {
    if (c.dtype != CHROMA_HIP_FLOAT32 && c.dtype != CHROMA_HIP_BFLOAT16) {
        return "dtype must be CHROMA_HIP_FLOAT32 or CHROMA_HIP_BFLOAT16";
    }
    if (c.rows < 1 || c.rows > 65535 || c.width < 1 || c.width >= int64_t(1) << 31) {
        return "want 1 to 65535 rows of 1 to 2147483647 logits";
    }
    if (c.x_stride < c.width || c.y_stride < c.width || (c.history && (c.history_width < 0 || c.history_stride < c.history_width)) ||
        (c.bias && c.bias_stride && c.bias_stride < c.width) || (c.mask && c.mask_stride && c.mask_stride < (c.width + 31) / 32)) {
        return "a stride is smaller than its row";
    }
    if (!c.x || !c.y) {
        return "null device pointer";
    }
    const uintptr_t size = c.dtype == CHROMA_HIP_FLOAT32 ? 4 : 2, x = reinterpret_cast<uintptr_t>(c.x), y = reinterpret_cast<uintptr_t>(c.y);
    if ((x | y) % size) {
        return "logits must lie on their own size";
    }
    const uintptr_t x_bytes = uintptr_t((c.rows - 1) * c.x_stride + c.width) * size, y_bytes = uintptr_t((c.rows - 1) * c.y_stride + c.width) * size;
    if (x == y ? c.rows > 1 && c.x_stride != c.y_stride : x < y + y_bytes && y < x + x_bytes) {
        return "y must be x with the same stride, or apart from it";
    }
    return nullptr;
}

}  // namespace

namespace chroma_adjust {

int launch_rows_adjust(const chroma_hip_adjust_call& c, hipStream_t stream, char* error, size_t error_size) {
    if (const char* wrong = mistake(c)) {
        return refuse(wrong, error, error_size);
    }
    const dim3 grid(unsigned((c.width + kSpan - 1) / kSpan), unsigned(c.rows));
    if (c.dtype == CHROMA_HIP_FLOAT32) {
        rows_adjust<float><<<grid, kThreads, 0, stream>>>(c);
    } else {
        rows_adjust<uint16_t><<<grid, kThreads, 0, stream>>>(c);
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
