// Internal interface between the runtime (runtime.cpp) and the logit adjustment kernel (adjust.hip).
#pragma once

#include "../../include/chroma_hip.h"

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace chroma_adjust {

// What is wrong with the call, or null.
inline const char* mistake(const chroma_hip_adjust_call& c) {
    if (c.dtype != CHROMA_HIP_FLOAT32 && c.dtype != CHROMA_HIP_BFLOAT16) {
        return "dtype must be CHROMA_HIP_FLOAT32 or CHROMA_HIP_BFLOAT16";
    }
    if (c.rows < 1 || c.rows > 65535 || c.width < 1 || c.width >= int64_t(1) << 31) {
        return "want 1 to 65535 rows of 1 to 2147483647 logits";
    }
    constexpr int64_t kStride = int64_t(1) << 40;
    if (c.x_stride > kStride || c.y_stride > kStride || c.history_stride > kStride || c.bias_stride > kStride || c.mask_stride > kStride) {
        return "a stride is out of range";
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

// Queue ``call`` on ``stream``. Returns a CHROMA_HIP_* status and writes a message on failure.
int launch_rows_adjust(const chroma_hip_adjust_call& call, hipStream_t stream, char* error, size_t error_size);

}  // namespace chroma_adjust
