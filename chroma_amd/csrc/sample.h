// Internal interface between the runtime (runtime.cpp) and the sampling kernels (sample.hip).
#pragma once

#include "../../include/chroma_hip.h"

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace chroma_sample {

// What is wrong with the call's extents, or null.
inline const char* mistake(const chroma_hip_sample_call& c) {
    if (c.dtype != CHROMA_HIP_FLOAT32 && c.dtype != CHROMA_HIP_BFLOAT16) {
        return "dtype must be CHROMA_HIP_FLOAT32 or CHROMA_HIP_BFLOAT16";
    }
    if (c.rows < 1 || c.rows > 65535 || c.width < 1 || c.width > (int64_t(1) << 19)) {  // sums of 2^19 weights fit 64 bits
        return "want 1 to 65535 rows of 1 to 524288 logits";
    }
    if (c.x_stride < c.width || c.x_stride > (int64_t(1) << 40)) {
        return "x_stride out of range";
    }
    return nullptr;
}

// Queue ``call`` on ``stream``, with the scratch that chroma_hip_rows_sample_workspace asks for. Returns a CHROMA_HIP_* status and
// writes a message on failure. (Weak: the runtime links without the kernels where nothing samples.)
__attribute__((weak)) size_t workspace_bytes(const chroma_hip_sample_call& call);
__attribute__((weak)) int launch_rows_sample(const chroma_hip_sample_call& call, void* workspace, size_t workspace_bytes, hipStream_t stream,
                                             char* error, size_t error_size);

}  // namespace chroma_sample
