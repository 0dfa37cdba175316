// Internal interface between the runtime (runtime.cpp) and the logit adjustment kernel (adjust.hip).
#pragma once

#include "../../include/chroma_hip.h"

#include <hip/hip_runtime_api.h>

namespace chroma_adjust {

// Queue ``call`` on ``stream``. Returns a CHROMA_HIP_* status and writes a message on failure.
int launch_rows_adjust(const chroma_hip_adjust_call& call, hipStream_t stream, char* error, size_t error_size);

}  // namespace chroma_adjust
