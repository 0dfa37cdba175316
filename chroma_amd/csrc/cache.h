// Internal interface between the runtime (runtime.cpp) and the cache row copies (cache.hip).
#pragma once

#include "../../include/chroma_hip.h"

#include <hip/hip_runtime_api.h>

namespace chroma_cache {

// Queue the moves on ``stream`` (see chroma_hip_cache_move). Returns a CHROMA_HIP_* status and writes a message on failure.
int launch_cache_move(const chroma_hip_cache_rows* to, const chroma_hip_cache_rows* from, int64_t layers, int64_t row_bytes,
                      const int64_t* moves, int64_t count, hipStream_t stream, char* error, size_t error_size);

}  // namespace chroma_cache
