// Host-memory stand-in for the HIP calls and kernels behind chroma_amd/csrc/runtime.cpp, so that the runtime's own logic
// (staging, scratch, captured graphs) runs and is counted without a GPU. Device memory is host memory, streams finish at
// once, a captured graph is the list of what was queued. A plan kernel ``copy_<bytes>`` copies from its first argument to
// its second; row selection and logit adjustment are plain loops over float rows.
#include "../chroma_amd/csrc/adjust.h"
#include "../chroma_amd/csrc/cache.h"
#include "../chroma_amd/csrc/copy.h"
#include "../chroma_amd/csrc/masks.h"
#include "../chroma_amd/csrc/select.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <limits>
#include <numeric>
#include <string>
#include <vector>

namespace {

using Work = std::vector<std::function<void()>>;
Work* recording = nullptr;
int64_t counts[4];  // device allocations, page-locked allocations, instantiated graphs, plan kernels and moves run

void queue(std::function<void()> work) {
    if (recording) {
        recording->push_back(std::move(work));
    } else {
        work();
    }
}

}  // namespace

extern "C" {

__attribute__((visibility("default"))) void stub_counts(int64_t* out) { std::copy(counts, counts + 4, out); }

hipError_t hipGetDevice(int* device) { return *device = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t* p, int) { return std::memset(p, 0, sizeof *p), std::strcpy(p->name, "stub"), hipSuccess; }
hipError_t hipDeviceGetAttribute(int* value, hipDeviceAttribute_t, int) { return *value = 1, hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipMalloc(void** p, size_t bytes) { return ++counts[0], *p = std::aligned_alloc(256, (bytes + 255) / 256 * 256), hipSuccess; }
hipError_t hipHostMalloc(void** p, size_t bytes, unsigned) { return ++counts[1], *p = std::calloc(1, bytes), hipSuccess; }
hipError_t hipFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipHostFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipMemcpy(void* to, const void* from, size_t n, hipMemcpyKind) { return std::memcpy(to, from, n), hipSuccess; }
hipError_t hipMemcpyAsync(void* to, const void* from, size_t n, hipMemcpyKind, hipStream_t) { return std::memcpy(to, from, n), hipSuccess; }
hipError_t hipMemcpy2DAsync(void*, size_t, const void*, size_t, size_t, size_t, hipMemcpyKind, hipStream_t) { return hipErrorNotSupported; }
// addresses from 2^60 on stand for memory of device 1, and those below 4096 for memory that HIP does not know
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* a, const void* p) {
    std::memset(a, 0, sizeof *a);
    a->type = hipMemoryTypeDevice;
    a->device = reinterpret_cast<uintptr_t>(p) >> 60 ? 1 : 0;
    return reinterpret_cast<uintptr_t>(p) < 4096 ? hipErrorInvalidValue : hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipMemset(void* p, int value, size_t n) { return std::memset(p, value, n), hipSuccess; }
hipError_t hipMemsetAsync(void* p, int value, size_t n, hipStream_t) { return std::memset(p, value, n), hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = nullptr, hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { return *e = nullptr, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return *e = nullptr, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 0.0f, hipSuccess; }
hipError_t hipModuleLoad(hipModule_t*, const char*) { return hipSuccess; }
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t, const char* name) {
    return *f = reinterpret_cast<hipFunction_t>(std::strtoull(name + sizeof("copy_") - 1, nullptr, 10)), hipSuccess;
}
hipError_t hipModuleOccupancyMaxActiveBlocksPerMultiprocessor(int* n, hipFunction_t, int, size_t) { return *n = 1, hipSuccess; }
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, hipStream_t, void** arguments,
                                 void**) {
    const void* from = *static_cast<void**>(arguments[0]);
    void* to = *static_cast<void**>(arguments[1]);
    queue([=] { ++counts[3], std::memcpy(to, from, reinterpret_cast<size_t>(f)); });
    return hipSuccess;
}
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) { return recording = new Work, hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) { return *g = reinterpret_cast<hipGraph_t>(recording), recording = nullptr, hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t g, hipGraphNode_t*, char*, size_t) {
    return ++counts[2], *e = reinterpret_cast<hipGraphExec_t>(new Work(*reinterpret_cast<Work*>(g))), hipSuccess;
}
hipError_t hipGraphLaunch(hipGraphExec_t e, hipStream_t) {
    for (const auto& work : *reinterpret_cast<Work*>(e)) {
        work();
    }
    return hipSuccess;
}
hipError_t hipGraphDestroy(hipGraph_t g) { return delete reinterpret_cast<Work*>(g), hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t e) { return delete reinterpret_cast<Work*>(e), hipSuccess; }

}  // extern "C"

namespace chroma_select {
size_t workspace_bytes(size_t, size_t, int) { return 64; }
int launch_rows_topk(const void* x, int, size_t rows, size_t width, int k, int, void* values, int64_t* ids, void*, size_t, hipStream_t, char*, size_t) {
    queue([=] {
        for (size_t r = 0; r < rows; ++r) {
            const float* row = static_cast<const float*>(x) + r * width;
            std::vector<int64_t> order(width);
            std::iota(order.begin(), order.end(), 0);
            std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return row[a] > row[b]; });
            for (int i = 0; i < k; ++i) {
                ids[r * k + i] = order[i];
                static_cast<float*>(values)[r * k + i] = row[order[i]];
            }
        }
    });
    return 0;
}
}  // namespace chroma_select

namespace chroma_adjust {
int launch_rows_adjust(const chroma_hip_adjust_call& c, hipStream_t, char* error, size_t size) {
    if (const char* wrong = mistake(c)) {
        return std::snprintf(error, size, "%s", wrong), CHROMA_HIP_RUNTIME_ERROR;
    }
    for (int64_t r = 0; r < c.rows; ++r) {
        const float* x = static_cast<const float*>(c.x) + r * c.x_stride;
        float* y = static_cast<float*>(c.y) + r * c.y_stride;
        const int64_t length = !c.history ? 0 : c.history_lengths ? std::clamp<int64_t>(c.history_lengths[r], 0, c.history_width) : c.history_width;
        std::vector<int> times(c.width);
        for (int64_t i = 0; i < length; ++i) {
            const int64_t id = c.history[r * c.history_stride + i];
            if (id >= 0 && id < c.width) {
                ++times[id];
            }
        }
        for (int64_t v = 0; v < c.width; ++v) {
            float value = x[v];
            if (times[v]) {
                const float factor = c.repetition ? c.repetition[r] : 1.0f;
                value = value > 0.0f ? value / factor : value * factor;
                value -= (c.presence ? c.presence[r] : 0.0f) + (c.frequency ? c.frequency[r] : 0.0f) * float(times[v]);
            }
            if (c.bias) {
                value += c.bias[r * c.bias_stride + v];
            }
            const bool allowed = !c.mask || (c.mask[r * c.mask_stride + v / 32] >> (v % 32) & 1u);
            y[v] = allowed ? value : -std::numeric_limits<float>::infinity();
        }
    }
    return 0;
}
}  // namespace chroma_adjust

namespace chroma_copy {
int launch_copy_rects(const Rect*, int, hipStream_t, char*, size_t) { return CHROMA_HIP_RUNTIME_ERROR; }
}
namespace chroma_masks {
int launch_decoder_masks(const int64_t*, int64_t, int64_t, int64_t, int64_t, bool, void*, void*, hipStream_t, char*, size_t) { return CHROMA_HIP_RUNTIME_ERROR; }
}
namespace chroma_cache {
int launch_cache_move(const chroma_hip_cache_rows*, const chroma_hip_cache_rows*, int64_t, int64_t, const int64_t*, int64_t, hipStream_t, char*, size_t) {
    return ++counts[3], CHROMA_HIP_OK;
}
}
