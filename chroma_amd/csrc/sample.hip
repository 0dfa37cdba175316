// ``chroma_hip_rows_sample``: a token drawn from each row of logits under temperature, top-k, top-p and min-p.
//
// Every filter keeps a prefix of the row's descending order, and the drawn token is a place in it, so that all of them ask the
// same question: after which token does a running count, or a running sum of weights, reach a goal. It is answered by
// descending on the order's 32-bit key (larger means earlier), a histogram of counts and weights per step.
//
// A weight exp((x - max) / temperature) is evaluated in 64 bits and rounded to units of 2^-44: sums are integers, and the same
// in whatever order they are taken. In 32 bits the place that a random number names among 200,000 tokens moves by more than
// some tokens hold.
#include "../../include/chroma_hip.h"

#include <hip/hip_runtime.h>

#include <chroma_hip/device.h>

#include "ranges.h"

#include <cstdint>
#include <cstdio>

namespace {

using Call = chroma_hip_sample_call;

constexpr int kOne = 44;  // a weight of 1 is 2^kOne
constexpr uint32_t kThreads = 1024, kBuckets = 2048;

template <class T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<uint16_t>(uint16_t v) { return chroma::bf16_to_f32(v); }

__device__ __forceinline__ uint32_t order_of(float v) { return uint32_t(chroma::topk_key(v, 0u, true) >> 32); }
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

// Weights of one row, relative to its largest logit. An infinite largest one leaves the others nothing.
struct Weights {
    double top, rate;  // rate: log2(e) / temperature
    __device__ __forceinline__ Weights(float top, float temperature)
        : top(double(top)), rate(1.4426950408889634074 / double(temperature)) {}
    // log2 of the inverse weight, 0 or more
    __device__ __forceinline__ double depth(float x) const { return double(x) == top ? 0.0 : (top - double(x)) * rate; }
    __device__ __forceinline__ uint64_t operator()(float x) const {
        const double y = depth(x);
        if (!(y < double(kOne + 1))) {
            return 0u;
        }
        // 2^-y = 2^-n 2^-f, |f| <= 1/2: the series of exp(-f ln 2) to the 12th power (the 13th is below 2^-52)
        const double n = __builtin_rint(y), f = (n - y) * 0.69314718055994530942;
        double p = 1.0 / 479001600.0;
        p = __builtin_fma(p, f, 1.0 / 39916800.0);
        p = __builtin_fma(p, f, 1.0 / 3628800.0);
        p = __builtin_fma(p, f, 1.0 / 362880.0);
        p = __builtin_fma(p, f, 1.0 / 40320.0);
        p = __builtin_fma(p, f, 1.0 / 5040.0);
        p = __builtin_fma(p, f, 1.0 / 720.0);
        p = __builtin_fma(p, f, 1.0 / 120.0);
        p = __builtin_fma(p, f, 1.0 / 24.0);
        p = __builtin_fma(p, f, 1.0 / 6.0);
        p = __builtin_fma(p, f, 0.5);
        p = __builtin_fma(p, f, 1.0);
        p = __builtin_fma(p, f, 1.0);
        const double scale = __longlong_as_double(int64_t(1023 + kOne - int(n)) << 52);
        // (adding 2^52 rounds to a whole number, which then lies in the low bits)
        return uint64_t(__double_as_longlong(__builtin_fma(p, scale, 4503599627370496.0))) & 0xfffffffffffffull;
    }
};

// floor(sum * v) and the remainder's being there, of a float v in (0, 1).
__device__ __forceinline__ uint64_t share_of(uint64_t sum, float v, bool& more) {
    const uint32_t bits = __float_as_uint(v);
    const int exponent = int(bits >> 23), shift = 150 - (exponent ? exponent : 1);  // v = mantissa 2^-shift
    const uint64_t mantissa = (bits & 0x7fffffu) | (exponent ? 0x800000u : 0u);
    const unsigned __int128 product = static_cast<unsigned __int128>(sum) * mantissa;
    if (shift >= 128) {
        more = product != 0;
        return 0u;
    }
    const unsigned __int128 whole = product >> shift;
    more = (whole << shift) != product;
    return uint64_t(whole);
}

struct Sums {
    uint64_t weight;
    uint32_t count;
};

// A place in the descending order: the tokens before those of key ``order``, and how many of those.
struct Place {
    uint32_t order, ties;
    Sums before;
    uint64_t each;  // weight of one of them
    __device__ __forceinline__ uint64_t count() const { return uint64_t(before.count) + ties; }
    __device__ __forceinline__ uint64_t weight() const { return before.weight + each * ties; }
};

template <class T> struct Row {
    const T* x;
    uint32_t width;
    uint64_t (*weight)[kBuckets];  // [2][kBuckets], LDS: the first step's histogram and the later ones'
    uint32_t (*count)[kBuckets];
    Sums* waves;  // [kThreads / 64]
    Place* found;

    // Sums of the tokens whose order is ``prefix`` above its bits [shift, shift + bits), by those bits.
    __device__ void histogram(const Weights& w, uint32_t which, uint32_t prefix, uint32_t shift, uint32_t bits) {
        for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
            weight[which][i] = 0u;
            count[which][i] = 0u;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < width; i += kThreads) {
            const float v = widen<T>(x[i]);
            const uint32_t order = order_of(v);
            if (uint64_t(order) >> (shift + bits) == prefix) {
                const uint32_t bucket = (order >> shift) & ((1u << bits) - 1u);
                const uint64_t mine = w(v);
                atomicAdd(&count[which][bucket], 1u);
                if (mine) {
                    atomicAdd(reinterpret_cast<unsigned long long*>(&weight[which][bucket]), static_cast<unsigned long long>(mine));
                }
            }
        }
        __syncthreads();
    }

    // The highest bucket at whose end the sums before it and those down to it reach the goal, and the sums above it.
    __device__ uint32_t descend(uint32_t which, bool by_count, uint64_t goal, Sums& before) {
        constexpr uint32_t PER = kBuckets / kThreads;
        const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u, top = kBuckets - 1u - threadIdx.x * PER;
        Sums own{0u, 0u};
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            own.weight += weight[which][top - k];
            own.count += count[which][top - k];
        }
        Sums upto = own;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const uint64_t ww = __shfl_up(static_cast<unsigned long long>(upto.weight), step, 64);
            const uint32_t cc = __shfl_up(upto.count, step, 64);
            if (lane >= uint32_t(step)) {
                upto.weight += ww;
                upto.count += cc;
            }
        }
        if (lane == 63u) {
            waves[wave] = upto;
        }
        __syncthreads();
        Sums at = before;
        for (uint32_t w = 0; w < wave; ++w) {
            at.weight += waves[w].weight;
            at.count += waves[w].count;
        }
        at.weight += upto.weight - own.weight;
        at.count += upto.count - own.count;
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            const Sums next{at.weight + weight[which][top - k], at.count + count[which][top - k]};
            const uint64_t reached = by_count ? next.count : next.weight, short_of = by_count ? at.count : at.weight;
            if (reached >= goal && short_of < goal) {  // one thread
                found->order = top - k;
                found->before = at;
            }
            at = next;
        }
        __syncthreads();
        before = found->before;
        const uint32_t bucket = found->order;
        __syncthreads();
        return bucket;
    }

    // The place at which a count or a sum of weights reaches ``goal``, from 1 to all there is.
    __device__ Place reach(const Weights& w, bool by_count, uint64_t goal) {
        Place p;
        p.before = Sums{0u, 0u};
        const uint32_t high = descend(0u, by_count, goal, p.before);
        histogram(w, 1u, high, 10u, 11u);
        const uint32_t middle = high << 11 | descend(1u, by_count, goal, p.before);
        histogram(w, 1u, middle, 0u, 10u);
        p.order = middle << 10 | descend(1u, by_count, goal, p.before);
        p.each = w(value_of(p.order));
        const uint64_t left = goal - (by_count ? p.before.count : p.before.weight);
        p.ties = uint32_t(by_count ? left : (left + p.each - 1u) / p.each);
        return p;
    }

    // Sums over the workgroup.
    __device__ Sums all(Sums own) {
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            own.weight += __shfl_xor(static_cast<unsigned long long>(own.weight), step, 64);
            own.count += __shfl_xor(own.count, step, 64);
        }
        if (threadIdx.x % 64u == 0u) {
            waves[threadIdx.x / 64u] = own;
        }
        __syncthreads();
        Sums sum{0u, 0u};
        for (uint32_t v = 0; v < kThreads / 64u; ++v) {
            sum.weight += waves[v].weight;
            sum.count += waves[v].count;
        }
        __syncthreads();
        return sum;
    }

    // The largest logit's order and id, as a selection key.
    __device__ uint64_t largest() {
        uint64_t best = 0;
        for (uint32_t i = threadIdx.x; i < width; i += kThreads) {
            const uint64_t key = chroma::topk_key(widen<T>(x[i]), i, true);
            best = key > best ? key : best;
        }
        best = chroma::wave_max_u64(best);
        if (threadIdx.x % 64u == 0u) {
            waves[threadIdx.x / 64u].weight = best;
        }
        __syncthreads();
        for (uint32_t v = 0; v < kThreads / 64u; ++v) {
            best = waves[v].weight > best ? waves[v].weight : best;
        }
        __syncthreads();
        return best;
    }

    // The id of the ``nth`` token of this order, from 1 on, by id: every wave counts a span, one looks it up.
    __device__ void id_of(uint32_t order, uint32_t nth, int64_t* id) {
        const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u, span = (width + kThreads - 1u) / kThreads * 64u;
        const uint32_t begin = min(wave * span, width), end = min(begin + span, width);
        const auto matches = [&](uint32_t i) { return __ballot(i + lane < end && order_of(widen<T>(x[min(i + lane, width - 1u)])) == order); };
        uint32_t own = 0;
        for (uint32_t i = begin; i < end; i += 64u) {
            own += __popcll(matches(i));
        }
        if (lane == 0u) {
            waves[wave].count = own;
        }
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t v = 0; v < wave; ++v) {
            before += waves[v].count;
        }
        if (before < nth && nth <= before + own) {
            for (uint32_t i = begin; i < end; i += 64u) {
                const unsigned long long some = matches(i);
                const uint32_t here = __popcll(some);
                if (nth <= before + here) {
                    if (((some >> lane) & 1ull) && before + __popcll(some & ((2ull << lane) - 1ull)) == nth) {
                        *id = int64_t(i + lane);
                    }
                    break;
                }
                before += here;
            }
        }
    }
};

// grid: rows
template <class T> __global__ void __launch_bounds__(kThreads) sample_rows(Call c) {
    __shared__ uint64_t weight[2][kBuckets];
    __shared__ uint32_t count[2][kBuckets];
    __shared__ Sums waves[kThreads / 64u];
    __shared__ Place found;
    const uint64_t r = blockIdx.x;
    Row<T> row{static_cast<const T*>(c.x) + r * uint64_t(c.x_stride), uint32_t(c.width), weight, count, waves, &found};
    const float temperature = c.temperature ? c.temperature[r] : 1.0f;
    const uint64_t best = row.largest();
    const uint32_t order = uint32_t(best >> 32);
    const float top = value_of(order);
    if (order == 0xffffffffu || top == -__builtin_inff() || !(temperature > 0.0f)) {
        if (threadIdx.x == 0u) {
            const bool nan = order == 0xffffffffu, nothing = !nan && top == -__builtin_inff();
            c.ids[r] = nothing ? -1 : int64_t(0xffffffffu - uint32_t(best));
            if (c.logprobs) {
                c.logprobs[r] = nan ? __builtin_nanf("") : nothing ? top : 0.0f;
            }
        }
        return;
    }
    const Weights w(top, temperature);
    row.histogram(w, 0u, 0u, 21u, 11u);
    Sums own{0u, 0u};
    for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
        own.weight += weight[0][i];
        own.count += count[0][i];
    }
    Sums kept = row.all(own);
    const int64_t k = c.top_k ? c.top_k[r] : 0;
    if (k > 0 && k < c.width) {
        const Place p = row.reach(w, true, uint64_t(k));
        kept = Sums{p.weight(), uint32_t(p.count())};
    }
    const float top_p = c.top_p ? c.top_p[r] : 1.0f;
    if (top_p < 1.0f) {
        bool more = false;
        const uint64_t whole = top_p > 0.0f ? share_of(kept.weight, top_p, more) : 0u;
        const uint64_t goal = whole + (more ? 1u : 0u);
        const Place p = row.reach(w, false, goal ? goal : 1u);
        kept = Sums{p.weight(), uint32_t(p.count())};
    }
    const float min_p = c.min_p ? c.min_p[r] : 0.0f;
    if (min_p > 0.0f) {
        const double least = __builtin_ceil(double(min_p > 2.0f ? 2.0f : min_p) * double(1ull << kOne));
        const uint64_t floor = uint64_t(least);
        own = Sums{0u, 0u};
        for (uint32_t i = threadIdx.x; i < row.width; i += kThreads) {
            const uint64_t mine = w(widen<T>(row.x[i]));
            own.weight += mine >= floor ? mine : 0u;
            own.count += mine >= floor ? 1u : 0u;
        }
        Sums high = row.all(own);
        if (!high.count) {
            high = Sums{1ull << kOne, 1u};
        }
        kept = high.count < kept.count ? high : kept;
    }
    const float given = c.uniform[r];
    bool more = false;
    const uint64_t goal = 1u + (given > 0.0f ? share_of(kept.weight, given < 1.0f ? given : __uint_as_float(0x3f7fffffu), more) : 0u);
    const Place drawn = row.reach(w, false, goal);
    row.id_of(drawn.order, drawn.ties, c.ids + r);
    if (threadIdx.x == 0u && c.logprobs) {
        const double share = double(kept.weight) * (1.0 / double(1ull << kOne));
        c.logprobs[r] = float(-w.depth(value_of(drawn.order)) * 0.69314718055994530942 - log(share));
    }
}

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "rows_sample: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

// What is wrong with the call's extents, or null.
const char* mistake(const Call& c) {
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

}  // namespace

extern "C" {

__attribute__((visibility("default"))) size_t chroma_hip_rows_sample_workspace(const Call* call) {
    return 0;
}

__attribute__((visibility("default"))) int chroma_hip_rows_sample(const Call* call, void* workspace, size_t workspace_bytes, void* stream,
                                                                  char* error, size_t error_size) {
    if (!call) {
        return refuse("null call", error, error_size);
    }
    const Call& c = *call;
    if (const char* wrong = mistake(c)) {
        return refuse(wrong, error, error_size);
    }
    if (!c.x || !c.uniform || !c.ids) {
        return refuse("null device pointer", error, error_size);
    }
    const uint64_t size = c.dtype == CHROMA_HIP_FLOAT32 ? 4 : 2, n = uint64_t(c.rows);
    if (reinterpret_cast<uintptr_t>(c.x) % size) {
        return refuse("logits must lie on their own size", error, error_size);
    }
    const size_t need = chroma_hip_rows_sample_workspace(call);
    if (need && (!workspace || workspace_bytes < need)) {
        return refuse("workspace smaller than chroma_hip_rows_sample_workspace", error, error_size);
    }
    if (need && (reinterpret_cast<uintptr_t>(workspace) & 15u)) {
        return refuse("the workspace must start on 16 bytes", error, error_size);
    }
    const chroma_ranges::Range ranges[] = {
        {c.ids, n * 8u, true}, {c.logprobs, n * 4u, true}, {workspace, need, true}, {c.x, ((n - 1u) * uint64_t(c.x_stride) + uint64_t(c.width)) * size, false},
        {c.temperature, n * 4u, false}, {c.top_k, n * 8u, false}, {c.top_p, n * 4u, false}, {c.min_p, n * 4u, false}, {c.uniform, n * 4u, false}};
    if (chroma_ranges::overlap(ranges)) {
        return refuse("ids, logprobs or the workspace overlap another array", error, error_size);
    }
    if (c.dtype == CHROMA_HIP_FLOAT32) {
        sample_rows<float><<<unsigned(c.rows), kThreads, 0, static_cast<hipStream_t>(stream)>>>(c);
    } else {
        sample_rows<uint16_t><<<unsigned(c.rows), kThreads, 0, static_cast<hipStream_t>(stream)>>>(c);
    }
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? CHROMA_HIP_OK : refuse(hipGetErrorString(status), error, error_size);
}

}  // extern "C"
