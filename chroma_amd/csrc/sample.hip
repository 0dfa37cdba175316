// ``chroma_hip_rows_sample``: a token drawn from each row of logits under temperature, top-k, top-p and min-p.
//
// Every filter keeps a prefix of the row's descending order, and the drawn token is a place in it, so that all of them ask the
// same question: after which token does a running count, or a running sum of weights, reach a goal. A histogram of weights
// (of counts where a top-k cuts the row) over the depths below the maximum answers it but for the tokens of a few buckets;
// those are listed, and the places among them found by descending on their keys. A row is read three times: for its ends, by which
// the buckets are spread over the depths that it has, for the histogram, for the list; the second and third time it lies in the
// caches.
//
// Narrow rows have a workgroup each and one launch. Wide ones are cut into spans, and the three readings are launches of their
// own; the workgroup that comes last with a row's histogram decides what is listed, and a fourth launch draws. Rows of up to kList tokens
// are listed whole. Where the listed buckets hold more than kList tokens (rows of few values), a workgroup descends on the
// keys of the whole row.
//
// What bounds it: one row of 201088 float logits (28 us) the four launches' chains (3.6, 14, 4.1 and 7.1 us; of the second
// 3 are the span's weights and 8 the sum of 24 spans' histograms and the cuts); 256 rows of 100003 (86 us) the weights' vector work:
// 31 instructions a token, 36 us, where the first reading takes 19-21 (5 TB/s), the third 22 and the token 10.
//
// A weight exp((x - max) / temperature) is evaluated in 64 bits and rounded to units of 2^-44: sums are integers, and the same
// in whatever order they are taken. In 32 bits the place that a random number names among 200,000 tokens moves by more than
// some tokens hold.
#include "sample.h"

#include <hip/hip_runtime.h>

#include <chroma_hip/device.h>

#include "ranges.h"

#include <cstdint>
#include <cstdio>

namespace {

using Call = chroma_hip_sample_call;

constexpr int kOne = 44;                        // a weight of 1 is 2^kOne
constexpr uint64_t kWhole = uint64_t(1) << kOne;
constexpr uint32_t kThreads = 512, kBuckets = 2048, kPer = kBuckets / kThreads;
constexpr uint32_t kList = 4096;   // listed tokens of a row
constexpr int64_t kMostTop = 1024;  // a larger top_k descends on the whole row
constexpr float kDepths = 44.0f;   // buckets of the histogram for a factor of 2, where not all of a row lies in fewer factors
constexpr float kFinest = 65536.0f;  // and at most: more would not be exact in float
constexpr int kDeepest = 64;       // depths (in factors of 2) past which weights are not evaluated; from kOne + 1 on they are 0
static_assert(float(kBuckets) < kDepths * float(kDeepest - 1) && float(kBuckets - 1u) > kDepths * float(kOne + 2), "buckets");

__device__ __forceinline__ uint64_t lesser(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t greater(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <class T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<uint16_t>(uint16_t v) { return chroma::bf16_to_f32(v); }

__device__ __forceinline__ uint32_t order_of(float v) { return uint32_t(chroma::topk_key(v, 0u, true) >> 32); }
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

// 2^(i / 256) and 2^(i / 65536) of i < 256, in LDS.
struct Powers {
    double high[256], low[256];
    __device__ __forceinline__ void fill() {
        if (threadIdx.x < 512u) {
            const uint32_t i = threadIdx.x % 256u;
            // the series of exp(f ln 2), |f| <= 1/2, to the 12th power (the 13th is below 2^-52)
            const double y = double(i) * (threadIdx.x < 256u ? 1.0 / 256.0 : 1.0 / 65536.0), n = __builtin_rint(y), f = (y - n) * 0.69314718055994530942;
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
            (threadIdx.x < 256u ? high : low)[i] = n == 1.0 ? 2.0 * p : p;
        }
        __syncthreads();
    }
};

// Weights of one row, relative to its largest logit. An infinite largest one leaves the others nothing.
struct Weights {
    const Powers& powers;
    double top, rate;  // rate: 65536 log2(e) / temperature
    __device__ __forceinline__ Weights(const Powers& powers, float top, float temperature)
        : powers(powers), top(double(top)), rate(65536.0 * 1.4426950408889634074 / double(temperature)) {}
    // The weight of a logit of finite depth, at most kDeepest.
    __device__ __forceinline__ uint64_t near(float x) const {
        // log2 of the weight in units of 2^-16 is n + f, n whole (adding 1.5 2^52 rounds, and n then lies in the low bits:
        // conversions are slow); 2^(n >> 16), 2^(its next 8 bits / 256) and 2^(the last 8 / 65536) from the powers,
        // exp(f ln 2 / 65536) from three terms of its series.
        constexpr double c = 0.69314718055994530942 / 65536.0, whole = 6755399441055744.0;
        const double d = double(x) - top, sum = __builtin_fma(d, rate, whole), f = __builtin_fma(d, rate, whole - sum);
        const double p = __builtin_fma(f, __builtin_fma(f, 0.5 * c * c, c), 1.0);
        const uint32_t n = uint32_t(__double_as_longlong(sum));
        const double scale = __hiloint2double(int(((n & 0xffff0000u) << 4) + ((1023u + kOne) << 20)), 0);
        const double all = powers.high[(n >> 8) & 255u] * powers.low[n & 255u] * p;
        return uint64_t(__double_as_longlong(__builtin_fma(all, scale, 4503599627370496.0))) & 0xfffffffffffffull;
    }
    // log2 of the inverse weight, 0 or more
    __device__ __forceinline__ double depth(float x) const { return double(x) == top ? 0.0 : (top - double(x)) * (rate * (1.0 / 65536.0)); }
    __device__ __forceinline__ uint64_t operator()(float x) const {
        return double(x) == top ? kWhole : depth(x) < double(kDeepest) ? near(x) : 0u;
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

// LDS of a workgroup that takes a histogram, and of one that draws.
struct Waves {
    Sums waves[kThreads / 64u];
    uint32_t last;
};
struct Depths : Waves {  // (at most 40 KB: four workgroups of a compute unit)
    uint64_t weight[kBuckets];
    uint64_t before[kBuckets + 1];  // sums before each bucket, and of all
    Powers powers;
    __device__ __forceinline__ uint32_t* counts() { return reinterpret_cast<uint32_t*>(before); }
};
static_assert(sizeof(Depths) <= 40u * 1024u, "LDS");
struct Shared : Depths {
    uint32_t count[kBuckets];
    uint64_t list[kList];  // selection keys
    uint64_t few[64];
    uint64_t ends[kThreads / 64u];
    Place found;
    uint32_t listed, fews;
};

// LDS of a workgroup that only lists.
struct Gathered {
    uint64_t list[kList];
    uint32_t listed, begin;
};

// Running sums over a wave's lanes without LDS: DPP shifts inside rows of 16 lanes, then the last lane of the rows before.
// (A shift's lanes without a source receive 0.)
template <int Control, int Rows> __device__ __forceinline__ uint32_t dpp_from(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), Control, Rows, 0xF, false));
}
template <int Control, int Rows> __device__ __forceinline__ uint64_t dpp_from(uint64_t v) {
    return uint64_t(dpp_from<Control, Rows>(uint32_t(v >> 32))) << 32 | dpp_from<Control, Rows>(uint32_t(v));
}
template <class V> __device__ __forceinline__ V wave_scan(V v) {
    v += dpp_from<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v += dpp_from<0x112, 0xF>(v);
    v += dpp_from<0x114, 0xF>(v);
    v += dpp_from<0x118, 0xF>(v);
    v += dpp_from<0x142, 0xA>(v);  // row_bcast 15: rows 1 and 3
    v += dpp_from<0x143, 0xC>(v);  // row_bcast 31: rows 2 and 3
    return v;
}
// The largest of a wave's values, in all lanes (lanes without a source see 0, which is no larger).
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    const auto with = [&](uint32_t other) { v = other > v ? other : v; };
    with(dpp_from<0x111, 0xF>(v));
    with(dpp_from<0x112, 0xF>(v));
    with(dpp_from<0x114, 0xF>(v));
    with(dpp_from<0x118, 0xF>(v));
    with(dpp_from<0x142, 0xA>(v));
    with(dpp_from<0x143, 0xC>(v));
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, uint32_t lane) {
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(v >> 32), lane))) << 32 | uint32_t(__builtin_amdgcn_readlane(uint32_t(v), lane));
}
__device__ __forceinline__ uint64_t wave_total(uint64_t v) { return lane_u64(wave_scan(v), 63u); }
// The largest: by the high words, then by the low words of those that have the largest one.
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    const uint32_t high = wave_max(uint32_t(v >> 32)), low = wave_max(uint32_t(v >> 32) == high ? uint32_t(v) : 0u);
    return uint64_t(high) << 32 | low;
}

// Sums over the workgroup.
__device__ Sums sum_all(Waves& s, Sums own) {
    const Sums wave{wave_total(own.weight), uint32_t(__builtin_amdgcn_readlane(wave_scan(own.count), 63))};
    if (threadIdx.x % 64u == 0u) {
        s.waves[threadIdx.x / 64u] = wave;
    }
    __syncthreads();
    Sums sum{0u, 0u};
#pragma unroll
    for (uint32_t v = 0; v < kThreads / 64u; ++v) {
        sum.weight += s.waves[v].weight;
        sum.count += s.waves[v].count;
    }
    __syncthreads();
    return sum;
}

// The largest of the workgroup's values.
__device__ uint64_t max_all(Waves& s, uint64_t own) {
    own = wave_max(own);
    if (threadIdx.x % 64u == 0u) {
        s.waves[threadIdx.x / 64u].weight = own;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t v = 0; v < kThreads / 64u; ++v) {
        own = s.waves[v].weight > own ? s.waves[v].weight : own;
    }
    __syncthreads();
    return own;
}

// Inclusive sums over the workgroup's threads, in their order.
__device__ Sums scan_all(Waves& s, Sums own) {
    const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u;
    own.weight = wave_scan(own.weight);
    own.count = wave_scan(own.count);
    if (lane == 63u) {
        s.waves[wave] = own;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t v = 0; v + 1u < kThreads / 64u; ++v) {
        own.weight += v < wave ? s.waves[v].weight : 0u;
        own.count += v < wave ? s.waves[v].count : 0u;
    }
    __syncthreads();
    return own;
}

// f(value, id) of the tokens [begin, end), 16 bytes of them a load, several under way.
template <class T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Several {
    T v[N];
};
template <class T, class F> __device__ __forceinline__ void visit(const T* x, uint32_t begin, uint32_t end, F f) {
    constexpr uint32_t N = 16u / sizeof(T), AHEAD = 16u / N;
    using Vector = Several<T, N>;
    const uint32_t vectors = (end - begin) / N;
    const auto at = [&](uint32_t v) { return *reinterpret_cast<const Vector*>(x + begin + v * N); };
    const auto take = [&](const Vector& some, uint32_t v) {
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) {
            f(widen<T>(some.v[e]), begin + v * N + e);
        }
    };
    for (uint32_t v = threadIdx.x; v < vectors; v += AHEAD * kThreads) {
        Vector some[AHEAD];
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {  // (clamped: a guarded load would end its branch with a wait)
            some[k] = at(min(v + k * kThreads, vectors - 1u));
        }
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
            if (v + k * kThreads < vectors) {
                take(some[k], v + k * kThreads);
            }
        }
    }
    if (const uint32_t i = begin + vectors * N + threadIdx.x; i < end) {
        f(widen<T>(x[i]), i);
    }
}

constexpr uint32_t kFinite = 0x00800000u;  // the least finite value's order

// The ends of a row: its largest logit's order and the lowest id that has it, as a selection key, and its least finite logit.
struct Ends {
    uint64_t best;
    uint32_t least;  // its order from kFinite on, inverted; 0: there is none
    __device__ __forceinline__ float low() const { return value_of(~least + kFinite); }  // (-inf)
};
// Of [begin, end).
template <class T> __device__ Ends ends_of(Waves& s, const T* x, uint32_t begin, uint32_t end) {
    uint32_t best = 0, id = 0xffffffffu, least = 0xffffffffu;
    visit(x, begin, end, [&](float v, uint32_t i) {
        const uint32_t order = order_of(v);
        id = order > best ? i : id;  // (a thread's ids ascend)
        best = order > best ? order : best;
        least = min(least, order - kFinite);  // (-inf wraps)
    });
    const Sums wave{wave_max(uint64_t(best) << 32 | uint64_t(0xffffffffu - id)), wave_max(~least)};
    if (threadIdx.x % 64u == 0u) {
        s.waves[threadIdx.x / 64u] = wave;
    }
    __syncthreads();
    Ends ends{0u, 0u};
#pragma unroll
    for (uint32_t v = 0; v < kThreads / 64u; ++v) {
        ends.best = greater(s.waves[v].weight, ends.best);
        ends.least = max(s.waves[v].count, ends.least);
    }
    __syncthreads();
    return ends;
}

// A whole row, for descending on its keys.
template <class T> struct Row {
    const T* x;
    uint32_t width;
    Shared& s;
    __device__ uint64_t* weight(uint32_t which) const { return which ? s.before : s.weight; }
    __device__ uint32_t* count(uint32_t which) const { return which ? reinterpret_cast<uint32_t*>(s.list) : s.count; }

    // Sums of the tokens whose order is ``prefix`` above its bits [shift, shift + bits), by those bits.
    __device__ void histogram(const Weights& w, uint32_t which, uint32_t prefix, uint32_t shift, uint32_t bits) {
        for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
            weight(which)[i] = 0u;
            count(which)[i] = 0u;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < width; i += kThreads) {
            const float v = widen<T>(x[i]);
            const uint32_t order = order_of(v);
            if (uint64_t(order) >> (shift + bits) == prefix) {
                const uint32_t bucket = (order >> shift) & ((1u << bits) - 1u);
                const uint64_t mine = w(v);
                atomicAdd(&count(which)[bucket], 1u);
                if (mine) {
                    atomicAdd(reinterpret_cast<unsigned long long*>(&weight(which)[bucket]), static_cast<unsigned long long>(mine));
                }
            }
        }
        __syncthreads();
    }

    // The highest bucket at whose end the sums before it and those down to it reach the goal, and the sums above it.
    __device__ uint32_t descend(uint32_t which, bool by_count, uint64_t goal, Sums& before) {
        constexpr uint32_t PER = kBuckets / kThreads;
        const uint32_t top = kBuckets - 1u - threadIdx.x * PER;
        Sums own{0u, 0u};
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            own.weight += weight(which)[top - k];
            own.count += count(which)[top - k];
        }
        const Sums upto = scan_all(s, own);
        Sums at{before.weight + upto.weight - own.weight, before.count + upto.count - own.count};
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            const Sums next{at.weight + weight(which)[top - k], at.count + count(which)[top - k]};
            const uint64_t reached = by_count ? next.count : next.weight, short_of = by_count ? at.count : at.weight;
            if (reached >= goal && short_of < goal) {  // one thread
                s.found.order = top - k;
                s.found.before = at;
            }
            at = next;
        }
        __syncthreads();
        before = s.found.before;
        const uint32_t bucket = s.found.order;
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
            s.waves[wave].count = own;
        }
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t v = 0; v < wave; ++v) {
            before += s.waves[v].count;
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

// A row's settings, and its weights.
struct Settings {
    float top, temperature, top_p, min_p, uniform;
    int64_t top_k;
    uint32_t best;  // id of the largest logit
    bool nan;
    float depths;  // buckets for a factor of 2: the last one holds what weighs nothing, the others all the rest
    __device__ __forceinline__ Settings(const Call& c, uint64_t r, const Ends& ends) : Settings(c, r, ends.best) {
        const float factors = 2.0f * 1.44269504088896341f * (0.5f * top - 0.5f * ends.low()) / temperature;
        depths = factors * kDepths < float(kBuckets - 2u) ? fminf(float(kBuckets - 2u) / factors, kFinest) : kDepths;
    }

private:
    __device__ __forceinline__ Settings(const Call& c, uint64_t r, uint64_t key)
        : temperature(c.temperature ? c.temperature[r] : 1.0f), top_p(c.top_p ? c.top_p[r] : 1.0f), min_p(c.min_p ? c.min_p[r] : 0.0f),
          uniform(c.uniform[r]), top_k(c.top_k ? c.top_k[r] : 0), best(0xffffffffu - uint32_t(key)), nan(key >> 32 == 0xffffffffu) {
        top = value_of(uint32_t(key >> 32));
        top_k = top_k >= c.width || top_k < 0 ? 0 : top_k;
    }

public:
    // Whether the largest logit decides alone; ``finish`` then writes the result.
    __device__ __forceinline__ bool greedy() const { return nan || top == -__builtin_inff() || !(temperature > 0.0f); }
    __device__ __forceinline__ void finish(const Call& c, uint64_t r) const {
        const bool nothing = !nan && top == -__builtin_inff();
        c.ids[r] = nothing ? -1 : int64_t(best);
        if (c.logprobs) {
            c.logprobs[r] = nan ? __builtin_nanf("") : nothing ? top : 0.0f;
        }
    }
    __device__ __forceinline__ Weights weights(const Depths& s) const { return Weights(s.powers, top, temperature); }
    // The histogram's bucket of a logit: it never falls as the logit falls. (Halves: the difference itself may overflow.)
    __device__ __forceinline__ uint32_t bucket(float x, float rate) const {
        return x == top ? 0u : bucket_of_finite(x, rate);
    }
    __device__ __forceinline__ uint32_t bucket_of_finite(float x, float rate) const {
        return uint32_t(fminf((0.5f * top - 0.5f * x) * rate, float(kBuckets - 1u)));
    }
    __device__ __forceinline__ float rate() const { return 2.0f * depths * 1.44269504088896341f / temperature; }
    // The sum of weights that the kept tokens of ``sum`` must reach under top_p (at least the first one's).
    __device__ __forceinline__ uint64_t nucleus(uint64_t sum) const {
        bool more = false;
        const uint64_t whole = top_p > 0.0f ? share_of(sum, top_p, more) : 0u, goal = whole + (more ? 1u : 0u);
        return goal ? goal : 1u;
    }
    // The least weight that min_p keeps.
    __device__ __forceinline__ uint64_t least() const { return uint64_t(__builtin_ceil(double(min_p > 2.0f ? 2.0f : min_p) * double(kWhole))); }
    // The sum of weights that reaches the drawn token.
    __device__ __forceinline__ uint64_t place(uint64_t kept) const {
        bool more = false;
        return 1u + (uniform > 0.0f ? share_of(kept, uniform < 1.0f ? uniform : __uint_as_float(0x3f7fffffu), more) : 0u);
    }
    __device__ __forceinline__ float logprob(const Weights& w, float x, uint64_t kept) const {
        return float(-w.depth(x) * 0.69314718055994530942 - log(double(kept) * (1.0 / double(kWhole))));
    }
};

// The token of a whole row, by descending on its keys.
template <class T> __device__ void descend_row(const Call& c, uint64_t r, const Settings& set, const T* x, Shared& s) {
    Row<T> row{x, uint32_t(c.width), s};
    const Weights w = set.weights(s);
    row.histogram(w, 0u, 0u, 21u, 11u);
    Sums own{0u, 0u};
    for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
        own.weight += s.weight[i];
        own.count += s.count[i];
    }
    uint64_t kept = sum_all(s, own).weight;
    if (set.top_k) {
        kept = row.reach(w, true, uint64_t(set.top_k)).weight();
    }
    if (set.top_p < 1.0f) {
        kept = row.reach(w, false, set.nucleus(kept)).weight();
    }
    if (set.min_p > 0.0f) {
        const uint64_t least = set.least();
        own = Sums{0u, 0u};
        visit(x, 0u, row.width, [&](float v, uint32_t) {
            const uint64_t mine = w(v);
            own.weight += mine >= least ? mine : 0u;
        });
        const uint64_t high = sum_all(s, own).weight;
        kept = lesser(kept, greater(high, kWhole));
    }
    const Place drawn = row.reach(w, false, set.place(kept));
    row.id_of(drawn.order, drawn.ties, c.ids + r);
    if (threadIdx.x == 0u && c.logprobs) {
        c.logprobs[r] = set.logprob(w, value_of(drawn.order), kept);
    }
}

// Which tokens of a row are listed: those of buckets up to ``top`` (a top-k's), or those of three ranges of buckets, in which the
// top-p's cut, the min-p's and the drawn token lie; ``whole``: none, the whole row is descended on.
struct Listing {
    uint32_t whole, by_count;
    uint32_t nucleus, least_low, least_high, drawn_low, drawn_high;
    __device__ __forceinline__ bool holds(uint32_t b) const {
        return by_count ? b <= drawn_high : b == nucleus || (b >= least_low && b <= least_high) || (b >= drawn_low && b <= drawn_high);
    }
};
constexpr uint32_t kNone = 0x7fffffffu;

// The histogram of [begin, end) in s.weight: weights, or counts where a top-k cuts the row; the last bucket's are left out (its
// tokens weigh nothing, and most of a row may lie there).
template <class T> __device__ void depths(const Settings& set, const T* x, uint32_t begin, uint32_t end, Depths& s) {
    uint32_t* counts = s.counts();
    for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
        s.weight[i] = 0u;
        counts[i] = 0u;
    }
    __syncthreads();
    const float rate = set.rate();
    if (set.top_k) {
        visit(x, begin, end, [&](float v, uint32_t) {
            const uint32_t bucket = set.bucket(v, rate);
            if (bucket < kBuckets - 1u) {
                atomicAdd(&counts[bucket], 1u);
            }
        });
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
            s.weight[i] = counts[i];
        }
    } else {
        const Weights w = set.weights(s);
        const auto add = [&](uint32_t bucket, uint64_t weight) {
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.weight[bucket]), static_cast<unsigned long long>(weight));
        };
        if (set.top == __builtin_inff()) {
            visit(x, begin, end, [&](float v, uint32_t) {
                if (v == set.top) {
                    add(0u, kWhole);
                }
            });
        } else {
            visit(x, begin, end, [&](float v, uint32_t) {
                const uint32_t bucket = set.bucket_of_finite(v, rate);
                if (bucket < kBuckets - 1u) {
                    add(bucket, w.near(v));
                }
            });
        }
    }
    __syncthreads();
}

// The bucket in which the sums reach ``goal``, from 1 to all there is.
__device__ uint32_t bucket_of(Depths& s, uint64_t goal) {
    for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
        if (s.before[i] < goal && s.before[i + 1u] >= goal) {
            s.last = i;
        }
    }
    __syncthreads();
    const uint32_t found = s.last;
    __syncthreads();
    return found;
}

// From the row's histogram in s.weight: its running sums in s.before, and what is listed.
__device__ Listing list_of(const Settings& set, Depths& s) {
    const uint32_t first = threadIdx.x * kPer;
    uint64_t own = 0;
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) {
        own += s.weight[first + k];
    }
    const uint64_t upto = scan_all(s, Sums{own, 0u}).weight;
    uint64_t sum = upto - own;
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) {
        s.before[first + k] = sum;
        sum += s.weight[first + k];
    }
    if (threadIdx.x == kThreads - 1u) {
        s.before[kBuckets] = upto;
    }
    __syncthreads();
    Listing l{0u, 0u, kNone, kNone, 0u, kNone, 0u};
    if (!(set.rate() < __builtin_inff())) {  // a temperature below 2^-121 has no depths in float
        l.whole = 1u;
        return l;
    }
    if (set.top_k) {
        l.by_count = 1u;
        // (a top-k that takes tokens of the last bucket takes all the others)
        l.drawn_high = bucket_of(s, lesser(uint64_t(set.top_k), s.before[kBuckets]));
        l.whole = set.top_k > kMostTop || s.before[l.drawn_high + 1u] > kList ? 1u : 0u;
        return l;
    }
    const uint64_t all = s.before[kBuckets];
    uint64_t low = all, high = all;  // bounds of the kept sum
    if (set.top_p < 1.0f) {
        const uint64_t goal = set.nucleus(all);
        l.nucleus = bucket_of(s, goal);
        low = goal;
        high = s.before[l.nucleus + 1u];
    }
    if (set.min_p > 0.0f) {
        // the least weight's bucket, and one on either side for the rounding of a logit's
        const float t = -__log2f(set.min_p > 1.0f ? 1.0f : set.min_p) * set.depths;
        const uint32_t bucket = t < float(kBuckets - 1u) ? uint32_t(t) : kBuckets - 1u;
        l.least_low = bucket ? bucket - 1u : 0u;
        l.least_high = min(bucket + 1u, kBuckets - 2u);
        low = lesser(low, greater(s.before[l.least_low], kWhole));
        high = lesser(high, greater(s.before[l.least_high + 1u], kWhole));
    }
    l.drawn_low = bucket_of(s, set.place(low));
    l.drawn_high = bucket_of(s, set.place(high));
    return l;
}

// A listed token at which sums reach a goal.
struct Listed {
    uint64_t key, before;  // before: the sum of weights (or the count) of the tokens before it
};

// Among those of the ``n`` keys of s.list that ``in`` takes, all in some range of them: where counts or weights, ``before`` of
// them before the first, reach ``goal``. Eleven bits of the keys a step, until 64 keys are left; each wave then compares those
// by itself.
template <class F> __device__ Listed reach_list(const Weights& w, Shared& s, uint32_t n, bool by_count, uint64_t before, uint64_t goal, F in) {
    uint64_t low = 0, high = ~0ull;
    const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u;
    const auto weight_of = [&](uint64_t key) { return by_count ? uint64_t(1) : w(value_of(uint32_t(key >> 32))); };
    for (int step = 0; step < 8; ++step) {
        uint64_t most = 0, least = 0;  // least: of the inverted keys
        uint32_t left = 0;
        if (threadIdx.x == 0u) {
            s.fews = 0u;
        }
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint64_t key = s.list[i];
            if (step ? key >= low && key <= high : in(key)) {
                most = greater(key, most);
                least = greater(~key, least);
                ++left;
            }
        }
        most = wave_max(most);
        least = wave_max(least);
        left = uint32_t(__builtin_amdgcn_readlane(wave_scan(left), 63));
        if (lane == 0u) {
            s.waves[wave] = Sums{most, left};
            s.ends[wave] = least;
        }
        __syncthreads();
        left = 0u;
#pragma unroll
        for (uint32_t v = 0; v < kThreads / 64u; ++v) {
            most = greater(most, s.waves[v].weight);
            least = greater(least, s.ends[v]);
            left += s.waves[v].count;
        }
        least = ~least;
        low = greater(low, least);
        high = lesser(high, most);
        if (left <= 64u) {
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
                const uint64_t key = s.list[i];
                if (key >= low && key <= high) {
                    s.few[atomicAdd(&s.fews, 1u)] = key;
                }
            }
            __syncthreads();
            const uint64_t key = lane < left ? s.few[lane] : 0u, mine = lane < left ? weight_of(key) : 0u;
            uint64_t above = before;
            for (uint32_t i = 0; i < left; ++i) {
                above += lane_u64(key, i) > key ? lane_u64(mine, i) : 0u;
            }
            const uint32_t at = __builtin_ctzll(__ballot(lane < left && above < goal && above + mine >= goal) | 1ull << 63);  // (one lane)
            __syncthreads();  // s.few and s.waves have been read
            return Listed{lane_u64(key, at), lane_u64(above, at)};
        }
        const int bits = 64 - __builtin_clzll(most ^ least), shift = bits > 11 ? bits - 11 : 0;
        for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
            s.weight[i] = 0u;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint64_t key = s.list[i];
            if (key >= low && key <= high) {
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.weight[(key >> shift) % kBuckets]), static_cast<unsigned long long>(weight_of(key)));
            }
        }
        __syncthreads();
        const uint32_t top = kBuckets - 1u - threadIdx.x * kPer;
        uint64_t own = 0;
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            own += s.weight[top - k];
        }
        uint64_t at = before + scan_all(s, Sums{own, 0u}).weight - own;
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            const uint64_t next = at + s.weight[top - k];
            if (at < goal && next >= goal) {  // one thread
                s.found.order = top - k;
                s.found.before.weight = at;
            }
            at = next;
        }
        __syncthreads();
        before = s.found.before.weight;
        const uint64_t above = most >> shift >> 11 << 11 | s.found.order;  // the keys' bits from ``shift`` on
        low = greater(low, above << shift);  // (other buckets' keys may lie in the step's range)
        high = lesser(high, above << shift | ((1ull << shift) - 1u));
        __syncthreads();
    }
    return Listed{low, before};
}

// The bin of a key whose bits from ``shift`` + 11 on are those of all others: bin 0 holds the largest ones.
__device__ __forceinline__ uint32_t bin_of(uint64_t key, uint32_t shift) { return kBuckets - 1u - uint32_t(key >> shift) % kBuckets; }

// The ``n`` > 1 listed keys in bins by their first eleven bits that differ: counts and weights before each bin in s.count and
// s.before (and of all in s.before[kBuckets]). Returns the bits' shift.
__device__ uint32_t ordered(const Weights& w, Shared& s, uint32_t n) {
    uint64_t most = 0, least = 0;  // least: of the inverted keys
    for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
        s.weight[i] = 0u;
        s.count[i] = 0u;
    }
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        most = greater(s.list[i], most);
        least = greater(~s.list[i], least);
    }
    most = max_all(s, most);
    least = ~max_all(s, least);
    const int bits = 64 - __builtin_clzll(most ^ least);
    const uint32_t shift = bits > 11 ? uint32_t(bits - 11) : 0u;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t key = s.list[i];
        const uint32_t bin = bin_of(key, shift);
        atomicAdd(&s.count[bin], 1u);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.weight[bin]), static_cast<unsigned long long>(w(value_of(uint32_t(key >> 32)))));
    }
    __syncthreads();
    const uint32_t first = threadIdx.x * kPer;
    Sums own{0u, 0u};
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) {
        own.weight += s.weight[first + k];
        own.count += s.count[first + k];
    }
    const Sums upto = scan_all(s, own);
    Sums at{upto.weight - own.weight, upto.count - own.count};
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) {
        const Sums here{s.weight[first + k], s.count[first + k]};
        s.before[first + k] = at.weight;
        s.count[first + k] = at.count;
        at.weight += here.weight;
        at.count += here.count;
    }
    if (threadIdx.x == kThreads - 1u) {
        s.before[kBuckets] = upto.weight;
    }
    __syncthreads();
    return shift;
}

// Lists the tokens of [begin, end): s.listed of them, the first kList to come in s.list.
template <class T, class S> __device__ void gather(const Settings& set, const Listing& l, const T* x, uint32_t begin, uint32_t end, S& s) {
    if (threadIdx.x == 0u) {
        s.listed = 0u;
    }
    __syncthreads();
    const float rate = set.rate();
    visit(x, begin, end, [&](float v, uint32_t i) {
        if (l.holds(set.bucket(v, rate))) {
            const uint32_t at = atomicAdd(&s.listed, 1u);
            if (at < kList) {
                s.list[at] = chroma::topk_key(v, i, true);
            }
        }
    });
    __syncthreads();
}

// The token of a row that a top-k cuts to what the first ``n`` <= 64 of ``keys`` hold, by each wave alone.
__device__ void choose_few(const Call& c, uint64_t r, const Settings& set, const Weights& w, const uint64_t* keys, uint32_t n) {
    const uint32_t lane = threadIdx.x % 64u;
    const uint64_t key = lane < n ? keys[lane] : 0u, all = lane < n ? w(value_of(uint32_t(key >> 32))) : 0u;
    uint32_t rank = 0;
    uint64_t above = 0;  // weights of larger keys
    for (uint32_t i = 0; i < n; ++i) {
        const bool larger = lane_u64(key, i) > key;
        above += larger ? lane_u64(all, i) : 0u;
        rank += larger ? 1u : 0u;
    }
    const uint64_t mine = rank < uint64_t(set.top_k) ? all : 0u;
    const auto at = [&](uint64_t goal) { return __builtin_ctzll(__ballot(above < goal && above + mine >= goal) | 1ull << 63); };
    uint64_t kept = wave_total(mine);
    if (set.top_p < 1.0f) {
        kept = lane_u64(above + mine, at(set.nucleus(kept)));
    }
    if (set.min_p > 0.0f) {
        kept = lesser(kept, greater(wave_total(mine >= set.least() ? mine : 0u), kWhole));
    }
    const uint64_t drawn = lane_u64(key, at(set.place(kept)));
    if (threadIdx.x == 0u) {
        c.ids[r] = int64_t(0xffffffffu - uint32_t(drawn));
        if (c.logprobs) {
            c.logprobs[r] = set.logprob(w, value_of(uint32_t(drawn >> 32)), kept);
        }
    }
}

// The token, from the ``n`` listed keys in s.list; ``below(b)``: the histogram's sums before bucket b.
template <class B> __device__ void choose(const Call& c, uint64_t r, const Settings& set, const Listing& l, uint32_t n, B below, Shared& s) {
    const Weights w = set.weights(s);
    const float rate = set.rate();
    const auto reach = [&](uint32_t b, uint64_t goal) {
        return reach_list(w, s, n, false, below(b), goal, [&](uint64_t key) { return set.bucket(value_of(uint32_t(key >> 32)), rate) == b; });
    };
    const auto weight_of = [&](uint64_t key) { return w(value_of(uint32_t(key >> 32))); };
    const auto at_least = [&](uint64_t least, uint32_t from, uint32_t to) {  // sum of the listed weights of these buckets
        Sums own{0u, 0u};
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const float v = value_of(uint32_t(s.list[i] >> 32));
            const uint32_t b = set.bucket(v, rate);
            const uint64_t mine = w(v);
            own.weight += mine >= least && b >= from && b <= to ? mine : 0u;
        }
        return sum_all(s, own).weight;
    };
    uint64_t kept;
    Listed drawn;
    if (l.by_count) {
        if (n <= 64u) {
            choose_few(c, r, set, w, s.list, n);
            return;
        }
        // One histogram over the keys' first bits that differ answers every cut but for the keys of a bin (fewer than top_k are
        // listed where the top-k takes tokens that weigh nothing).
        const uint32_t shift = ordered(w, s, n);
        const auto within = [&](uint32_t bin, bool by_count, uint64_t goal) {
            return reach_list(w, s, n, by_count, by_count ? uint64_t(s.count[bin]) : s.before[bin], goal, [&](uint64_t key) { return bin_of(key, shift) == bin; });
        };
        kept = s.before[kBuckets];
        if (n > uint64_t(set.top_k)) {
            for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
                if (s.count[i] < set.top_k && (i + 1u < kBuckets ? s.count[i + 1u] : n) >= set.top_k) {
                    s.last = i;
                }
            }
            __syncthreads();
            const uint32_t bin = s.last;
            const uint64_t last = within(bin, true, uint64_t(set.top_k)).key;
            Sums own{0u, 0u};
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
                own.weight += s.list[i] >= last && bin_of(s.list[i], shift) == bin ? weight_of(s.list[i]) : 0u;
            }
            kept = s.before[bin] + sum_all(s, own).weight;
        }
        if (set.top_p < 1.0f) {
            const uint64_t goal = set.nucleus(kept);
            const Listed cut = within(bucket_of(s, goal), false, goal);
            kept = cut.before + weight_of(cut.key);
        }
        if (set.min_p > 0.0f) {
            kept = lesser(kept, greater(at_least(set.least(), 0u, kBuckets), kWhole));
        }
        const uint64_t goal = set.place(kept);
        drawn = within(bucket_of(s, goal), false, goal);
    } else {
        kept = below(kBuckets);
        if (set.top_p < 1.0f) {
            const Listed cut = reach(l.nucleus, set.nucleus(kept));
            kept = cut.before + weight_of(cut.key);
        }
        if (set.min_p > 0.0f) {
            const uint64_t high = below(l.least_low) + at_least(set.least(), l.least_low, l.least_high);
            kept = lesser(kept, greater(high, kWhole));
        }
        const uint64_t goal = set.place(kept);
        uint32_t b = l.drawn_low;
        while (b < l.drawn_high && below(b + 1u) < goal) {
            ++b;
        }
        drawn = reach(b, goal);
    }
    if (threadIdx.x == 0u) {
        c.ids[r] = int64_t(0xffffffffu - uint32_t(drawn.key));
        if (c.logprobs) {
            c.logprobs[r] = set.logprob(w, value_of(uint32_t(drawn.key >> 32)), kept);
        }
    }
}

// One workgroup a row. grid: rows
template <class T> __global__ void __launch_bounds__(kThreads) sample_rows(Call c) {
    __shared__ Shared s;
    s.powers.fill();
    const uint64_t r = blockIdx.x;
    const T* x = static_cast<const T*>(c.x) + r * uint64_t(c.x_stride);
    const uint32_t width = uint32_t(c.width);
    const Settings set(c, r, ends_of(s, x, 0u, width));
    if (set.greedy()) {
        if (threadIdx.x == 0u) {
            set.finish(c, r);
        }
        return;
    }
    depths(set, x, 0u, width, s);
    const Listing l = list_of(set, s);
    if (l.whole) {
        descend_row(c, r, set, x, s);
        return;
    }
    gather(set, l, x, 0u, width, s);
    const uint32_t n = s.listed;
    if (n > kList) {
        descend_row(c, r, set, x, s);
        return;
    }
    choose(c, r, set, l, n, [&](uint32_t b) { return s.before[b]; }, s);
}

// Scratch of a row that is cut into spans.
struct Scratch {
    uint64_t* best;       // [spans], largest key and least order
    uint64_t* histogram;  // [spans, kBuckets]
    uint64_t* before;     // [kBuckets + 1]
    uint64_t* list;       // [kList]
    Listing* listing;
    uint32_t* tickets;  // workgroups that are done with the histogram; listed tokens
    static __host__ __device__ uint64_t words(uint64_t spans) { return spans * (2u + kBuckets) + kBuckets + 1u + kList + 8u; }
    __device__ Scratch(uint64_t* base, uint64_t r, uint32_t spans) {
        best = base + r * words(spans);
        histogram = best + 2u * spans;
        before = histogram + uint64_t(spans) * kBuckets;
        list = before + kBuckets + 1u;
        listing = reinterpret_cast<Listing*>(list + kList);
        tickets = reinterpret_cast<uint32_t*>(list + kList + 4u);
    }
};
static_assert(sizeof(Listing) <= 32, "scratch");

struct Span {
    uint32_t begin, end;
    __device__ Span(const Call& c, uint32_t spans, uint32_t i) {
        const uint32_t width = uint32_t(c.width), each = ((width + spans - 1u) / spans + 7u) / 8u * 8u;
        begin = min(i * each, width);
        end = min(begin + each, width);
    }
};

// The first reading: each span's largest logit. grid: (spans, rows)
template <class T> __global__ void __launch_bounds__(kThreads, 8) sample_best(Call c, uint64_t* scratch) {
    __shared__ Waves s;
    const uint64_t r = blockIdx.y;
    const Scratch mine(scratch, r, gridDim.x);
    const Span span(c, gridDim.x, blockIdx.x);
    const Ends ends = ends_of(s, static_cast<const T*>(c.x) + r * uint64_t(c.x_stride), span.begin, span.end);
    if (threadIdx.x == 0u) {
        mine.best[2u * blockIdx.x] = ends.best;
        mine.best[2u * blockIdx.x + 1u] = ends.least;
        if (blockIdx.x == 0u) {
            mine.tickets[0] = 0u;
            mine.tickets[1] = 0u;
        }
    }
}

__device__ Ends ends_of(const Scratch& mine, uint32_t spans) {
    Ends ends{0u, 0u};
    for (uint32_t i = threadIdx.x % 64u; i < spans; i += 64u) {
        ends.best = greater(ends.best, mine.best[2u * i]);
        ends.least = max(ends.least, uint32_t(mine.best[2u * i + 1u]));
    }
    return Ends{wave_max(ends.best), wave_max(ends.least)};
}

// Whether this workgroup is the last of the row's to come here, after its device-scope stores.
__device__ bool comes_last(uint32_t* ticket, Waves& s) {
    chroma::device_stores_complete();
    __syncthreads();
    if (threadIdx.x == 0u) {
        s.last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    const bool last = s.last == gridDim.x - 1u;
    __syncthreads();
    return last;
}

// The second reading: the histogram, and what is listed. grid: (spans, rows)
template <class T> __global__ void __launch_bounds__(kThreads, 8) sample_depths(Call c, uint64_t* scratch) {
    __shared__ Depths s;
    s.powers.fill();
    const uint64_t r = blockIdx.y;
    const uint32_t spans = gridDim.x;
    const Scratch mine(scratch, r, spans);
    const Settings set(c, r, ends_of(mine, spans));
    if (set.greedy()) {
        if (blockIdx.x == 0u && threadIdx.x == 0u) {
            set.finish(c, r);
        }
        return;
    }
    const Span span(c, spans, blockIdx.x);
    depths(set, static_cast<const T*>(c.x) + r * uint64_t(c.x_stride), span.begin, span.end, s);
    uint64_t* to = mine.histogram + uint64_t(blockIdx.x) * kBuckets;
    for (uint32_t i = threadIdx.x; i < kBuckets; i += kThreads) {
        chroma::store_device(to + i, s.weight[i]);
    }
    if (!comes_last(mine.tickets, s)) {
        return;
    }
    uint64_t sums[kPer] = {};
    for (uint32_t k0 = 0; k0 < spans; k0 += 4u) {  // (16 loads under way)
        uint64_t some[4][kPer];
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) {
                some[k][e] = chroma::load_device(mine.histogram + uint64_t(min(k0 + k, spans - 1u)) * kBuckets + threadIdx.x + e * kThreads);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) {
                sums[e] += k0 + k < spans ? some[k][e] : 0u;
            }
        }
    }
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) {
        s.weight[threadIdx.x + e * kThreads] = sums[e];
    }
    __syncthreads();
    const Listing l = list_of(set, s);
    for (uint32_t i = threadIdx.x; i <= kBuckets; i += kThreads) {
        mine.before[i] = s.before[i];
    }
    if (threadIdx.x == 0u) {
        *mine.listing = l;
    }
}

// The third reading: the list. grid: (spans, rows)
template <class T> __global__ void __launch_bounds__(kThreads, 8) sample_listed(Call c, uint64_t* scratch) {
    __shared__ Gathered s;
    const uint64_t r = blockIdx.y;
    const Scratch mine(scratch, r, gridDim.x);
    const Settings set(c, r, ends_of(mine, gridDim.x));
    const Listing l = *mine.listing;
    if (set.greedy() || l.whole) {
        return;
    }
    const Span span(c, gridDim.x, blockIdx.x);
    gather(set, l, static_cast<const T*>(c.x) + r * uint64_t(c.x_stride), span.begin, span.end, s);
    if (threadIdx.x == 0u) {
        s.begin = atomicAdd(mine.tickets + 1, s.listed);
    }
    __syncthreads();
    const uint32_t begin = s.begin, own = min(s.listed, kList);
    for (uint32_t i = threadIdx.x; i < own && begin + i < kList; i += kThreads) {
        mine.list[begin + i] = s.list[i];
    }
}

// The token. grid: rows
template <class T> __global__ void __launch_bounds__(kThreads) sample_token(Call c, uint64_t* scratch, uint32_t spans) {
    __shared__ Shared s;
    const uint64_t r = blockIdx.x;
    const Scratch mine(scratch, r, spans);
    const Settings set(c, r, ends_of(mine, spans));
    if (set.greedy()) {
        return;
    }
    s.powers.fill();
    const Listing l = *mine.listing;
    const uint32_t n = mine.tickets[1];
    if (l.whole || n > kList) {
        descend_row(c, r, set, static_cast<const T*>(c.x) + r * uint64_t(c.x_stride), s);
        return;
    }
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        s.list[i] = mine.list[i];
    }
    __syncthreads();
    choose(c, r, set, l, n, [&](uint32_t b) { return mine.before[b]; }, s);
}

// Spans of a row, of 8192 tokens at least: two workgroups for each compute unit and four for a row; 1: one launch of a
// workgroup a row. 64 rows of 201088 bfloat16 logits cut to 50 tokens: 8 spans 39 us, 16 48, 32 (of 4096) 80; 256 rows with
// settings of their own: 2 spans 152 us, 4 123, 8 131. Thousands of rows fill the chip by themselves.
uint32_t spans_of(const Call& c) {
    const int64_t wanted = c.rows > 2048 ? 1 : c.rows >= 128 ? 4 : 512 / c.rows, most = c.width / 8192;
    return uint32_t(wanted < 2 || most < 2 ? 1 : wanted < most ? wanted : most);
}

template <class T> void launch(const Call& c, uint64_t* scratch, hipStream_t stream) {
    const uint32_t spans = spans_of(c);
    if (spans == 1u) {
        sample_rows<T><<<unsigned(c.rows), kThreads, 0, stream>>>(c);
        return;
    }
    const dim3 grid(spans, unsigned(c.rows));
    sample_best<T><<<grid, kThreads, 0, stream>>>(c, scratch);
    sample_depths<T><<<grid, kThreads, 0, stream>>>(c, scratch);
    sample_listed<T><<<grid, kThreads, 0, stream>>>(c, scratch);
    sample_token<T><<<unsigned(c.rows), kThreads, 0, stream>>>(c, scratch, spans);
}

int refuse(const char* message, char* error, size_t size) {
    if (error && size) {
        std::snprintf(error, size, "rows_sample: %s", message);
    }
    return CHROMA_HIP_RUNTIME_ERROR;
}

}  // namespace

namespace chroma_sample {

size_t workspace_bytes(const Call& c) {
    const uint32_t spans = mistake(c) ? 1u : spans_of(c);
    return spans > 1u ? size_t(c.rows) * Scratch::words(spans) * sizeof(uint64_t) : 0;
}

int launch_rows_sample(const Call& c, void* workspace, size_t workspace_size, hipStream_t stream, char* error, size_t error_size) {
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
    const size_t need = workspace_bytes(c);
    if (need && (!workspace || workspace_size < need)) {
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
        launch<float>(c, static_cast<uint64_t*>(workspace), stream);
    } else {
        launch<uint16_t>(c, static_cast<uint64_t*>(workspace), stream);
    }
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? CHROMA_HIP_OK : refuse(hipGetErrorString(status), error, error_size);
}

}  // namespace chroma_sample

extern "C" {

__attribute__((visibility("default"))) size_t chroma_hip_rows_sample_workspace(const Call* call) { return call ? chroma_sample::workspace_bytes(*call) : 0; }

__attribute__((visibility("default"))) int chroma_hip_rows_sample(const Call* call, void* workspace, size_t workspace_bytes, void* stream,
                                                                  char* error, size_t error_size) {
    if (!call) {
        return refuse("null call", error, error_size);
    }
    return chroma_sample::launch_rows_sample(*call, workspace, workspace_bytes, static_cast<hipStream_t>(stream), error, error_size);
}

}  // extern "C"
