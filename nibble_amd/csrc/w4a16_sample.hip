// Sampling a token from each row of logits (include/w4a16_sample.h).
//
// Mathematics. With m the row's largest logit and T the temperature, token i has
// the weight w_i = 2^((x_i - m) log2(e) / T), held as the whole number
// W_i = round(2^44 w_i). In 64 bits the sums of such numbers are exact in any
// order, so neither the split over lanes nor the order of atomics changes a
// result, and a threshold found in one pass means the same in the next. A weight
// is off by 2^-45 of the largest one and by about 2^-46 of itself.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "w4a16_hip.h"
#include "w4a16_kv.h"
#include "w4a16_kv_device.h"
#include "w4a16_kv_host.h"
#include "w4a16_sample.h"

namespace w4a16 {

struct SampleArgs {
    const uint8_t* logits;
    int64_t row_bytes;   // from one row to the next
    const float* random;
    int64_t* tokens;
    w4a16_sample_settings settings;
    int n;
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr double kOne = 0x1p44;   // the weight of the largest logit
constexpr int kLowestPower = -46; // weights below 2^-46 are 0

// ---------------------------------------------------------------------------
// Scans over the workgroup. Every thread takes part.
// ---------------------------------------------------------------------------
struct Scratch {
    uint64_t sums[kWaves];
    uint64_t found[3];
    float tops[kWaves];
    int firsts[kWaves];
};

__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {   // sums of the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t other = __shfl_up((unsigned long long)v, d);
        if ((int)(threadIdx.x & 63) >= d) v += other;
    }
    return v;
}

// The entry at which the running sum reaches a target, the sum before it, and
// the sum of all entries. `target_of(total)` gives the target, at least 1;
// index -1 where the total stays below it. Two entries a thread, in order.
struct Found {
    int index;
    uint64_t before, total;
};
template <typename Entry, typename Target>
__device__ __forceinline__ Found find(Scratch& s, int entries, Entry entry, Target target_of) {
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t a = 2 * tid < entries ? entry(2 * tid) : 0, b = 2 * tid + 1 < entries ? entry(2 * tid + 1) : 0;
    const uint64_t upto = wave_scan(a + b);
    if ((tid & 63) == 63) s.sums[wave] = upto;
    if (tid == 0) s.found[0] = ~0ull;
    __syncthreads();
    uint64_t before = upto - (a + b), total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += s.sums[w];
        total += s.sums[w];
    }
    const uint64_t target = target_of(total);
    if (before < target && before + a + b >= target) {
        const bool first = before + a >= target;
        s.found[0] = 2 * tid + (first ? 0 : 1);
        s.found[1] = before + (first ? 0 : a);
    }
    __syncthreads();
    const Found f = {(int)s.found[0], s.found[1], total};
    __syncthreads();   // the scratch may be written again
    return f;
}

// ---------------------------------------------------------------------------
// A row of logits: vector j of a thread holds the elements (1024 j + thread) VE
// .. + VE - 1; those behind the row read as -inf. Every pass reads them again.
// ---------------------------------------------------------------------------
template <int TYPE>
struct Row {
    static constexpr int VE = TYPE == W4A16_FP32 ? 4 : 8, SIZE = 16 / VE;
    const uint8_t* p;
    int n, vectors;

    // unaligned: a row may start at any element
    struct __attribute__((packed, aligned(2))) Loose {
        uint32_t w[4];
    };
    __device__ __forceinline__ u32x4 read(int j) const {
        const int v = j * kThreads + (int)threadIdx.x;
        constexpr uint32_t lowest = TYPE == W4A16_FP32 ? 0xFF800000u : TYPE == W4A16_FP16 ? 0xFC00FC00u : 0xFF80FF80u;
        u32x4 x = {lowest, lowest, lowest, lowest};
        if ((v + 1) * VE <= n) {
            const Loose w = *reinterpret_cast<const Loose*>(p + (int64_t)v * 16);
            x = (u32x4){w.w[0], w.w[1], w.w[2], w.w[3]};
        } else if (v * VE < n) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                if (v * VE + e >= n) continue;
                if constexpr (TYPE == W4A16_FP32) {
                    x[e] = *reinterpret_cast<const uint32_t*>(p + (int64_t)v * 16 + 4 * e);
                } else {
                    const uint32_t bits = *reinterpret_cast<const uint16_t*>(p + (int64_t)v * 16 + 2 * e);
                    x[e >> 1] = e & 1 ? (x[e >> 1] & 0xFFFFu) | bits << 16 : (x[e >> 1] & 0xFFFF0000u) | bits;
                }
            }
        }
        return x;
    }
    // f(j, vector) for the thread's vectors, every lane taking part
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
        for (int j = 0; j * kThreads < vectors; ++j) f(j, read(j));
    }
    __device__ __forceinline__ static float value(const u32x4& v, int e) {
        const uint32_t word = v[TYPE == W4A16_FP32 ? e : e >> 1];
        if constexpr (TYPE == W4A16_FP32)
            return __builtin_bit_cast(float, word);   // of the copy: of v[e] it is that of v[0]
        else
            return widen16<TYPE>(e & 1 ? word >> 16 : word & 0xFFFFu);
    }
    __device__ __forceinline__ static int index(int j, int e) { return (j * kThreads + (int)threadIdx.x) * VE + e; }
    // Values in their order as whole numbers (of the type's bits): equal ones
    // equal, -0 as 0.
    __device__ __forceinline__ static uint32_t key(float x) {
        x += 0.0f;
        const uint32_t b = __builtin_bit_cast(uint32_t, x);
        const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
        if constexpr (TYPE == W4A16_FP32) return k;
        if constexpr (TYPE == W4A16_BF16) return k >> 16;
        const uint32_t h = __builtin_bit_cast(uint16_t, (f16)x);
        return (h ^ (h >> 15 ? 0xFFFFu : 0x8000u)) & 0xFFFFu;
    }
};

// 2^y of y <= 0 as a double, by its power series: 2^f, |f| <= 1/2, off by
// (ln 2 / 2)^12 / 12! = 2^-47.
__device__ __forceinline__ double exp2_series(double y) {
    const double whole = __builtin_rint(y);
    const double f = y - whole;
    double s = 4.44553827187081e-10;   // ln(2)^k / k!, k = 11 .. 0
    s = __builtin_fma(s, f, 7.054911620801121e-09);
    s = __builtin_fma(s, f, 1.0178086009239696e-07);
    s = __builtin_fma(s, f, 1.3215486790144305e-06);
    s = __builtin_fma(s, f, 1.5252733804059838e-05);
    s = __builtin_fma(s, f, 0.00015403530393381606);
    s = __builtin_fma(s, f, 0.0013333558146428441);
    s = __builtin_fma(s, f, 0.009618129107628477);
    s = __builtin_fma(s, f, 0.055504108664821576);
    s = __builtin_fma(s, f, 0.2402265069591007);
    s = __builtin_fma(s, f, 0.6931471805599453);
    s = __builtin_fma(s, f, 1.0);
    return __builtin_ldexp(s, (int)whole);
}

// The weights of a row's logits.
struct Weights {
    double top, factor, least;   // least: of the smallest weight that min_p keeps (0: all)
    float top_f;
    __device__ __forceinline__ double power(float x) const { return ((double)x - top) * factor; }
    // the largest logit, also an infinite one, weighs 1
    __device__ __forceinline__ double weight(float x) const {
        const double y = power(x);
        const double w = y > (double)kLowestPower ? exp2_series(y) : 0.0;
        return x == top_f ? 1.0 : w;
    }
    static __device__ __forceinline__ double whole(double w) { return __builtin_rint(w * kOne); }
    __device__ __forceinline__ double kept(float x) const {   // with min_p
        const double w = weight(x);
        return w >= least ? whole(w) : 0.0;
    }
};

__device__ __forceinline__ float block_max(Scratch& s, float v) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) s.tops[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v = fmaxf(v, s.tops[w]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ int block_min(Scratch& s, int v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = min(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) s.firsts[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v = min(v, s.firsts[w]);
    return v;
}

// What of a row is kept: values above `value`, and the first `ties` that equal it.
struct Limit {
    float value;
    int64_t ties;
};

template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    using R = Row<TYPE>;
    __shared__ Scratch scratch;
    __shared__ uint64_t bins[kBins];
    __shared__ uint32_t counts[kBins];

    const int row = blockIdx.x, tid = threadIdx.x;
    R r;
    r.p = a.logits + row * a.row_bytes;
    r.n = a.n;
    r.vectors = (a.n + R::VE - 1) / R::VE;
    const float u = a.random[row];
    const double temperature = a.settings.temperatures ? (double)a.settings.temperatures[row] : a.settings.temperature;
    const int64_t top_k = a.settings.top_ks ? a.settings.top_ks[row] : a.settings.top_k;
    const double top_p = a.settings.top_ps ? (double)a.settings.top_ps[row] : a.settings.top_p;
    const double min_p = a.settings.min_ps ? (double)a.settings.min_ps[row] : a.settings.min_p;

    float top = -__builtin_inff();
    bool strange = false;
    r.each([&](int, const u32x4& v) {
#pragma unroll
        for (int e = 0; e < R::VE; ++e) {
            const float x = R::value(v, e);
            top = fmaxf(top, x);
            strange |= x != x;
        }
    });
    top = block_max(scratch, top);
    strange = __syncthreads_or(strange);
    // the first of the largest; a NaN counts as the largest, as in argmax
    if (strange || !(temperature > 0.0) || top == -__builtin_inff() || top_k == 1) {
        int first = a.n;
        r.each([&](int j, const u32x4& v) {
#pragma unroll
            for (int e = 0; e < R::VE; ++e) {
                const float x = R::value(v, e);
                if (strange ? x != x : x == top) first = min(first, R::index(j, e));
            }
        });
        first = block_min(scratch, first);
        if (tid == 0) a.tokens[row] = first;
        return;
    }
    const Weights weights = {(double)top, 1.4426950408889634 / temperature, min_p > 0.0 ? fmin(min_p, 1.0) : 0.0, top};

    // The value at which the running sum of `amount` over the values in falling
    // order reaches `target_of(total)`, level by level of 2048 ranges of whole
    // numbers, the first from the largest value down to the lowest that has a
    // weight. `only(x)`: the values taken into account; `beside`: amount of ties
    // of a value `tied` that stand for themselves.
    const uint32_t top_key = R::key(top);
    auto select = [&](auto only, auto amount, float tied, uint64_t beside, auto target_of, uint64_t& rest) {
        const double reach = (double)kLowestPower / weights.factor;
        const float lowest = (float)fmax((double)top + reach - 1e-6 * fabs(reach), -3.4028234663852886e38);
        uint32_t from = 0, range = top_key - R::key(lowest);
        int shift = max(0, 21 - __builtin_clz(range | 1));
        uint64_t target = 0;
        bool first = true;
        while (true) {
            for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
            __syncthreads();
            auto add = [&](float x, uint64_t v) {
                const uint32_t d = top_key - R::key(x) - from;
                if (d <= range && v != 0) atomicAdd((unsigned long long*)&bins[d >> shift], (unsigned long long)v);
            };
            r.each([&](int, const u32x4& v) {
#pragma unroll
                for (int e = 0; e < R::VE; ++e) {
                    const float x = R::value(v, e);
                    if (x >= lowest && only(x)) {
                        const uint32_t d = top_key - R::key(x) - from;
                        if (d <= range) {
                            const uint64_t w = amount(x);
                            if (w != 0) atomicAdd((unsigned long long*)&bins[d >> shift], (unsigned long long)w);
                        }
                    }
                }
            });
            if (tid == 0 && beside != 0) add(tied, beside);
            __syncthreads();
            const Found f = find(scratch, kBins, [&](int i) { return bins[i]; },
                                 [&](uint64_t total) { return first ? target_of(total) : target; });
            if (first) target = target_of(f.total);
            first = false;
            if (f.index < 0) return false;
            target -= f.before;
            from += (uint32_t)f.index << shift;
            range = (1u << shift) - 1;
            if (shift == 0) break;
            shift = max(0, shift - 11);
        }
        rest = target;
        // the value whose key it is
        const uint32_t k = top_key - from;
        if constexpr (TYPE == W4A16_FP32)
            tied = __builtin_bit_cast(float, k >> 31 ? k ^ 0x80000000u : ~k);
        else
            tied = widen16<TYPE>((k >> 15 ? k ^ 0x8000u : ~k) & 0xFFFFu);
        scratch.tops[0] = tied;   // the same from every thread
        return true;
    };

    Limit limit = {-__builtin_inff(), a.n};
    if (top_k > 0 && top_k < a.n) {
        uint64_t rest;
        if (select([](float) { return true; }, [](float) { return (uint64_t)1; }, 0.0f, 0,
                   [&](uint64_t) { return (uint64_t)top_k; }, rest)) {
            __syncthreads();
            limit = {scratch.tops[0], (int64_t)rest};
            __syncthreads();
        }
    }
    if (top_p < 1.0) {
        const uint64_t tie = (uint64_t)Weights::whole(weights.weight(limit.value));
        const uint64_t beside = limit.value == -__builtin_inff() ? 0 : tie * (uint64_t)limit.ties;
        uint64_t rest;
        const float before = limit.value;
        if (select([&](float x) { return x > before; }, [&](float x) { return (uint64_t)Weights::whole(weights.weight(x)); },
                   before, beside,
                   [&](uint64_t total) {
                       const double t = __builtin_ceil(top_p * (double)total);
                       return t >= 1.0 ? min((uint64_t)t, total) : (uint64_t)1;
                   }, rest)) {
            __syncthreads();
            const float value = scratch.tops[0];
            __syncthreads();
            const uint64_t w = (uint64_t)Weights::whole(weights.weight(value));
            limit = {value, (int64_t)((rest + w - 1) / w)};
        }
    }

    // Sums of what is kept, for each vector of a wavefront (512 or 256
    // neighbours), ties apart as their places are not known yet.
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int entries = (r.vectors + kThreads - 1) / kThreads * kWaves;
    const uint64_t tie = (uint64_t)weights.kept(limit.value);
    r.each([&](int j, const u32x4& v) {
        double sum = 0.0;
        int ties = 0;
#pragma unroll
        for (int e = 0; e < R::VE; ++e) {
            const float x = R::value(v, e);
            if (x > limit.value) sum += weights.kept(x);
            ties += x == limit.value ? 1 : 0;
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            sum += __shfl_xor(sum, d);
            ties += __shfl_xor(ties, d);
        }
        if (lane == 0) {
            bins[j * kWaves + wave] = (uint64_t)sum;
            counts[j * kWaves + wave] = (uint32_t)ties;
        }
    });
    __syncthreads();
    // ties before each entry
    {
        const uint32_t c0 = 2 * tid < entries ? counts[2 * tid] : 0, c1 = 2 * tid + 1 < entries ? counts[2 * tid + 1] : 0;
        const uint64_t upto = wave_scan((uint64_t)c0 + c1);
        if (lane == 63) scratch.sums[wave] = upto;
        __syncthreads();
        uint64_t before = upto - c0 - c1;
        for (int w = 0; w < wave; ++w) before += scratch.sums[w];
        auto put = [&](int i, uint32_t c, uint64_t at) {
            const int64_t free = max((int64_t)0, limit.ties - (int64_t)at);
            bins[i] += tie * (uint64_t)min(free, (int64_t)c);
            counts[i] = (uint32_t)at;
        };
        if (2 * tid < entries) put(2 * tid, c0, before);
        if (2 * tid + 1 < entries) put(2 * tid + 1, c1, before + c0);
        __syncthreads();
    }
    uint64_t target = 0;
    const Found f = find(scratch, entries, [&](int i) { return bins[i]; }, [&](uint64_t total) {
        const double at = (u > 0.0f ? (double)u : 0.0) * (double)total;   // NaN as 0
        target = at < (double)total ? min((uint64_t)at, total - 1) + 1 : total;
        return target;
    });
    if (f.index % kWaves != wave) return;
    // the wavefront that holds it
    target -= f.before;
    const int j = f.index / kWaves;
    const u32x4 v = r.read(j);
    uint64_t own[R::VE], sum = 0;
    int ties = 0;
#pragma unroll
    for (int e = 0; e < R::VE; ++e) ties += R::value(v, e) == limit.value ? 1 : 0;
    int64_t at = (int64_t)counts[f.index] + (int64_t)wave_scan((uint64_t)ties) - ties;
#pragma unroll
    for (int e = 0; e < R::VE; ++e) {
        const float x = R::value(v, e);
        own[e] = 0;
        if (x > limit.value) own[e] = (uint64_t)weights.kept(x);
        if (x == limit.value) own[e] = at++ < limit.ties ? tie : 0;
        sum += own[e];
    }
    uint64_t before = wave_scan(sum) - sum;
    if (before < target && before + sum >= target) {
        int e = 0;
#pragma unroll
        for (int i = 0; i < R::VE; ++i) {
            before += own[i];
            if (before < target) e = i + 1;
        }
        a.tokens[row] = R::index(j, e);
    }
}

}  // namespace w4a16

namespace {

using namespace w4a16;
using w4a16_internal::kv_fail;

constexpr int64_t kMostLogits = 1 << 19;   // sums of 2^44 each stay below 2^63

}  // namespace

extern "C" {

int w4a16_sample(const void* logits, int64_t rows, int64_t n, int64_t row_stride, int type, const float* random,
                 const w4a16_sample_settings* settings, int64_t* tokens, void* stream) {
    if (type != W4A16_FP16 && type != W4A16_BF16 && type != W4A16_FP32)
        return kv_fail(W4A16_ERR_CONFIG, "logits must be fp16, bf16 or fp32");
    if (settings == nullptr) return kv_fail(W4A16_ERR_NULL, "settings must be non-NULL");
    const w4a16_sample_settings& s = *settings;
    if (s.temperatures == nullptr && !(s.temperature >= 0.0))
        return kv_fail(W4A16_ERR_CONFIG, "temperature must not be negative");
    if (s.top_ks == nullptr && s.top_k < 0) return kv_fail(W4A16_ERR_CONFIG, "top_k must not be negative");
    if (s.top_ps == nullptr && !(s.top_p >= 0.0 && s.top_p <= 1.0))
        return kv_fail(W4A16_ERR_CONFIG, "top_p must be between 0 and 1");
    if (s.min_ps == nullptr && !(s.min_p >= 0.0 && s.min_p <= 1.0))
        return kv_fail(W4A16_ERR_CONFIG, "min_p must be between 0 and 1");
    if (rows < 0 || n < 1) return kv_fail(W4A16_ERR_SHAPE, "a row must have at least one logit");
    if (n > kMostLogits) return kv_fail(W4A16_ERR_TOO_LARGE, "a row may have at most 524288 logits");
    if (!w4a16_internal::launch_fits(rows, kThreads)) return kv_fail(W4A16_ERR_TOO_LARGE, "too many rows for one launch");
    if (rows == 0) return W4A16_OK;
    if (logits == nullptr || random == nullptr || tokens == nullptr)
        return kv_fail(W4A16_ERR_NULL, "logits, random and tokens must be non-NULL");
    const int size = type == W4A16_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, "logits must be aligned to their size");
    SampleArgs a{};
    a.logits = static_cast<const uint8_t*>(logits);
    a.row_bytes = row_stride * size;
    a.random = random;
    a.tokens = tokens;
    a.settings = s;
    a.n = (int)n;
    const dim3 grid((unsigned)rows), threads(kThreads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (type == W4A16_FP16)
        hipLaunchKernelGGL((sample_kernel<W4A16_FP16>), grid, threads, 0, st, a);
    else if (type == W4A16_BF16)
        hipLaunchKernelGGL((sample_kernel<W4A16_BF16>), grid, threads, 0, st, a);
    else
        hipLaunchKernelGGL((sample_kernel<W4A16_FP32>), grid, threads, 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return kv_fail(W4A16_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(e));
    return W4A16_OK;
}

}  // extern "C"
