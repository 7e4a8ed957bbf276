// Sampling a token from each row of logits (include/w4a16_sample.h).
//
// Mathematics. With m the row's largest logit and T the temperature, token i has
// the weight w_i = 2^((x_i - m) log2(e) / T), held as the whole number
// W_i = round(2^44 w_i). In 64 bits the sums of such numbers are exact in any
// order, so neither the split over lanes nor the order of atomics changes a
// result, and a threshold found in one pass means the same in the next. A weight
// is off by 2^-45 of the largest one and by 2^-38 of itself.
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
constexpr int kMostEntries = 512;    // sums of places: 2^19 fp32 logits
constexpr int kList = 256;           // candidates that are compared with each other
constexpr int kMostNear = 4096;      // logits near a limit that are listed, with places that stay empty
constexpr int kStaged = 4;           // vectors of a thread that stay in LDS: a group, 64 KB
constexpr int kTiny = 64;            // bf16 logits between 0 and 2^-20 that are listed
constexpr int kValues = 7168;        // bf16 values that a row's weights may take
constexpr uint64_t kOne = 1ull << 44;   // the weight of the largest logit
constexpr float kOctaves = 48.0f;    // below the largest weight that the bins of falling weight reach
constexpr float kBinsPerOctave = kBins / kOctaves;

struct Candidate {
    float x;
    int index;
    uint64_t weight;
};

// What a workgroup keeps in LDS beside the row.
struct Shared {
    union {
        struct {
            uint64_t bins[kBins];
            uint32_t counts[kBins + 32];   // the last ones of logits without a weight, spread over the banks
            int near[kMostNear];
        };
        struct {
            uint64_t value_weights[kValues + 32];   // of bf16 values in falling order, then of those without a weight
            uint32_t value_counts[kValues + 32];
        };
        struct {
            uint64_t bins_too[kBins];
            uint32_t counts_too[kBins + 32];
            Candidate list[kList];
            uint64_t before[kList];   // weight of the better candidates, or of the earlier ones
            int rank[kList];
        };
    };
    uint64_t kept[kMostEntries];   // sums of the kept weights of a wavefront's logits of a group
    uint32_t ties[kMostEntries];   // and how many of them equal the limit
    uint64_t sums[2 * kWaves];
    uint64_t found[2];
    float tops[kWaves];
    int firsts[kWaves];
    int listed, tinies;
    int tiny[kTiny];
};

// ---------------------------------------------------------------------------
// Scans over a wavefront and over the workgroup. Every thread takes part.
// ---------------------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t plus_dpp(uint64_t v) {   // lanes without a source add 0
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + ((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ uint64_t row_scan(uint64_t v) {   // sums of the lanes up to this one, of each 16
    v = plus_dpp<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
    v = plus_dpp<0x112, 0xF>(v);
    v = plus_dpp<0x114, 0xF>(v);
    return plus_dpp<0x118, 0xF>(v);
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {   // of all lanes
    v = row_scan(v);
    v = plus_dpp<0x142, 0xA>(v);   // row_bcast 15: lane 15 to the next row, 47 to the last
    v = plus_dpp<0x143, 0xC>(v);   // row_bcast 31: lane 31 to the upper half
    return v;
}

// The entry at which the running sum reaches a target, the sum before it, and
// the sum of all entries. `target_of(total)` gives the target, at least 1;
// index -1 where the total stays below it. PER entries a thread, in order.
struct Found {
    int index;
    uint64_t before, total;
};
template <int PER = 2, typename Value, typename Target>
__device__ __forceinline__ Found find(Shared& s, int n, Value value, Target target_of) {
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint64_t own[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        own[i] = PER * tid + i < n ? value(PER * tid + i) : 0;
        sum += own[i];
    }
    const uint64_t upto = wave_scan(sum);
    if ((tid & 63) == 63) s.sums[wave] = upto;
    if (tid == 0) s.found[0] = ~0ull;
    __syncthreads();
    const uint64_t waves = row_scan(s.sums[tid & 15]);
    uint64_t before = upto - sum + (wave > 0 ? lane_of(waves, wave - 1) : 0);
    const uint64_t total = lane_of(waves, 15);
    const uint64_t target = target_of(total);
    if (before < target && before + sum >= target) {
        int at = 0;
        uint64_t below = before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            before += own[i];
            if (before < target) {
                at = i + 1;
                below = before;
            }
        }
        s.found[0] = PER * tid + at;
        s.found[1] = below;
    }
    __syncthreads();
    const Found f = {(int)s.found[0], s.found[1], total};
    __syncthreads();   // the memory may be written again
    return f;
}

// ---------------------------------------------------------------------------
// A row of logits, in groups of 4 x 1024 vectors (fewer in the last): a wavefront
// has 4 x 64 vectors of a group in a row, of which lane l of its i-th load holds
// the (64 i + l)-th; elements behind the row read as -inf. The first group is kept
// in LDS, the others read again in every pass. Short passes go group by group, the
// next one under way (`each4`); long ones vector by vector, four under way
// (`each`): a row takes a pass only a few times round, and new code comes slowly
// (top_p of 256 x 128000 logits with all passes unrolled cost a fifth more).
// ---------------------------------------------------------------------------
template <int TYPE>
struct Row {
    static constexpr int VE = TYPE == W4A16_FP32 ? 4 : 8;
    const uint8_t* p;
    u32x4* staged;
    int n, rounds;

    // unaligned: a row may start at any element
    struct __attribute__((packed, aligned(2))) Loose {
        uint32_t w[4];
    };
    __device__ __forceinline__ int vector(int j, int wave) const {   // of another wavefront's lane
        const int group = j & ~3, each = min(4, rounds - group);
        return (group * kWaves + wave * each + (j & 3)) * 64 + (int)(threadIdx.x & 63);
    }
    __device__ __forceinline__ int vector(int j) const {
        return vector(j, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    }
    // The entry of the sums that a vector belongs to: a wavefront's of a group.
    __device__ __forceinline__ int entry(int index) const {
        const int v = index / (64 * VE), group = v / (4 * kWaves), each = min(4, rounds - 4 * group);
        return group * kWaves + (v - group * 4 * kWaves) / each;
    }
    __device__ __forceinline__ bool ends_group(int j) const { return (j & 3) == 3 || j + 1 == rounds; }
    __device__ __forceinline__ u32x4 read(int v) const {
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
    __device__ __forceinline__ u32x4 fetch(int j) const {
        if (j < kStaged) return staged[j * kThreads + threadIdx.x];
        return read(vector(min(j, rounds - 1)));
    }
    __device__ __forceinline__ u32x4 fetch(int j, int wave) const {
        if (j < kStaged) return staged[j * kThreads + wave * 64 + (threadIdx.x & 63)];
        return read(vector(j, wave));
    }
    // f(j, vector) for the thread's vectors, every lane taking part
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        u32x4 a = fetch(0), b = fetch(1), c = fetch(2), d = fetch(3);
#pragma unroll 1
        for (int j = 0; j < rounds; ++j) {
            const u32x4 now = a;
            a = b;
            b = c;
            c = d;
            d = fetch(j + 4);
            f(j, now);
        }
    }
    template <bool FIRST>
    __device__ __forceinline__ void fetch4(int group, u32x4 (&v)[4]) const {
        if (!FIRST && group == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = staged[i * kThreads + threadIdx.x];
        } else if ((group + 1) * 4 * kThreads * VE <= n) {
            const uint8_t* at = p + (int64_t)vector(4 * group) * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Loose w = *reinterpret_cast<const Loose*>(at + 1024 * i);
                v[i] = (u32x4){w.w[0], w.w[1], w.w[2], w.w[3]};
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = read(vector(min(4 * group + i, rounds - 1)));
        }
    }
    // the same; FIRST: the pass that brings the row in
    template <bool FIRST = false, typename F>
    __device__ __forceinline__ void each4(F f) const {
        u32x4 next[4], now[4];
        fetch4<FIRST>(0, next);
#pragma unroll 1
        for (int j = 0; j < rounds; j += 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) now[i] = next[i];
            if (j + 4 < rounds) fetch4<FIRST>(j / 4 + 1, next);
            if (FIRST && j == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) staged[i * kThreads + threadIdx.x] = now[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i == 0 || j + i < rounds) f(j + i, now[i]);
        }
    }
    __device__ __forceinline__ static float value(const u32x4& v, int e) {
        const uint32_t word = v[TYPE == W4A16_FP32 ? e : e >> 1];
        if constexpr (TYPE == W4A16_FP32)
            return __builtin_bit_cast(float, word);   // of the copy: of v[e] it is that of v[0]
        else
            return widen16<TYPE>(e & 1 ? word >> 16 : word & 0xFFFFu);
    }
    __device__ __forceinline__ float at(int index) const {
        if constexpr (TYPE == W4A16_FP32)
            return *reinterpret_cast<const float*>(p + 4 * (int64_t)index);
        else
            return widen16<TYPE>(*reinterpret_cast<const uint16_t*>(p + 2 * (int64_t)index));
    }
    __device__ __forceinline__ int index(int j, int e) const { return vector(j) * VE + e; }
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
    __device__ __forceinline__ static float of_key(uint32_t k) {
        if constexpr (TYPE == W4A16_FP32)
            return __builtin_bit_cast(float, k >> 31 ? k ^ 0x80000000u : ~k);
        else
            return widen16<TYPE>((k >> 15 ? k ^ 0x8000u : ~k) & 0xFFFFu);
    }
};

// a b + c, c in scalar registers: the compiler copies a coefficient into the result
// before each step otherwise (half of the weights' time).
__device__ __forceinline__ double fma_scalar(double a, double b, double c) {
    double r;
    asm volatile("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// The weights of a row's logits (the largest of them finite).
struct Weights {
    double top, factor, lowest;   // lowest: -60 / factor
    // 2^y of y = (x - top) factor <= 0: the whole part joins the exponent, 2^f with
    // |f| <= 1/2 is 1 + f times the polynomial that meets (2^f - 1) / f at the 8 Chebyshev
    // points of [-1/2, 1/2], off by 2^-38.7. What lies far below gives 2^-60. N of them step
    // by step together, as each operation waits for the one before (a pass over 50257
    // logits 11.2 us, one by one 12).
    template <int N>
    __device__ __forceinline__ void weights(const float (&x)[N], double (&w)[N]) const {
        constexpr double round = 0x1.8p52;
        double t[N], f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __builtin_fmax((double)x[i] - top, lowest);
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = __builtin_fma(f[i], factor, round);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __builtin_fma(f[i], factor, round - t[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = 1.325080551750225e-06;
        constexpr double terms[7] = {1.5303700711365693e-05, 0.00015403475186530786, 0.0013333478473685416,
                                     0.00961812913523614, 0.055504109063258665, 0.24022650695888503, 0.6931471805568324};
#pragma unroll
        for (int k = 0; k < 7; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = fma_scalar(w[i], f[i], terms[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = __builtin_fma(w[i], f[i], 1.0);
            w[i] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, w[i]) + (__builtin_bit_cast(uint64_t, t[i]) << 52));
        }
    }
    __device__ __forceinline__ double weight(float x) const {
        const float one[1] = {x};
        double w[1];
        weights(one, w);
        return w[0];
    }
    // round(2^44 w): the last bits of 2^8 + w
    __device__ __forceinline__ static uint64_t rounded(double w) {
        return __builtin_bit_cast(uint64_t, w + 0x1p8) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ uint64_t of(float x) const { return rounded(weight(x)); }
    // the same as doubles, multiples of 2^-44: sums below 2^9 of such are exact
    template <int N>
    __device__ __forceinline__ void parts(const float (&x)[N], double (&w)[N]) const {
        weights(x, w);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = (w[i] + 0x1p8) - 0x1p8;
    }
    __device__ __forceinline__ double part(float x) const { return (weight(x) + 0x1p8) - 0x1p8; }
};
__device__ __forceinline__ uint64_t whole(double parts) { return (uint64_t)(parts * (double)kOne); }

// The largest value of the workgroup; NaN if a thread brings `strange`. `flag`: of any thread.
__device__ __forceinline__ float block_max(Shared& s, float v, bool strange, bool& flag) {
    v = wave_max(v);
    if (__any(strange)) v = __builtin_nanf("");
    const int flags = __any(flag);
    if ((threadIdx.x & 63) == 0) {
        s.tops[threadIdx.x >> 6] = v;
        s.firsts[threadIdx.x >> 6] = flags;
    }
    __syncthreads();
    flag = __any(s.firsts[threadIdx.x & 15]);
    v = s.tops[threadIdx.x & 15];
    if (__any(v != v)) return __builtin_nanf("");
    v = fmaxf(v, dpp<0xB1>(v));
    v = fmaxf(v, dpp<0x4E>(v));
    v = fmaxf(v, dpp<0x141>(v));
    v = fmaxf(v, dpp<0x140>(v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ int block_min(Shared& s, int v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = min(v, __shfl_xor(v, d));
    __syncthreads();   // the memory may be read still
    if ((threadIdx.x & 63) == 0) s.firsts[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v = min(v, s.firsts[w]);
    return v;
}

// The sums of two values over the workgroup.
__device__ __forceinline__ void block_sums(Shared& s, uint64_t& a, uint64_t& b) {
    a = wave_scan(a);
    b = wave_scan(b);
    if ((threadIdx.x & 63) == 63) {
        s.sums[2 * (threadIdx.x >> 6)] = a;
        s.sums[2 * (threadIdx.x >> 6) + 1] = b;
    }
    __syncthreads();
    a = lane_of(row_scan(s.sums[2 * (threadIdx.x & 15)]), 15);
    b = lane_of(row_scan(s.sums[2 * (threadIdx.x & 15) + 1]), 15);
    __syncthreads();
}

// Bins of falling weight: 42 2/3 to a power of two, in fp32, so that a larger
// value never lies in a later bin; from kBins on they are of values without a weight. A
// value of bin i weighs 2^-(i .. i + 1) / 42.67, up to a thousandth of a bin
// (temperatures past 10^35 aside, whose bins do not tell the weights).
struct Bins {
    float top, quarter, per, lowest, none;   // per: bins to 4 units of the logits; lowest: of the values with a weight
    __device__ __forceinline__ int of(float x) const {
        // a quarter of the distance, which does not overflow
        return (int)__builtin_amdgcn_fmed3f(__builtin_fmaf(x, -0.25f, quarter) * per, 0.0f, none);
    }
};

__device__ __forceinline__ Bins bins_of(const Weights& w, float top) {
    const double reach = kOctaves / w.factor;
    return {top, 0.25f * top, (float)fmin(fmax(4.0 * w.factor * kBinsPerOctave, 2e-38), 3e38),
            (float)fmax(w.top - reach, -3.4028234663852886e38), (float)(kBins + (int)(threadIdx.x & 31))};
}

// Keys of values, from the largest of the bins `first` .. `last` to the smallest, a step wider.
struct Keys {
    uint32_t high, low;
};
template <typename R>
__device__ __forceinline__ Keys keys_of(const Bins& b, int first, int last) {
    const uint32_t top = R::key(b.top), lowest = R::key(b.lowest);
    Keys k = {top, lowest};
    const double bin = 4.0 / (double)b.per;
    if (first > 0) {
        const double x = (double)b.top - (first - 0.01) * bin;
        k.high = x > (double)b.lowest ? min(top, R::key((float)x) + 1) : lowest;
    }
    if (last < kBins - 1) {
        const double x = (double)b.top - (last + 1.01) * bin;
        k.low = x > (double)b.lowest ? max(lowest, R::key((float)x) - 1) : lowest;
    }
    return k;
}

__device__ __forceinline__ int shift_of(uint32_t range) { return max(0, 21 - __builtin_clz(range | 1)); }

__device__ __forceinline__ void clear_bins(Shared& s) {
    s.bins[threadIdx.x] = 0;
    s.bins[threadIdx.x + kThreads] = 0;
}

// The value at which the running sum of amount(x) over some values in falling order
// reaches `target`, level by level of 2048 ranges of their keys; `rest`: what of the
// target is left for that value. False where the sum stays below. `beside` is added
// for the value `tied`. each(f) calls f(x) for the values of a thread.
template <typename R, typename Each, typename Amount>
__device__ __forceinline__ bool select(Shared& s, Keys keys, uint64_t target, float tied, uint64_t beside, Each each,
                                       Amount amount, float& value, uint64_t& rest) {
    uint32_t from = keys.high, range = keys.high - keys.low;
    int shift = shift_of(range);
    while (true) {
        clear_bins(s);
        __syncthreads();
        each([&](float x) {
            const uint32_t d = from - R::key(x);
            if (d <= range) atomicAdd((unsigned long long*)&s.bins[d >> shift], (unsigned long long)amount(x));
        });
        if (threadIdx.x == 0 && beside != 0) {
            const uint32_t d = from - R::key(tied);
            if (d <= range) atomicAdd((unsigned long long*)&s.bins[d >> shift], (unsigned long long)beside);
        }
        __syncthreads();
        const Found f = find(s, kBins, [&](int i) { return s.bins[i]; }, [&](uint64_t) { return target; });
        if (f.index < 0) return false;
        target -= f.before;
        from -= (uint32_t)f.index << shift;
        range = (1u << shift) - 1;
        if (shift == 0) break;
        shift = max(0, shift - 11);
    }
    rest = target;
    value = R::of_key(from);
    return true;
}

// Appends indices to s.near, N a lane at most: a wavefront takes 64 places at a time (a
// count that all share for each vector is waited for: 600 of 50257 logits in 10.5 us, this
// way in 8). Past kMostNear they are only counted.
struct Near {
    int base = 0, room = 0;   // the wavefront's next place, and how many it has
    template <int N, typename Index>
    __device__ __forceinline__ void list(Shared& s, const bool (&has)[N], Index index) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < N; ++e) any |= has[e];
        if (!__any(any)) return;
        int total = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) total += __builtin_popcountll(__ballot(has[e]));
        if (total > room) {
            finish(s);
            room = max(total, 64);
            int at = 0;
            if ((threadIdx.x & 63) == 0) at = atomicAdd(&s.listed, room);
            base = __builtin_amdgcn_readfirstlane(at);
        }
        room -= total;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint64_t who = __ballot(has[e]);
            const int own =
                base + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
            if (has[e] && own < kMostNear) s.near[own] = index(e);
            base += __builtin_popcountll(who);
        }
    }
    // places that stay empty, fewer than 64
    __device__ __forceinline__ void finish(Shared& s) const {
        const int lane = threadIdx.x & 63;
        if (lane < room && base + lane < kMostNear) s.near[base + lane] = -1;
    }
};

// The sum and the ties of a wavefront's group that ends with vector j.
__device__ __forceinline__ void put_entry(Shared& s, int j, uint64_t sum, int equal) {
    sum = wave_scan(sum);
    if ((threadIdx.x & 63) != 63) return;
    const int at = (j >> 2) * kWaves + (threadIdx.x >> 6);
    s.kept[at] = sum;
    s.ties[at] = (uint32_t)equal;
}

// The logits that s.near lists, up to four a thread, -inf where there are none.
template <typename R>
__device__ __forceinline__ void load_near(const Shared& s, const R& r, float (&x)[kMostNear / kThreads]) {
#pragma unroll
    for (int i = 0; i < kMostNear / kThreads; ++i) {
        const int at = (int)threadIdx.x + i * kThreads, index = at < s.listed ? s.near[at] : -1;
        x[i] = index >= 0 ? r.at(index) : -__builtin_inff();
    }
}

// The draw among at most kList candidates that hold the top_k tokens, all
// comparisons and running sums by pairs: the pairs of candidate i = thread mod
// 64, 128 or 256 with a part of the others.
__device__ __forceinline__ void draw_listed(Shared& s, const Weights& weights, int64_t top_k, double top_p,
                                            float least, float u, int64_t* token) {
    const int tid = threadIdx.x, m = s.listed;
    const int width = m <= 64 ? 64 : m <= 128 ? 128 : 256;
    const int i = tid & (width - 1), parts = kThreads / width;
    const int per = (m + parts - 1) / parts, j0 = (tid / width) * per, j1 = min(j0 + per, m);
    if (tid < kList) {
        s.rank[tid] = 0;
        s.before[tid] = 0;
        if (tid < m) s.list[tid].weight = weights.of(s.list[tid].x);
    }
    __syncthreads();
    const Candidate own = s.list[min(i, m - 1)];
    {
        int rank = 0;
        uint64_t before = 0;
        for (int j = j0; j < j1; ++j) {
            const Candidate c = s.list[j];
            const bool better = c.x > own.x || (c.x == own.x && c.index < own.index);
            rank += better ? 1 : 0;
            before += better ? c.weight : 0;
        }
        if (i < m && rank != 0) {
            atomicAdd(&s.rank[i], rank);
            atomicAdd((unsigned long long*)&s.before[i], (unsigned long long)before);
        }
    }
    __syncthreads();
    // the weight of the top_k; the workgroup's first threads hold a candidate each
    uint64_t kept = tid < m && s.rank[tid] < top_k ? s.list[tid].weight : 0;
    const uint64_t better = tid < m ? s.before[tid] : 0;
    auto total_of = [&](uint64_t v) {
        const uint64_t sum = wave_scan(v);
        if ((tid & 63) == 63) s.sums[tid >> 6] = sum;
        __syncthreads();
        uint64_t total = 0;
#pragma unroll
        for (int w = 0; w < kList / 64; ++w) total += s.sums[w];
        __syncthreads();
        return total;
    };
    if (top_p < 1.0) {
        const double needed = fmax(__builtin_ceil(top_p * (double)total_of(kept)), 1.0);
        if ((double)better >= needed) kept = 0;
    }
    if (kept != 0 && s.list[tid].x < least) kept = 0;
    if (tid < m) s.list[tid].weight = kept;
    if (tid < kList) s.before[tid] = 0;
    const uint64_t total = total_of(kept);
    {
        uint64_t before = 0;
        for (int j = j0; j < j1; ++j) {
            const Candidate c = s.list[j];
            before += c.index < own.index ? c.weight : 0;
        }
        if (i < m && before != 0) atomicAdd((unsigned long long*)&s.before[i], (unsigned long long)before);
    }
    __syncthreads();
    const double at = (u > 0.0f ? (double)u : 0.0) * (double)total;   // NaN as 0
    const uint64_t target = at < (double)total ? min((uint64_t)at, total - 1) + 1 : total;
    if (tid < m && s.before[tid] < target && s.before[tid] + kept >= target) *token = s.list[tid].index;
}

// The smallest value whose weight is at least min_p of the largest one: 64 keys at a time.
template <typename R>
__device__ __forceinline__ float least_of(const Weights& w, const Bins& b, double min_p) {
    uint32_t low = R::key(b.lowest), high = R::key(b.top);   // the largest weighs enough
    while (low < high) {
        const uint32_t step = (high - low + 63) / 64;
        const uint32_t k = min(low + step * (threadIdx.x & 63), high);
        const uint64_t enough = __ballot(w.weight(R::of_key(k)) >= min_p);
        const int first = enough ? __builtin_ctzll(enough) : 64;
        const uint32_t up = min(low + step * first, high);
        low = first == 0 ? low : min(low + step * (first - 1) + 1, high);
        high = first == 0 ? low : up;
    }
    return R::of_key(high);
}

// What of a row is kept: values above `value`, and the first `ties` of those that equal it.
struct Limit {
    float value;
    int64_t ties;
};

// bf16 logits in falling order as whole numbers from the top's 0: by their bits,
// all magnitudes below 2^-20 as one. NaN have none.
struct Places {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    typedef int16_t s16x2 __attribute__((ext_vector_type(2)));
    static constexpr int kSmall = 0x357F;   // bits of the largest magnitude below 2^-20
    int top;
    u16x2 end;   // behind the values with a weight, lane by lane
    static __device__ __forceinline__ int level(float x) {
        const int bits = (int)(__builtin_bit_cast(uint32_t, x) >> 16);
        const int size = max((bits & 0x7FFF) - kSmall, 0);
        return bits & 0x8000 ? -size : size;
    }
    __device__ __forceinline__ int of(float x) const { return top - level(x); }
    __device__ __forceinline__ float value(int i) const {
        const int at = top - i;
        const uint32_t bits = at == 0 ? 0u : at > 0 ? (uint32_t)(at + kSmall) : (uint32_t)(kSmall - at) | 0x8000u;
        return __builtin_bit_cast(float, bits << 16);
    }
    // the smaller of `least` and the bits of two logits' magnitudes less 1 (0: none)
    static __device__ __forceinline__ u16x2 smaller(u16x2 least, uint32_t word) {
        return __builtin_elementwise_min(least, (__builtin_bit_cast(u16x2, word) & (u16x2)(0x7FFF)) - (u16x2)(1));
    }
    __device__ __forceinline__ u16x2 of(uint32_t word) const {   // of two logits, at most `end`
        const u16x2 bits = __builtin_bit_cast(u16x2, word);
        const u16x2 size = __builtin_elementwise_sub_sat(bits & (u16x2)(0x7FFF), (u16x2)((uint16_t)kSmall));
        const u16x2 sign = __builtin_bit_cast(u16x2, __builtin_bit_cast(s16x2, bits) >> (s16x2)(15));
        return __builtin_elementwise_min((u16x2)((uint16_t)top) - ((size ^ sign) - sign), end);
    }
};

// ---------------------------------------------------------------------------
// A workgroup a row.
//
// The row is read once: its largest value and each thread's. With a small top_k
// the threads' largest values give a bound that at least top_k values reach; the
// few that do are listed and drawn from. Else
//  - bf16 rows are counted by value where these are few: sums over the values
//    give the limits, and each value has its weight looked up;
//  - other rows are counted in bins of falling weight, which tell the bin that the
//    top_k-th token lies in, and between which bins top_p ends: one pass forms
//    every weight, sums those before by their places, and those between by their
//    values as well; what lies between is listed, so that the kept ones join the
//    sums of their places when the limit is known.
// The token is found by the sums of places, and then within a wavefront's vector.
//
// Bound: the instructions of one compute unit, as a row is a workgroup's: an
// instruction for every logit is 0.85 us of 128000, and a weight takes about twenty,
// most of them in 64 bits. One row of 32000 fp16 logits with top_k 50 and top_p:
// 9.3 us, of which 1.5 read it. fp32 rows of 50257 logits: without limits 18 us, by
// top_p 37 (2.5 to read, 4.5 to count, 2.5 for the bracket, 19 for the weights, 4 near
// the limit, 3 for the token), by a top_k of 600 31, by a narrower min_p 14 to 21. bf16
// rows by value: 16 of 32000 without limits 12.5 us, 256 of 128000 by top_p 43 us (65
// MB once: 13). fp16 rows without a small top_k go the fp32 rows' way (32000 logits by
// top_p 27 us, without limits 12; 50257: 37 and 17; 128000: 63 and 31). Not kept: a row in
// registers (their spills), weights eight at a time (the same). Not tried: a row over
// several workgroups, in launches that hand on the largest value, the sums and the limit
// (they would divide the reading, the counting and the weights, 26 of the 37 us).
// ---------------------------------------------------------------------------
template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    using R = Row<TYPE>;
    __shared__ Shared s;
    __shared__ u32x4 staged[kStaged * kThreads];

    const int row = blockIdx.x, tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    R r;
    r.p = a.logits + row * a.row_bytes;
    r.staged = staged;
    r.n = a.n;
    r.rounds = ((a.n + R::VE - 1) / R::VE + kThreads - 1) / kThreads;
    const float u = a.random[row];
    const double temperature = a.settings.temperatures ? (double)a.settings.temperatures[row] : a.settings.temperature;
    const int64_t top_k = a.settings.top_ks ? a.settings.top_ks[row] : a.settings.top_k;
    const double top_p = a.settings.top_ps ? (double)a.settings.top_ps[row] : a.settings.top_p;
    const double min_p = a.settings.min_ps ? (double)a.settings.min_ps[row] : a.settings.min_p;

    float mine = -__builtin_inff();
    bool strange = false;
    Places::u16x2 smallest = (Places::u16x2)(0xFFFF);   // bits of the smallest bf16 magnitudes but 0, less 1
    r.template each4<true>([&](int, const u32x4& v) {
        if constexpr (TYPE == W4A16_BF16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) smallest = Places::smaller(smallest, v[e]);
        }
#pragma unroll
        for (int e = 0; e < R::VE; ++e) {
            const float x = R::value(v, e);
            mine = fmaxf(mine, x);
            strange |= x != x;
        }
    });
    bool tiny = min(smallest.x, smallest.y) < Places::kSmall;   // the row has bf16 logits between 0 and 2^-20
    const float top = block_max(s, mine, strange, tiny);
    strange = top != top;
    // the first of the largest; a NaN counts as the largest, as in argmax
    if (strange || !(temperature > 0.0) || top == -__builtin_inff() || top_k == 1) {
        int first = a.n;
        r.each4([&](int j, const u32x4& v) {
#pragma unroll
            for (int e = 0; e < R::VE; ++e) {
                const float x = R::value(v, e);
                if (strange ? x != x : x == top) first = min(first, r.index(j, e));
            }
        });
        first = block_min(s, first);
        if (tid == 0) a.tokens[row] = first;
        return;
    }
    // the factor stays a number, and its product with a difference one
    const double factor = fmin(fmax(1.4426950408889634 / temperature, 1e-300), 1e200);
    const Weights weights = {(double)top, factor, -60.0 / factor};
    const Bins bins = bins_of(weights, top);
    const bool some = top_k > 0 && top_k < a.n, nucleus = top_p < 1.0;
    auto needed_of = [&](uint64_t total) {   // of the kept weight, at least 1
        const double needed = __builtin_ceil(top_p * (double)total);
        return needed >= 1.0 ? min((uint64_t)needed, total) : (uint64_t)1;
    };

    Limit limit = {-__builtin_inff(), a.n};
    uint64_t tie = 0;          // weight of a value that equals the limit
    bool summed = false;       // the entries hold the kept weights but for ties, whose counts are there where tie != 0
    if (top == __builtin_inff()) {   // infinite logits weigh 1, the others nothing
        int equal = 0;
        r.each([&](int, const u32x4& v) {
#pragma unroll
            for (int e = 0; e < R::VE; ++e) equal += R::value(v, e) == top ? 1 : 0;
        });
        uint64_t count = (uint64_t)equal, none = 0;
        block_sums(s, count, none);
        if (some) count = min(count, (uint64_t)top_k);
        limit = {top, (int64_t)(nucleus ? needed_of(count) : count)};
        tie = kOne;
    } else {
        const float least = min_p > 0.0 ? least_of<R>(weights, bins, fmin(min_p, 1.0)) : -__builtin_inff();
        if (some && top_k <= kList * 3 / 4) {
            // at least top_k values reach the bin that the top_k-th of the threads' largest values lies in
            s.counts[tid] = s.counts[tid + kThreads] = 0;
            if (tid == 0) s.listed = 0;
            __syncthreads();
            atomicAdd(&s.counts[bins.of(mine)], 1u);
            __syncthreads();
            const Found f = find(s, kBins, [&](int i) { return (uint64_t)s.counts[i]; },
                                 [&](uint64_t) { return (uint64_t)top_k; });
            const int last = f.index < 0 ? kBins - 1 : f.index;
            const float bound = R::of_key(keys_of<R>(bins, 0, last).low);
            r.each4([&](int j, const u32x4& v) {
                float most = R::value(v, 0);
#pragma unroll
                for (int e = 1; e < R::VE; ++e) most = fmaxf(most, R::value(v, e));
                if (most < bound) return;
#pragma unroll
                for (int e = 0; e < R::VE; ++e) {
                    const float x = R::value(v, e);
                    if (x >= bound) {
                        const int i = atomicAdd(&s.listed, 1);
                        if (i < kList) {
                            s.list[i].x = x;
                            s.list[i].index = r.index(j, e);
                        }
                    }
                }
            });
            __syncthreads();
            if (s.listed <= kList) {
                draw_listed(s, weights, top_k, top_p, least, u, &a.tokens[row]);
                return;
            }
            __syncthreads();
        }
        bool limited = false;
        if constexpr (TYPE == W4A16_BF16) {
            Places places;
            places.top = Places::level(top);
            const int end = places.of(bins.lowest) + 1;
            if (end <= kValues && (some || nucleus || a.n > end) && !(tiny && places.top <= 0)) {
                places.end = (Places::u16x2)((uint16_t)(end + (tid & 31)));
                const int small = places.top >= 0 ? places.top : -1;   // the place of magnitudes below 2^-20
                const bool counted = some || nucleus;   // else min_p alone gives a limit
                if (counted) {
                    for (int i = tid; i < end + 32; i += kThreads) s.value_counts[i] = 0;
                    __syncthreads();
                    r.each4([&](int, const u32x4& v) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const Places::u16x2 at = places.of(v[e]);
                            atomicAdd(&s.value_counts[at.x], 1u);
                            atomicAdd(&s.value_counts[at.y], 1u);
                        }
                    });
                }
                __syncthreads();
                for (int i = tid; i < end; i += kThreads)
                    if (!counted || s.value_counts[i] != 0) s.value_weights[i] = weights.of(places.value(i));
                __syncthreads();
                // magnitudes between 0 and 2^-20, which share a place with 0: the few that there
                // may be have their weights added apart
                uint64_t excess = 0, all_excess = 0;
                if (tiny) {
                    if (tid == 0) s.tinies = 0;
                    __syncthreads();
                    r.each4([&](int j, const u32x4& v) {
                        Places::u16x2 own = (Places::u16x2)(0xFFFF);
#pragma unroll
                        for (int e = 0; e < 4; ++e) own = Places::smaller(own, v[e]);
                        if (min(own.x, own.y) >= Places::kSmall) return;
#pragma unroll
                        for (int e = 0; e < R::VE; ++e) {
                            const float x = R::value(v, e);
                            if (fabsf(x) < 0x1p-20f && x != 0.0f) {
                                const int i = atomicAdd(&s.tinies, 1);
                                if (i < kTiny) s.tiny[i] = r.index(j, e);
                            }
                        }
                    });
                    __syncthreads();
                    if (lane < s.tinies && lane < kTiny) excess = weights.of(r.at(s.tiny[lane])) - weights.of(0.0f);
                    all_excess = lane_of(wave_scan(excess), 63);
                }
                int last = end - 1;        // the limit's place
                uint64_t ties = ~0ull;
                if (some) {
                    const Found f = find<7>(s, end, [&](int i) { return (uint64_t)s.value_counts[i]; },
                                            [&](uint64_t) { return (uint64_t)top_k; });
                    if (f.index >= 0) {   // else fewer have a weight
                        last = f.index;
                        ties = (uint64_t)top_k - f.before;
                    }
                }
                const bool among = tiny && last == small;   // top_k ends among different values of one place
                if (nucleus) {
                    uint64_t target = 0;
                    const Found f = find<7>(s, end, [&](int i) {
                        const uint64_t n = i < last ? s.value_counts[i] : i == last ? min((uint64_t)s.value_counts[i], ties) : 0;
                        return n == 0 ? 0 : n * s.value_weights[i] + (i == small ? all_excess : 0);
                    }, [&](uint64_t total) { return target = needed_of(total); });
                    last = f.index;
                    const uint64_t w = max(s.value_weights[last], (uint64_t)1);
                    ties = (target - f.before + w - 1) / w;
                }
                if (least > places.value(last)) {
                    last = places.of(least);
                    ties = least > places.value(last) ? 0 : ~0ull;   // a bound between 0 and 2^-20 keeps no 0
                }
                // a limit there, or too many of them: the other way
                if (!tiny || (!among && last != small && s.tinies <= kTiny)) {
                    limited = true;
                    limit = {places.value(last), (int64_t)min(ties, (uint64_t)a.n)};
                    tie = !counted || s.value_counts[last] != 0 ? s.value_weights[last] : 0;
                    // each value's weight is looked up, 0 of the limit and below
                    __syncthreads();
                    for (int i = tid; i < end + 32; i += kThreads)
                        if (i >= last || (counted && s.value_counts[i] == 0)) s.value_weights[i] = 0;
                    __syncthreads();
                    const uint16_t last16 = (uint16_t)last;
                    places.end = (Places::u16x2)((uint16_t)(last + 1 + (tid & 31)));   // zeros of many banks
                    uint64_t sum = 0;
                    int equal = 0;
                    r.each4([&](int j, const u32x4& v) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const Places::u16x2 at = places.of(v[e]);
                            sum += s.value_weights[at.x] + s.value_weights[at.y];
                            equal += __builtin_popcountll(__ballot(at.x == last16)) +
                                     __builtin_popcountll(__ballot(at.y == last16));
                        }
                        if (!r.ends_group(j)) return;
                        put_entry(s, j, sum, equal);
                        sum = 0;
                        equal = 0;
                    });
                    __syncthreads();
                    if (tiny && small < last) {
                        if (tid < s.tinies) atomicAdd((unsigned long long*)&s.kept[r.entry(s.tiny[tid])], (unsigned long long)excess);
                        __syncthreads();
                    }
                    summed = true;
                }
                __syncthreads();
            }
        }
        if (!limited && (some || nucleus)) {
            s.counts[tid] = s.counts[tid + kThreads] = 0;
            __syncthreads();
            r.each4([&](int, const u32x4& v) {
#pragma unroll
                for (int e = 0; e < R::VE; ++e) atomicAdd(&s.counts[bins.of(R::value(v, e))], 1u);
            });
            __syncthreads();
            int last_bin = kBins - 1;
            uint64_t in_last = ~0ull;   // tokens of the last bin that top_k leaves
            if (some) {
                const Found f = find(s, kBins, [&](int i) { return (uint64_t)s.counts[i]; },
                                     [&](uint64_t) { return (uint64_t)top_k; });
                if (f.index >= 0) {   // else fewer have a weight
                    last_bin = f.index;
                    in_last = (uint64_t)top_k - f.before;
                    uint64_t rest = 0;
                    // few kept tokens are listed all, else those of the last bin
                    const int from = top_k <= kMostNear * 5 / 8 ? 0 : last_bin;
                    if (tid == 0) s.listed = 0;
                    __syncthreads();
                    // (wider than the bins by a little)
                    const Keys bounds = keys_of<R>(bins, from, last_bin);
                    const float high = from > 0 ? R::of_key(bounds.high) : __builtin_inff();
                    const float low = fmaxf(R::of_key(bounds.low), -3.4028234663852886e38f);
                    Near listed;
                    r.each4([&](int j, const u32x4& v) {
                        bool in[R::VE];
#pragma unroll
                        for (int e = 0; e < R::VE; ++e) in[e] = R::value(v, e) <= high && R::value(v, e) >= low;
                        listed.list<R::VE>(s, in, [&](int e) { return r.index(j, e); });
                    });
                    listed.finish(s);
                    __syncthreads();
                    const Keys keys = keys_of<R>(bins, last_bin, last_bin);
                    auto one = [](float) { return (uint64_t)1; };
                    const bool near = s.listed <= kMostNear;   // all are listed
                    float x[kMostNear / kThreads];
                    if (near) {
                        load_near(s, r, x);
                        select<R>(s, keys, in_last, 0.0f, 0, [&](auto f) {
#pragma unroll
                            for (int i = 0; i < kMostNear / kThreads; ++i)
                                if (x[i] > -__builtin_inff() && bins.of(x[i]) == last_bin) f(x[i]);
                        }, one, limit.value, rest);
                    } else {
                        select<R>(s, keys, in_last, 0.0f, 0, [&](auto f) {
                            r.each([&](int, const u32x4& v) {
#pragma unroll
                                for (int e = 0; e < R::VE; ++e)
                                    if (bins.of(R::value(v, e)) == last_bin) f(R::value(v, e));
                            });
                        }, one, limit.value, rest);
                    }
                    limit.ties = (int64_t)rest;
                    if (from == 0 && near) {   // all that follows is about the listed ones
                        limited = summed = true;
                        auto above = [&](auto f) {
#pragma unroll
                            for (int i = 0; i < kMostNear / kThreads; ++i)
                                if (x[i] > limit.value) f(x[i]);
                        };
                        if (nucleus) {
                            uint64_t total = 0, none = 0;
                            above([&](float y) { total += weights.of(y); });
                            block_sums(s, total, none);
                            const uint64_t beside = weights.of(limit.value) * rest;
                            total += beside;
                            float value = limit.value;
                            select<R>(s, keys_of<R>(bins, 0, last_bin), needed_of(total), limit.value, beside, above,
                                      [&](float y) { return weights.of(y); }, value, rest);
                            const uint64_t w = max(weights.of(value), (uint64_t)1);
                            limit = {value, (int64_t)((rest + w - 1) / w)};
                        }
                        if (least > limit.value) limit = {least, a.n};
                        tie = weights.of(limit.value);
                        for (int i = tid; i < kMostEntries; i += kThreads) {
                            s.kept[i] = 0;
                            s.ties[i] = 0;
                        }
                        __syncthreads();
#pragma unroll
                        for (int i = 0; i < kMostNear / kThreads; ++i) {
                            if (!(x[i] >= limit.value)) continue;
                            const int entry = r.entry(s.near[tid + i * kThreads]);
                            if (x[i] > limit.value)
                                atomicAdd((unsigned long long*)&s.kept[entry], (unsigned long long)weights.of(x[i]));
                            else
                                atomicAdd(&s.ties[entry], 1u);
                        }
                        __syncthreads();
                    }
                }
            }
            if (nucleus && !limited) {
                // The weight of bin i is at least its count times 2^-(i + 1.01) / 42.67, and less than 1.02 times that.
                auto least_weight = [&](int i) {
                    const uint64_t n = i < last_bin ? s.counts[i] : i == last_bin ? min((uint64_t)s.counts[i], in_last) : 0;
                    return (uint64_t)((double)n * (double)kOne * (double)__builtin_amdgcn_exp2f(-(i + 1.01f) / kBinsPerOctave));
                };
                // so for each bin the share up to it, and the share behind it, are known to 1.02
                const Found f0 = find(s, kBins, least_weight, [&](uint64_t total) {
                    return (uint64_t)fmax(fmax(top_p / 1.02, 1.0 - 1.02 * (1.0 - top_p)) * (double)total, 1.0);
                });
                const Found f1 = find(s, kBins, least_weight, [&](uint64_t total) {
                    return (uint64_t)fmax(fmin(1.02 * top_p, 1.0 - (1.0 - top_p) / 1.02) * (double)total, 1.0);
                });
                int first_bin = max(f0.index, 0), end_bin = f1.index >= 0 ? f1.index : kBins - 1;
                const Limit by_count = limit;
                const uint64_t beside =
                    by_count.value == -__builtin_inff() ? 0 : weights.of(by_count.value) * (uint64_t)by_count.ties;
                // Where min_p keeps none but of the bins before, all of which top_p keeps, the
                // sum is of no use (where the bins tell the weights: the share behind them
                // by far more than what 2^19 roundings of a weight make).
                const bool known = first_bin > 0 && top_p <= 0.999 && factor > 1e-30 && factor < 1e30 &&
                                   least > limit.value && least >= R::of_key(keys_of<R>(bins, first_bin, end_bin).high);
                while (!known) {
                    // what lies between, by value; from `high` on it is certain to be kept
                    const Keys keys = keys_of<R>(bins, first_bin, end_bin);
                    const float high = first_bin > 0 ? R::of_key(keys.high) : __builtin_inff(), low = R::of_key(keys.low);
                    if (tid == 0) s.listed = 0;
                    __syncthreads();
                    double all = 0.0, above = 0.0, group = 0.0;
                    r.each([&](int j, const u32x4& v) {
#pragma unroll
                        for (int e0 = 0; e0 < R::VE; e0 += 4) {
                            float x[4];
                            double w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = R::value(v, e0 + e);
                            weights.parts(x, w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const bool counts = x[e] > by_count.value;
                                w[e] = counts ? w[e] : 0.0;
                                all += w[e];
                                group += x[e] > high ? w[e] : 0.0;
                                if (counts && x[e] <= high && x[e] >= low) {   // few: one by one
                                    const int i = atomicAdd(&s.listed, 1);
                                    if (i < kMostNear) s.near[i] = r.index(j, e0 + e);
                                }
                            }
                        }
                        if (!r.ends_group(j)) return;
                        put_entry(s, j, whole(group), 0);
                        above += group;
                        group = 0.0;
                    });
                    uint64_t total = whole(all), sure = whole(above);
                    block_sums(s, total, sure);
                    total += beside;
                    const bool near = s.listed <= kMostNear;   // all are listed
                    const uint64_t target = needed_of(total);
                    uint64_t rest = 0;
                    float value = by_count.value;
                    const uint64_t tied = by_count.value <= high && by_count.value >= low ? beside : 0;
                    auto amount = [&](float x) { return weights.of(x); };
                    float x[kMostNear / kThreads];
                    bool found = target > sure;
                    if (near) {
                        load_near(s, r, x);
                        if (found)
                            found = select<R>(s, keys, target - sure, by_count.value, tied, [&](auto f) {
#pragma unroll
                                for (int i = 0; i < kMostNear / kThreads; ++i)
                                    if (x[i] > -__builtin_inff()) f(x[i]);
                            }, amount, value, rest);
                    } else if (found) {
                        found = select<R>(s, keys, target - sure, by_count.value, tied, [&](auto f) {
                            r.each([&](int, const u32x4& v) {
#pragma unroll
                                for (int e = 0; e < R::VE; ++e) {
                                    const float y = R::value(v, e);
                                    if (y <= high && y >= low && y > by_count.value) f(y);
                                }
                            });
                        }, amount, value, rest);
                    }
                    if (!found && (first_bin > 0 || end_bin < kBins - 1)) {   // the bins do not tell
                        first_bin = 0;
                        end_bin = kBins - 1;
                        __syncthreads();
                        continue;
                    }
                    const uint64_t w = max(weights.of(value), (uint64_t)1);
                    limit = {value, (int64_t)((rest + w - 1) / w)};
                    // of a value that ties at top_k none is listed
                    if (near && value != by_count.value && least <= value) {
                        summed = true;
                        __syncthreads();
#pragma unroll
                        for (int i = 0; i < kMostNear / kThreads; ++i) {
                            if (!(x[i] >= value)) continue;
                            const int entry = r.entry(s.near[tid + i * kThreads]);
                            if (x[i] > value)
                                atomicAdd((unsigned long long*)&s.kept[entry], (unsigned long long)weights.of(x[i]));
                            else
                                atomicAdd(&s.ties[entry], 1u);
                        }
                        __syncthreads();
                    }
                    break;
                }
            }
        }
        if (!limited && !summed) {
            if (least > limit.value) limit = {least, a.n};
            tie = limit.value == -__builtin_inff() ? 0 : weights.of(limit.value);
        } else if (!limited) {
            tie = weights.of(limit.value);
        }
    }

    if (!summed) {
        // sums of what is kept, ties apart as their places are not known yet
        const bool all = limit.value == -__builtin_inff();
        double sum = 0.0;
        int equal = 0;
        r.each([&](int j, const u32x4& v) {
            if (all) {
#pragma unroll
                for (int e0 = 0; e0 < R::VE; e0 += 4) {
                    float x[4];
                    double w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = R::value(v, e0 + e);
                    weights.parts(x, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += w[e];
                }
            } else {
                float most = R::value(v, 0);
#pragma unroll
                for (int e = 1; e < R::VE; ++e) most = fmaxf(most, R::value(v, e));
                if (__any(most >= limit.value)) {
#pragma unroll
                    for (int e = 0; e < R::VE; ++e) {
                        const float x = R::value(v, e);
                        const bool above = x > limit.value;
                        if (__any(above)) {
                            const double w = weights.part(x);
                            sum += above ? w : 0.0;
                        }
                        equal += __builtin_popcountll(__ballot(x == limit.value));
                    }
                }
            }
            if (!r.ends_group(j)) return;
            put_entry(s, j, whole(sum), equal);
            sum = 0.0;
            equal = 0;
        });
        __syncthreads();
    }

    // the wavefront and group that hold the token
    const int entries = (r.rounds + 3) / 4 * kWaves;
    if (tie != 0) {   // ties before each entry, and of the kept ones the weight
        const uint64_t own = tid < entries ? s.ties[tid] : 0;
        const uint64_t upto = wave_scan(own);
        if (lane == 63) s.sums[wave] = upto;
        __syncthreads();
        const uint64_t waves = row_scan(s.sums[tid & 15]);
        const int64_t before = (int64_t)(upto - own + (wave > 0 ? lane_of(waves, wave - 1) : 0));
        if (tid < entries) {
            s.kept[tid] += tie * (uint64_t)min(max((int64_t)0, limit.ties - before), (int64_t)own);
            s.ties[tid] = (uint32_t)before;
        }
        __syncthreads();
    }
    uint64_t target = 0;
    const Found f = find<1>(s, entries, [&](int i) { return s.kept[i]; }, [&](uint64_t total) {
        const double at = (u > 0.0f ? (double)u : 0.0) * (double)total;   // NaN as 0
        return target = at < (double)total ? min((uint64_t)at, total - 1) + 1 : total;
    });
    // and there the vector, a wavefront each, and the lane: what lies above the limit first
    const int owner = f.index % kWaves, j = f.index / kWaves * 4 + wave;
    const bool works = f.index >= 0 && wave < 4 && j < r.rounds;
    float x[R::VE];
    uint64_t own[R::VE], sum = 0, upto = 0;
    int equal = 0, equal_upto = 0;
    if (works) {
        const u32x4 v = r.fetch(j, owner);
#pragma unroll
        for (int e = 0; e < R::VE; ++e) x[e] = R::value(v, e);
#pragma unroll
        for (int e0 = 0; e0 < R::VE; e0 += 4) {
            const float y[4] = {x[e0], x[e0 + 1], x[e0 + 2], x[e0 + 3]};
            double w[4];
            weights.weights(y, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                own[e0 + e] = y[e] > limit.value ? Weights::rounded(w[e]) : 0;
                sum += own[e0 + e];
                equal += tie != 0 && y[e] == limit.value ? 1 : 0;
            }
        }
        upto = wave_scan(sum);
        if (tie != 0) equal_upto = (int)wave_scan((uint64_t)equal);
        if (lane == 63) {
            s.sums[wave] = upto;
            s.firsts[wave] = equal_upto;
        }
    }
    __syncthreads();
    if (!works) return;
    uint64_t before = f.before;
    int64_t left = tie != 0 ? limit.ties - (int64_t)s.ties[f.index] : 0;   // ties that are kept from here on
    auto kept_of = [&](int n) { return tie * (uint64_t)min(max(left, (int64_t)0), (int64_t)n); };
    for (int w = 0; w < wave; ++w) {
        before += s.sums[w] + kept_of(s.firsts[w]);
        left -= s.firsts[w];
    }
    uint64_t below = before + upto - sum + kept_of(equal_upto - equal);
    if (below >= target || before + upto + kept_of(equal_upto) < target) return;
    left -= equal_upto - equal;
    int e = 0;
#pragma unroll
    for (int i = 0; i < R::VE; ++i) {
        if (tie != 0 && x[i] == limit.value && left-- > 0) own[i] = tie;
        below += own[i];
        if (below < target) e = i + 1;
    }
    a.tokens[row] = r.vector(j, owner) * R::VE + e;
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
