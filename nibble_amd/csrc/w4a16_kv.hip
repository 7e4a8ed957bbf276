// The 8-bit key/value cache: rotary positions, writing tokens and reading the
// cache back (include/w4a16_kv.h states what each computes). Attention over
// the cache is in w4a16_kv_attn.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <utility>

#include "w4a16_hip.h"
#include "w4a16_kv_device.h"
#include "w4a16_kv_host.h"

namespace w4a16 {

// ---------------------------------------------------------------------------
// Rotary positions.
//
// Bound: memory, 2 bytes read and 2 written per value. A thread holds one unit
// of HPT heads of one token, so that a token's table rows are read once for HPT
// heads: two vectors of 8 values that rotate each other (dims 8 u and rot / 2 +
// 8 u), or any two of interleaved or copied dims, half a row apart, so that the
// lanes of a row lie next to each other.
// ---------------------------------------------------------------------------
struct Unit {
    int lo, hi;                  // dims of its two vectors of 8 values
    bool lo_turned, hi_turned;   // half layout: both or none
    int one, two;                // table columns of the pairs: 4 from each, or (half layout) 8 from the first
};
template <bool INTERLEAVED>
__device__ __forceinline__ Unit unit_of(int u, int dim, int rot) {
    Unit t;
    if constexpr (INTERLEAVED) {
        t.lo = 8 * u;
        t.hi = 8 * u + dim / 2;
        t.lo_turned = t.lo < rot;
        t.hi_turned = t.hi < rot;
        t.one = t.lo_turned ? t.lo / 2 : 0;
        t.two = t.hi_turned ? t.hi / 2 : 0;
    } else {
        const bool turned = 16 * u < rot;
        t.lo = turned ? 8 * u : 8 * u + rot / 2;
        t.hi = t.lo + (turned ? rot : dim - rot) / 2;
        t.lo_turned = t.hi_turned = turned;
        t.one = turned ? t.lo : 0;
        t.two = t.one + 4;
    }
    return t;
}

// The unit's vectors rotated where they are turned, rounded to the rows' type.
template <int TYPE, bool INTERLEAVED>
__device__ __forceinline__ void rotate_unit(const Unit& t, u32x4& a, u32x4& b, const float (&c)[8], const float (&s)[8]) {
    float x1[8], x2[8];
    widen8<TYPE>(a, x1);
    widen8<TYPE>(b, x2);
    if constexpr (INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            rotate_pair(x1[2 * j], x1[2 * j + 1], c[j], s[j]);
            rotate_pair(x2[2 * j], x2[2 * j + 1], c[4 + j], s[4 + j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) rotate_pair(x1[j], x2[j], c[j], s[j]);
    }
    const u32x4 r1 = narrow8<TYPE>(x1), r2 = narrow8<TYPE>(x2);
    a = t.lo_turned ? r1 : a;
    b = t.hi_turned ? r2 : b;
}

struct RotaryArgs {
    const uint16_t* x;
    uint16_t* out;
    const float *cos_table, *sin_table;
    const int64_t* positions;    // of (b, t), or, beside a write, start[b] + t
    const int64_t *start, *counts;
    int64_t xb, xt, xh, pb, pt, table_rows, slots;
    int batch, tokens, heads, dim, rot, head_groups;
};

template <int TYPE, bool INTERLEAVED, int HPT, bool BESIDE_WRITE>
__device__ __forceinline__ void rotary_units(const RotaryArgs& a, int64_t first) {
    const int units = a.dim >> 4;
    const int64_t total = (int64_t)a.batch * a.tokens * a.head_groups * units;
    if (first >= total) return;
    const int u = (int)(first % units);
    int64_t rest = first / units;
    const int hg = (int)(rest % a.head_groups);
    rest /= a.head_groups;
    const int t = (int)(rest % a.tokens), b = (int)(rest / a.tokens);

    const Unit unit = unit_of<INTERLEAVED>(u, a.dim, a.rot);
    uint16_t* out = a.out + ((int64_t)b * a.tokens + t) * a.heads * a.dim;
    if (BESIDE_WRITE && a.counts != nullptr && t >= a.counts[b]) {
        // padding: zeros, and the rows are not read
        for (int h = hg; h < a.heads; h += a.head_groups) {
            *reinterpret_cast<u32x4*>(out + (int64_t)h * a.dim + unit.lo) = (u32x4){0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4*>(out + (int64_t)h * a.dim + unit.hi) = (u32x4){0u, 0u, 0u, 0u};
        }
        return;
    }
    // Rows before positions where there are positions (12.5 against 14.5 us for 2 x 2011 tokens, 32 heads of 128),
    // and after the start beside a write (37.4 against 38.7 us for 4 x 2000 tokens, 32/8 heads of 128).
    int64_t p, limit;
    if constexpr (BESIDE_WRITE) {
        p = min(a.start[b], a.slots) + t;   // past the slots: outside, and no sum that wraps
        limit = a.slots;
    }
    u32x4 va[HPT], vb[HPT];
    const uint16_t* x = a.x + b * a.xb + t * a.xt;
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
        const uint16_t* row = x + min(hg + i * a.head_groups, a.heads - 1) * a.xh;
        va[i] = *reinterpret_cast<const u32x4*>(row + unit.lo);
        vb[i] = *reinterpret_cast<const u32x4*>(row + unit.hi);
    }
    if constexpr (!BESIDE_WRITE) {
        __builtin_amdgcn_sched_barrier(0);
        p = a.positions[b * a.pb + t * a.pt];
        limit = a.table_rows;
    }
    const bool known = p >= 0 && p < limit;
    float c[8], s[8];
    const int64_t at = (known ? p : 0) * (a.rot / 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = known ? a.cos_table[at + unit.one + i] : __builtin_nanf("");
        s[i] = known ? a.sin_table[at + unit.one + i] : __builtin_nanf("");
        c[4 + i] = known ? a.cos_table[at + unit.two + i] : __builtin_nanf("");
        s[4 + i] = known ? a.sin_table[at + unit.two + i] : __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
        const int h = hg + i * a.head_groups;
        if (h >= a.heads) break;
        rotate_unit<TYPE, INTERLEAVED>(unit, va[i], vb[i], c, s);
        uint16_t* row = out + (int64_t)h * a.dim;
        *reinterpret_cast<u32x4*>(row + unit.lo) = va[i];
        *reinterpret_cast<u32x4*>(row + unit.hi) = vb[i];
    }
}

template <int TYPE, bool INTERLEAVED, int HPT>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    rotary_units<TYPE, INTERLEAVED, HPT, false>(a, (int64_t)blockIdx.x * blockDim.x + threadIdx.x);
}

// Any even rot, any head_dim and any alignment: a thread per pair or copied value.
template <int TYPE, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_any_kernel(const RotaryArgs a) {
    const int half = a.rot / 2, per_head = half + a.dim - a.rot;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.batch * a.tokens * a.heads * per_head) return;
    const int j = (int)(i % per_head);
    int64_t rest = i / per_head;
    const int h = (int)(rest % a.heads);
    rest /= a.heads;
    const int t = (int)(rest % a.tokens), b = (int)(rest / a.tokens);
    const uint16_t* x = a.x + b * a.xb + t * a.xt + h * a.xh;
    uint16_t* out = a.out + (rest * a.heads + h) * a.dim;
    if (j >= half) {
        out[half + j] = x[half + j];   // dim rot + (j - half)
        return;
    }
    const int64_t p = a.positions[b * a.pb + t * a.pt];
    const bool known = p >= 0 && p < a.table_rows;
    const int64_t at = (known ? p : 0) * half + j;
    const float c = known ? a.cos_table[at] : __builtin_nanf(""), s = known ? a.sin_table[at] : __builtin_nanf("");
    const int one = INTERLEAVED ? 2 * j : j, two = INTERLEAVED ? one + 1 : one + half;
    float x1 = widen16<TYPE>(x[one]), x2 = widen16<TYPE>(x[two]);
    rotate_pair(x1, x2, c, s);
    out[one] = (uint16_t)narrow16<TYPE>(x1);
    out[two] = (uint16_t)narrow16<TYPE>(x2);
}

// ---------------------------------------------------------------------------
// Writing tokens.
//
// Bound: memory (2 bytes read and 1 written per value) for prompts, one chain
// of latencies (start, rows, scale, stores) for single tokens. A workgroup
// owns one block of one head's keys or values: it holds the block's new rows
// in registers (UPT units of 16 values a thread), reduces their magnitude, and
// writes codes under the joint scale, so that every value is read once and no
// other workgroup touches the block's scale. Only where the scale of a block
// with earlier tokens grows are those read and rescaled.
// ---------------------------------------------------------------------------
struct WriteSide {
    const uint16_t* x;
    uint8_t* codes;
    float* scales;
    int64_t xb, xt, xh, cb, ch, sb, sh;
    bool vec;   // rows are 16-byte aligned
};

struct WriteArgs {
    WriteSide side[2];   // keys, values
    const int64_t *start, *counts;
    const float *cos_table, *sin_table;   // of the keys, or NULL
    int64_t slots;
    int tokens, kv_heads, batch, dim, block, rot;
};

template <int TYPE, int CODES, bool ROTATE, bool INTERLEAVED, int UPT>
__device__ __forceinline__ void write_block(const WriteArgs& a, int item) {
    __shared__ float wave_amax[4];
    const int values = item & 1;   // 0 keys, 1 values
    item >>= 1;
    const int h = item % a.kv_heads;
    item /= a.kv_heads;
    const int b = item % a.batch, jrel = item / a.batch;
    const WriteSide& w = a.side[values];

    const int64_t start = min(a.start[b], a.slots);   // past the slots: nothing to write
    int64_t count = a.tokens;
    if (a.counts != nullptr) count = min(max(a.counts[b], (int64_t)0), count);
    const int64_t lo = max(start, (int64_t)0), hi = min(start + count, a.slots);
    const int64_t j = lo / a.block + jrel;
    const int64_t r0 = max(lo, j * a.block), r1 = min(hi, (j + 1) * a.block);
    if (r0 >= r1) return;   // the whole workgroup
    const int rows = (int)(r1 - r0), earlier = (int)(r0 - j * a.block);
    float* scale_at = w.scales + b * w.sb + h * w.sh + j;
    const float was = earlier > 0 ? *scale_at : 0.0f;

    const int per_row = a.dim >> 4;
    const int units = rows * per_row;
    const uint16_t* x = w.x + b * w.xb + h * w.xh + (r0 - start) * w.xt;
    const bool rotate = ROTATE && values == 0;
    float amax = 0.0f;
    u32x4 raw[UPT][2];
    Unit unit[UPT];
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
        const int u = min((int)(threadIdx.x + i * blockDim.x), units - 1);
        const int r = u / per_row;
        unit[i] = unit_of<INTERLEAVED>(u - r * per_row, a.dim, rotate ? a.rot : a.dim);
        raw[i][0] = load8(x + r * w.xt + unit[i].lo, w.vec);
        raw[i][1] = load8(x + r * w.xt + unit[i].hi, w.vec);
    }
    if constexpr (ROTATE) {
        if (rotate) {
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                const int u = min((int)(threadIdx.x + i * blockDim.x), units - 1);
                const int64_t at = (r0 + u / per_row) * (a.rot / 2);
                float c[8], s[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[e] = a.cos_table[at + unit[i].one + e];
                    s[e] = a.sin_table[at + unit[i].one + e];
                    c[4 + e] = a.cos_table[at + unit[i].two + e];
                    s[4 + e] = a.sin_table[at + unit[i].two + e];
                }
                // the cache holds keys as the rotary op returns them: rounded to the rows' type
                rotate_unit<TYPE, INTERLEAVED>(unit[i], raw[i][0], raw[i][1], c, s);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < UPT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v[8];
            widen8<TYPE>(raw[i][k], v);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = __builtin_fmaxf(amax, __builtin_fabsf(v[e]));   // (leaves NaN out)
        }
    amax = wave_max(amax);
    if (blockDim.x > 64) {
        if ((threadIdx.x & 63) == 0) wave_amax[threadIdx.x >> 6] = amax;
        __syncthreads();
        for (int i = 0; i < (int)(blockDim.x >> 6); ++i) amax = __builtin_fmaxf(amax, wave_amax[i]);
    }
    // infinities count as the largest finite value (bf16's lies past the scales' range, as infinity does)
    if constexpr (TYPE == W4A16_FP16) amax = __builtin_fminf(amax, 65504.0f);
    float scale = exp2_int(scale_exponent<CODES>(amax));
    if (earlier > 0) scale = __builtin_fmaxf(scale, was);
    const float inverse = exp2_int(-exponent_of(scale));

    uint8_t* codes = w.codes + b * w.cb + h * w.ch;
    uint8_t* fresh = codes + r0 * a.dim;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
        const int u = threadIdx.x + i * blockDim.x;
        if (u >= units) break;
        uint8_t* row = fresh + (u / per_row) * a.dim;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v[8];
            widen8<TYPE>(raw[i][k], v);
            uint32_t c[4];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] == v[e] ? v[e] * inverse : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = encode2<CODES>(v[2 * e], v[2 * e + 1]);
            *reinterpret_cast<uint2*>(row + (k ? unit[i].hi : unit[i].lo)) =
                make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
        }
    }
    if (threadIdx.x == 0) *scale_at = scale;
    if (earlier > 0 && scale > was) {
        const float ratio = was * inverse;
        uint2* held = reinterpret_cast<uint2*>(codes + j * a.block * a.dim);
        for (int u = threadIdx.x; u < earlier * (a.dim >> 3); u += blockDim.x) {
            const uint2 q = held[u];
            uint32_t o[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t word = e ? q.y : q.x;
                const f32x2 l = decode2_f32<CODES, false>(word), m = decode2_f32<CODES, true>(word);
                o[e] = encode2<CODES>(l.x * ratio, l.y * ratio) | (encode2<CODES>(m.x * ratio, m.y * ratio) << 16);
            }
            held[u] = make_uint2(o[0], o[1]);
        }
    }
}

// Workgroups 0 .. items - 1 write blocks; those behind rotate queries.
template <int TYPE, int CODES, bool ROTATE, bool INTERLEAVED, int UPT, int HPT>
__global__ void __launch_bounds__(256) write_kernel(const WriteArgs a, const RotaryArgs q, int items) {
    if ((int)blockIdx.x < items)
        write_block<TYPE, CODES, ROTATE, INTERLEAVED, UPT>(a, blockIdx.x);
    else if constexpr (ROTATE)
        rotary_units<TYPE, INTERLEAVED, HPT, true>(q, (int64_t)((int)blockIdx.x - items) * blockDim.x + threadIdx.x);
}

// ---------------------------------------------------------------------------
// Reading back: a thread turns 8 codes into 8 values; four vectors in flight.
// Bound: memory (1 byte read, 2 or 4 written per value).
// ---------------------------------------------------------------------------
constexpr int kReadVectors = 4;

template <int CODES, int OUT>
__global__ void __launch_bounds__(256)
read_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, void* __restrict__ out, int64_t cb,
            int64_t ch, int64_t sb, int64_t sh, int kv_heads, int64_t units, int dim, int block_log, int chunks) {
    const int bh = blockIdx.x / chunks;
    const int64_t first = (int64_t)(blockIdx.x - bh * chunks) * (256 * kReadVectors) + threadIdx.x;
    const int b = bh / kv_heads, h = bh - b * kv_heads;
    const uint2* src = reinterpret_cast<const uint2*>(codes + b * cb + h * ch);
    const float* sc = scales + b * sb + h * sh;
    uint2 raw[kReadVectors];
    float scale[kReadVectors];
#pragma unroll
    for (int i = 0; i < kReadVectors; ++i) {
        const int64_t u = min(first + 256 * i, units - 1);
        raw[i] = src[u];
        scale[i] = sc[(u / (dim >> 3)) >> block_log];
    }
#pragma unroll
    for (int i = 0; i < kReadVectors; ++i) {
        const int64_t u = first + 256 * i;
        if (u >= units) break;
        float x[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t word = e ? raw[i].y : raw[i].x;
            const f32x2 l = decode2_f32<CODES, false>(word), m = decode2_f32<CODES, true>(word);
            x[4 * e] = l.x * scale[i];
            x[4 * e + 1] = l.y * scale[i];
            x[4 * e + 2] = m.x * scale[i];
            x[4 * e + 3] = m.y * scale[i];
        }
        const int64_t at = (int64_t)bh * units + u;
        if constexpr (OUT == W4A16_FP32) {
            f32x4* o = static_cast<f32x4*>(out) + 2 * at;
            o[0] = (f32x4){x[0], x[1], x[2], x[3]};
            o[1] = (f32x4){x[4], x[5], x[6], x[7]};
        } else {
            if constexpr (OUT == W4A16_FP16) {   // bf16 holds every code * scale's magnitude
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = __builtin_fabsf(x[e]) > 65504.0f ? __builtin_copysignf(65504.0f, x[e]) : x[e];
            }
            static_cast<u32x4*>(out)[at] = narrow8<OUT>(x);
        }
    }
}

}  // namespace w4a16

namespace {

using namespace w4a16;
using w4a16_internal::kv_fail;
using w4a16_internal::launch_fits;

int finish() {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return kv_fail(W4A16_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(e));
    return W4A16_OK;
}

int check_rows(const w4a16_kv_rows* x, const char* name) {
    if (x == nullptr || x->data == nullptr) return kv_fail(W4A16_ERR_NULL, std::string(name) + " must be non-NULL");
    if ((reinterpret_cast<uintptr_t>(x->data) & 1u) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, std::string(name) + " must be 2-byte aligned");
    return W4A16_OK;
}

bool aligned16(const w4a16_kv_rows& x) {
    return (reinterpret_cast<uintptr_t>(x.data) & 15u) == 0 &&
           ((x.batch_stride | x.token_stride | x.head_stride) & 7) == 0;
}

// Heads a thread takes: four where that still leaves the chip full (4022 tokens
// of 32 heads of 128, interleaved: 12.5 us at four, 16.0 at one; 700 tokens of 32
// heads of 64: 5.0 and 4.6).
int heads_per_thread(int64_t batch, int64_t tokens, int64_t heads, int64_t dim) {
    return heads >= 4 && batch * tokens * heads * (dim / 16) >= 384 * 1024 ? 4 : 1;
}

template <int TYPE, int HPT>
void launch_rotary(const RotaryArgs& a, bool interleaved, int64_t grid, hipStream_t st) {
    if (interleaved)
        hipLaunchKernelGGL((rotary_kernel<TYPE, true, HPT>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((rotary_kernel<TYPE, false, HPT>), dim3((unsigned)grid), dim3(256), 0, st, a);
}

template <int TYPE>
void launch_rotary_any(const RotaryArgs& a, bool interleaved, int64_t grid, hipStream_t st) {
    if (interleaved)
        hipLaunchKernelGGL((rotary_any_kernel<TYPE, true>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((rotary_any_kernel<TYPE, false>), dim3((unsigned)grid), dim3(256), 0, st, a);
}

template <int TYPE, int CODES, bool ROTATE, bool INTERLEAVED, int HPT>
void launch_write_units(int upt, const WriteArgs& a, const RotaryArgs& q, int items, int64_t grid, int threads,
                        hipStream_t st) {
#define WRITE_UNITS(U)                                                                                        \
    hipLaunchKernelGGL((write_kernel<TYPE, CODES, ROTATE, INTERLEAVED, U, HPT>), dim3((unsigned)grid),        \
                       dim3((unsigned)threads), 0, st, a, q, items)
    if (upt <= 1)
        WRITE_UNITS(1);
    else if (upt <= 2)
        WRITE_UNITS(2);
    else if (upt <= 4)
        WRITE_UNITS(4);
    else
        WRITE_UNITS(8);
#undef WRITE_UNITS
}

template <int TYPE, int CODES>
void launch_write(bool rotate, bool interleaved, int hpt, int upt, const WriteArgs& a, const RotaryArgs& q, int items,
                  int64_t grid, int threads, hipStream_t st) {
    if (!rotate)
        launch_write_units<TYPE, CODES, false, false, 1>(upt, a, q, items, grid, threads, st);
    else if (interleaved && hpt == 1)
        launch_write_units<TYPE, CODES, true, true, 1>(upt, a, q, items, grid, threads, st);
    else if (interleaved)
        launch_write_units<TYPE, CODES, true, true, 4>(upt, a, q, items, grid, threads, st);
    else if (hpt == 1)
        launch_write_units<TYPE, CODES, true, false, 1>(upt, a, q, items, grid, threads, st);
    else
        launch_write_units<TYPE, CODES, true, false, 4>(upt, a, q, items, grid, threads, st);
}

// Memory that a write call changes: rows of `row` bytes, n[0] groups of n[1]
// of them, step[0] and step[1] bytes apart, ascending from `base`.
struct Region {
    __int128 base, row, step[2];
    int64_t n[2];
};

Region region_of(const void* data, int64_t row, int64_t batch, int64_t batch_stride, int64_t heads, int64_t head_stride,
                 int64_t size) {
    Region r{(__int128)reinterpret_cast<uintptr_t>(data), (__int128)row * size,
             {(__int128)batch_stride * size, (__int128)head_stride * size}, {batch, heads}};
    for (int i = 0; i < 2; ++i) {
        if (r.n[i] == 1) r.step[i] = 0;
        if (r.step[i] < 0) {
            r.base += r.step[i] * (r.n[i] - 1);
            r.step[i] = -r.step[i];
        }
    }
    if (r.n[0] == 1 || (r.n[1] > 1 && r.step[0] < r.step[1])) {
        std::swap(r.step[0], r.step[1]);
        std::swap(r.n[0], r.n[1]);
    }
    return r;
}

__int128 extent(const Region& r) { return r.step[0] * (r.n[0] - 1) + r.step[1] * (r.n[1] - 1) + r.row; }

// Whether no two of its rows share memory.
bool disjoint(const Region& r) {
    return (r.n[1] == 1 || r.step[1] >= r.row) && (r.n[0] == 1 || r.step[0] >= r.step[1] * (r.n[1] - 1) + r.row);
}

// Whether a row of one shares memory with a row of the other, both disjoint in
// themselves: for each row of `a` the last row of `b` that starts at or before
// it, and the first that starts behind it.
bool meet(const Region& a, const Region& b) {
    if (a.base + extent(a) <= b.base || b.base + extent(b) <= a.base) return false;
    for (int64_t i = 0; i < a.n[0]; ++i)
        for (int64_t j = 0; j < a.n[1]; ++j) {
            const __int128 x = a.base + a.step[0] * i + a.step[1] * j;
            if (x < b.base) {
                if (x + a.row > b.base) return true;
                continue;
            }
            const __int128 g = b.n[0] == 1 ? 0 : std::min<__int128>((x - b.base) / b.step[0], b.n[0] - 1);
            const __int128 group = b.base + g * b.step[0];
            const __int128 k = b.n[1] == 1 ? 0 : std::min<__int128>((x - group) / b.step[1], b.n[1] - 1);
            const __int128 before = group + k * b.step[1];
            if (before + b.row > x) return true;
            if (k + 1 < b.n[1] ? before + b.step[1] < x + a.row : g + 1 < b.n[0] && group + b.step[0] < x + a.row) return true;
        }
    return false;
}

// The memory of a cache's codes and scales: keys' and values' codes, then their scales.
void regions_of(const w4a16_kv_cache& c, Region (&r)[4]) {
    const int64_t blocks = (c.slots + c.block - 1) / c.block;
    for (int i = 0; i < 2; ++i) {
        const w4a16_kv_codes& side = i ? c.v : c.k;
        r[i] = region_of(side.codes, c.slots * c.head_dim, c.batch, side.batch_stride, c.kv_heads, side.head_stride, 1);
        r[2 + i] = region_of(side.scales, blocks, c.batch, side.scale_batch_stride, c.kv_heads, side.scale_head_stride, 4);
    }
}

}  // namespace

namespace w4a16_internal {

// Workgroups write their own block each: blocks that share memory would race.
int check_written(const w4a16_kv_cache& c) {
    Region r[4];
    regions_of(c, r);
    for (int i = 0; i < 4; ++i)
        if (!disjoint(r[i]))
            return kv_fail(W4A16_ERR_CONFIG, "codes and scales that are written must not overlap themselves");
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < 4; ++j)
            if (meet(r[i], r[j]))
                return kv_fail(W4A16_ERR_CONFIG, "keys and values, codes and scales must not share memory");
    return W4A16_OK;
}

int check_apart(const w4a16_kv_cache& read, const w4a16_kv_cache& written) {
    Region r[4], w[4];
    regions_of(read, r);
    regions_of(written, w);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (meet(r[i], w[j])) return kv_fail(W4A16_ERR_CONFIG, "the two caches must not share memory");
    return W4A16_OK;
}

}  // namespace w4a16_internal

namespace {

using w4a16_internal::check_written;

// Keys and values into the cache, and (q != NULL) the rotation of q and k.
int write_tokens(const w4a16_kv_rows* q, void* q_out, int64_t heads, const w4a16_kv_rows* k, const w4a16_kv_rows* v,
                 int64_t tokens, const float* cos_table, const float* sin_table, int64_t table_rows, int64_t rot,
                 int interleaved, const w4a16_kv_cache* cache, const int64_t* start, const int64_t* counts, int type,
                 void* stream) {
    int rc = w4a16_internal::check_kv_cache(cache);
    if (rc != W4A16_OK) return rc;
    if (type != W4A16_FP16 && type != W4A16_BF16) return kv_fail(W4A16_ERR_CONFIG, "tokens must be fp16 or bf16");
    if (tokens < 0 || heads < 0) return kv_fail(W4A16_ERR_SHAPE, "tokens and heads must be non-negative");
    if (tokens > (1 << 24) || heads > (1 << 16)) return kv_fail(W4A16_ERR_TOO_LARGE, "too many tokens or heads");
    if (q != nullptr) {
        if (rot < 16 || rot > cache->head_dim || rot % 16 != 0)
            return kv_fail(W4A16_ERR_SHAPE, "the rotated part must be a multiple of 16 of at most head_dim dims");
        if (table_rows < cache->slots)
            return kv_fail(W4A16_ERR_SHAPE, "the rotary tables must have a row for every slot");
    }
    if (cache->batch == 0 || tokens == 0) return W4A16_OK;
    if ((rc = check_rows(k, "k")) != W4A16_OK || (rc = check_rows(v, "v")) != W4A16_OK) return rc;
    if (start == nullptr) return kv_fail(W4A16_ERR_NULL, "start must be non-NULL");
    const int64_t block = cache->block;
    const int64_t blocks = (tokens + block - 2) / block + 1;   // most that a sequence's tokens touch
    const int64_t items = 2 * cache->kv_heads * cache->batch * blocks;
    // a workgroup's rows: at most a block's; one wavefront while they fit its lanes
    const int64_t units = (tokens < block ? tokens : block) * cache->head_dim / 16;
    const int threads = units <= 64 ? 64 : units <= 128 ? 128 : 256;
    const int upt = (int)((units + threads - 1) / threads);
    const int hpt = q == nullptr || heads == 0 ? 1 : heads_per_thread(cache->batch, tokens, heads, cache->head_dim);
    const int64_t head_groups = (heads + hpt - 1) / hpt;
    const __int128 work = q == nullptr ? 0 : (__int128)cache->batch * tokens * head_groups * (cache->head_dim / 16);
    const __int128 extra = (work + threads - 1) / threads;
    if (!launch_fits(items + extra, threads)) return kv_fail(W4A16_ERR_TOO_LARGE, "too many rows for one launch");
    if ((rc = check_written(*cache)) != W4A16_OK) return rc;
    if (q != nullptr) {
        if ((rc = check_rows(q, "q")) != W4A16_OK) return rc;
        if (q_out == nullptr || cos_table == nullptr || sin_table == nullptr)
            return kv_fail(W4A16_ERR_NULL, "the output and the rotary tables must be non-NULL");
        if (!aligned16(*q) || (reinterpret_cast<uintptr_t>(q_out) & 15u) != 0)
            return kv_fail(W4A16_ERR_ALIGNMENT, "q and its output must be 16-byte aligned with strides multiples of 8");
    }
    WriteArgs a{};
    const w4a16_kv_rows* rows[2] = {k, v};
    const w4a16_kv_codes* sides[2] = {&cache->k, &cache->v};
    for (int i = 0; i < 2; ++i) {
        const w4a16_kv_codes& c = *sides[i];
        a.side[i] = {static_cast<const uint16_t*>(rows[i]->data), static_cast<uint8_t*>(c.codes), c.scales,
                     rows[i]->batch_stride, rows[i]->token_stride, rows[i]->head_stride,
                     c.batch_stride, c.head_stride, c.scale_batch_stride, c.scale_head_stride, aligned16(*rows[i])};
    }
    a.start = start;
    a.counts = counts;
    a.cos_table = cos_table;
    a.sin_table = sin_table;
    a.slots = cache->slots;
    a.tokens = (int)tokens;
    a.kv_heads = (int)cache->kv_heads;
    a.batch = (int)cache->batch;
    a.dim = (int)cache->head_dim;
    a.block = (int)cache->block;
    a.rot = (int)rot;
    RotaryArgs r{};
    if (q != nullptr && heads > 0)
        r = RotaryArgs{static_cast<const uint16_t*>(q->data), static_cast<uint16_t*>(q_out), cos_table, sin_table,
                       nullptr, start, counts, q->batch_stride, q->token_stride, q->head_stride, 0, 0, table_rows,
                       cache->slots, (int)cache->batch, (int)tokens, (int)heads, (int)cache->head_dim, (int)rot,
                       (int)head_groups};
    const int64_t grid = items + (int64_t)extra;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool inter = interleaved != 0;
    if (type == W4A16_FP16 && cache->code_type == W4A16_KV_INT8)
        launch_write<W4A16_FP16, W4A16_KV_INT8>(q != nullptr, inter, hpt, upt, a, r, (int)items, grid, threads, st);
    else if (type == W4A16_FP16)
        launch_write<W4A16_FP16, W4A16_KV_FP8>(q != nullptr, inter, hpt, upt, a, r, (int)items, grid, threads, st);
    else if (cache->code_type == W4A16_KV_INT8)
        launch_write<W4A16_BF16, W4A16_KV_INT8>(q != nullptr, inter, hpt, upt, a, r, (int)items, grid, threads, st);
    else
        launch_write<W4A16_BF16, W4A16_KV_FP8>(q != nullptr, inter, hpt, upt, a, r, (int)items, grid, threads, st);
    return finish();
}

template <int CODES>
void launch_read(int out_type, int64_t grid, const w4a16_kv_codes& c, void* out, int64_t kv_heads, int64_t units,
                 int64_t dim, int block_log, int64_t chunks, hipStream_t st) {
#define READ(OUT)                                                                                               \
    hipLaunchKernelGGL((read_kernel<CODES, OUT>), dim3((unsigned)grid), dim3(256), 0, st,                       \
                       static_cast<const uint8_t*>(c.codes), c.scales, out, c.batch_stride, c.head_stride,      \
                       c.scale_batch_stride, c.scale_head_stride, (int)kv_heads, units, (int)dim, block_log,    \
                       (int)chunks)
    if (out_type == W4A16_FP16)
        READ(W4A16_FP16);
    else if (out_type == W4A16_BF16)
        READ(W4A16_BF16);
    else
        READ(W4A16_FP32);
#undef READ
}

}  // namespace

namespace w4a16_internal {

int kv_fail(int code, const std::string& message) {
    set_last_error(message);
    return code;
}

static int check_side(const w4a16_kv_codes& c, const char* name) {
    if (c.codes == nullptr || c.scales == nullptr)
        return kv_fail(W4A16_ERR_NULL, std::string(name) + " codes and scales must be non-NULL");
    if ((reinterpret_cast<uintptr_t>(c.codes) & 15u) != 0 || ((c.batch_stride | c.head_stride) & 15) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, std::string(name) + " codes must start on 16 bytes in every head");
    if ((reinterpret_cast<uintptr_t>(c.scales) & 3u) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, std::string(name) + " scales must be 4-byte aligned");
    return W4A16_OK;
}

int check_kv_block(int64_t block, int code_type) {
    if (block != 16 && block != 32 && block != 64 && block != 128)
        return kv_fail(W4A16_ERR_GROUP_SIZE, "a scale's block must be 16, 32, 64 or 128 slots");
    if (code_type != W4A16_KV_INT8 && code_type != W4A16_KV_FP8)
        return kv_fail(W4A16_ERR_CONFIG, "codes must be int8 or e4m3");
    return W4A16_OK;
}

int check_kv_cache(const w4a16_kv_cache* cache) {
    if (cache == nullptr) return kv_fail(W4A16_ERR_NULL, "cache must be non-NULL");
    int rc = check_kv_block(cache->block, cache->code_type);
    if (rc != W4A16_OK) return rc;
    if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256)
        return kv_fail(W4A16_ERR_SHAPE, "the cache's head_dim must be 64, 128 or 256");
    if (cache->batch < 0 || cache->kv_heads < 1 || cache->slots < 1)
        return kv_fail(W4A16_ERR_SHAPE, "the cache must have at least one KV head and one slot");
    if (cache->batch > (1 << 24) || cache->kv_heads > (1 << 16) || cache->slots > (1 << 30))
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many sequences, KV heads or slots");
    if (cache->batch == 0) return W4A16_OK;
    if ((rc = check_side(cache->k, "key")) != W4A16_OK) return rc;
    return check_side(cache->v, "value");
}

}  // namespace w4a16_internal

extern "C" {

int w4a16_rotary(const w4a16_kv_rows* x, void* out, int64_t batch, int64_t tokens, int64_t heads, int64_t head_dim,
                 const float* cos_table, const float* sin_table, int64_t table_rows, int64_t rot,
                 const int64_t* positions, int64_t pos_batch_stride, int64_t pos_token_stride, int interleaved,
                 int type, void* stream) {
    if (type != W4A16_FP16 && type != W4A16_BF16) return kv_fail(W4A16_ERR_CONFIG, "rows must be fp16 or bf16");
    if (batch < 0 || tokens < 0 || heads < 0 || head_dim < 1 || table_rows < 0)
        return kv_fail(W4A16_ERR_SHAPE, "sizes must be non-negative");
    if (rot < 2 || rot % 2 != 0 || rot > head_dim)
        return kv_fail(W4A16_ERR_SHAPE, "the rotated part must be an even number of at most head_dim dims");
    if (batch > INT32_MAX || tokens > INT32_MAX || heads > (1 << 24) || head_dim > (1 << 16))
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many rows");
    if (batch == 0 || tokens == 0 || heads == 0) return W4A16_OK;
    int rc = check_rows(x, "x");
    if (rc != W4A16_OK) return rc;
    if (out == nullptr || positions == nullptr || cos_table == nullptr || sin_table == nullptr)
        return kv_fail(W4A16_ERR_NULL, "out, positions and the rotary tables must be non-NULL");
    if ((reinterpret_cast<uintptr_t>(out) & 1u) != 0) return kv_fail(W4A16_ERR_ALIGNMENT, "out must be 2-byte aligned");
    RotaryArgs a{static_cast<const uint16_t*>(x->data), static_cast<uint16_t*>(out), cos_table, sin_table, positions,
                 nullptr, nullptr, x->batch_stride, x->token_stride, x->head_stride, pos_batch_stride,
                 pos_token_stride, table_rows, 0, (int)batch, (int)tokens, (int)heads, (int)head_dim, (int)rot, 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    // table_rows 0: every position lies outside, and no row may be read
    const bool vec = head_dim % 16 == 0 && rot % 16 == 0 && aligned16(*x) && table_rows > 0 &&
                     (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
    if (vec) {
        const int hpt = heads_per_thread(batch, tokens, heads, head_dim);
        a.head_groups = (int)((heads + hpt - 1) / hpt);
        const __int128 work = (__int128)batch * tokens * a.head_groups * (head_dim / 16);
        if (!launch_fits((work + 255) / 256, 256)) return kv_fail(W4A16_ERR_TOO_LARGE, "too many rows for one launch");
        const int64_t grid = ((int64_t)work + 255) / 256;
        if (type == W4A16_FP16 && hpt == 4)
            launch_rotary<W4A16_FP16, 4>(a, interleaved != 0, grid, st);
        else if (type == W4A16_FP16)
            launch_rotary<W4A16_FP16, 1>(a, interleaved != 0, grid, st);
        else if (hpt == 4)
            launch_rotary<W4A16_BF16, 4>(a, interleaved != 0, grid, st);
        else
            launch_rotary<W4A16_BF16, 1>(a, interleaved != 0, grid, st);
    } else {
        const __int128 work = (__int128)batch * tokens * heads * (head_dim - rot / 2);
        if (!launch_fits((work + 255) / 256, 256)) return kv_fail(W4A16_ERR_TOO_LARGE, "too many rows for one launch");
        const int64_t grid = ((int64_t)work + 255) / 256;
        if (type == W4A16_FP16)
            launch_rotary_any<W4A16_FP16>(a, interleaved != 0, grid, st);
        else
            launch_rotary_any<W4A16_BF16>(a, interleaved != 0, grid, st);
    }
    return finish();
}

int w4a16_kv_write(const w4a16_kv_rows* k, const w4a16_kv_rows* v, int64_t tokens, const w4a16_kv_cache* cache,
                   const int64_t* start, const int64_t* counts, int type, void* stream) {
    return write_tokens(nullptr, nullptr, 0, k, v, tokens, nullptr, nullptr, 0, 0, 0, cache, start, counts, type,
                        stream);
}

int w4a16_rotary_kv_write(const w4a16_kv_rows* q, void* q_out, int64_t heads, const w4a16_kv_rows* k,
                          const w4a16_kv_rows* v, int64_t tokens, const float* cos_table, const float* sin_table,
                          int64_t table_rows, int64_t rot, int interleaved, const w4a16_kv_cache* cache,
                          const int64_t* start, const int64_t* counts, int type, void* stream) {
    if (q == nullptr) return kv_fail(W4A16_ERR_NULL, "q must be non-NULL");
    return write_tokens(q, q_out, heads, k, v, tokens, cos_table, sin_table, table_rows, rot, interleaved, cache,
                        start, counts, type, stream);
}

int w4a16_kv_read(const w4a16_kv_codes* side, void* out, int64_t batch, int64_t kv_heads, int64_t slots,
                  int64_t head_dim, int64_t block, int code_type, int out_type, void* stream) {
    int rc = w4a16_internal::check_kv_block(block, code_type);
    if (rc != W4A16_OK) return rc;
    if (out_type != W4A16_FP16 && out_type != W4A16_BF16 && out_type != W4A16_FP32)
        return kv_fail(W4A16_ERR_CONFIG, "values must be fp16, bf16 or fp32");
    if (batch < 0 || kv_heads < 0 || slots < 0 || head_dim < 16 || head_dim % 16 != 0)
        return kv_fail(W4A16_ERR_SHAPE, "head_dim must be a multiple of 16 and the other sizes non-negative");
    if (batch > (1 << 24) || kv_heads > (1 << 16) || slots > (1 << 30) || head_dim > (1 << 16))
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many sequences, KV heads, slots or dims");
    if (batch == 0 || kv_heads == 0 || slots == 0) return W4A16_OK;
    if (side == nullptr || out == nullptr) return kv_fail(W4A16_ERR_NULL, "codes and out must be non-NULL");
    if ((rc = w4a16_internal::check_side(*side, "the")) != W4A16_OK) return rc;
    if ((reinterpret_cast<uintptr_t>(out) & 15u) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, "out must be 16-byte aligned");
    const int64_t units = slots * (head_dim / 8);
    const int64_t chunks = (units + 256 * kReadVectors - 1) / (256 * kReadVectors);
    if (!launch_fits((__int128)chunks * batch * kv_heads, 256))
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many values for one launch");
    const int64_t grid = chunks * batch * kv_heads;
    const int block_log = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (code_type == W4A16_KV_INT8)
        launch_read<W4A16_KV_INT8>(out_type, grid, *side, out, kv_heads, units, head_dim, block_log, chunks, st);
    else
        launch_read<W4A16_KV_FP8>(out_type, grid, *side, out, kv_heads, units, head_dim, block_log, chunks, st);
    return finish();
}

}  // extern "C"
