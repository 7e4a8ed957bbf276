// Device-side building blocks of the 8-bit key/value cache: its codes (int8
// and OCP e4m3), its power-of-two scales, and vectors of token rows.
#pragma once

#include "w4a16_attn_device.h"
#include "w4a16_kv.h"

namespace w4a16 {

constexpr int kKvLowest = -40, kKvHighest = 40;   // exponents of the scales

__device__ __forceinline__ float exp2_int(int e) {   // 2^e, -126 <= e <= 127
    return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ int exponent_of(float scale) {   // of a power of two
    return (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255u) - 127;
}

// The smallest e in [kKvLowest, kKvHighest] with amax <= M 2^e; M = 127 is
// 1.984375 2^6 and 448 is 1.75 2^8, so the mantissa decides by one step.
template <int CODES>
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
    constexpr uint32_t top = CODES == W4A16_KV_INT8 ? 0x7E0000u : 0x600000u;
    constexpr int shift = CODES == W4A16_KV_INT8 ? 6 : 8;
    const int e = (int)(bits >> 23) - 127 - shift + ((bits & 0x7FFFFFu) > top ? 1 : 0);
    return min(max(e, kKvLowest), kKvHighest);
}

// Two scaled values -> codes in the low 16 bits, half to even, saturated.
template <int CODES>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
    if constexpr (CODES == W4A16_KV_INT8) {
        const int x = (int)__builtin_fminf(__builtin_fmaxf(__builtin_rintf(a), -127.0f), 127.0f);
        const int y = (int)__builtin_fminf(__builtin_fmaxf(__builtin_rintf(b), -127.0f), 127.0f);
        return ((uint32_t)x & 0xFFu) | (((uint32_t)y & 0xFFu) << 8);
    } else {
        a = __builtin_fminf(__builtin_fmaxf(a, -448.0f), 448.0f);
        b = __builtin_fminf(__builtin_fmaxf(b, -448.0f), 448.0f);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xFFFFu;
    }
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Codes 2 HI and 2 HI + 1 of a word as fp32 values.
template <int CODES, bool HI>
__device__ __forceinline__ f32x2 decode2_f32(uint32_t w) {
    if constexpr (CODES == W4A16_KV_INT8) {
        const int s = HI ? 16 : 0;
        return (f32x2){(float)(int8_t)(w >> s), (float)(int8_t)(w >> (s + 8))};
    } else {
        return __builtin_amdgcn_cvt_pk_f32_fp8(w, HI);
    }
}

// Codes 2 HI and 2 HI + 1 of a word as fp16, exact: e4m3 by one conversion;
// int8 as 1152 + s through the mantissa of 1024 (s + 128 in [0, 255]). The
// caller has flipped the sign bits of int8 words (kv_bias).
template <int CODES>
__device__ __forceinline__ uint32_t kv_bias(uint32_t w) {
    return CODES == W4A16_KV_INT8 ? w ^ 0x80808080u : w;
}
template <int CODES, bool HI>
__device__ __forceinline__ f16x2 decode2_f16(uint32_t biased) {
    if constexpr (CODES == W4A16_KV_INT8) {
        const f16x2 offset = {(f16)-1152.0f, (f16)-1152.0f};
        return as_f16x2(perm(0x64646464u, biased, HI ? 0x04030402u : 0x04010400u)) + offset;
    } else {
        return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(biased, 1.0f, HI));
    }
}

// 16-bit floats of token rows and outputs. TYPE is W4A16_FP16 or W4A16_BF16.
template <int TYPE>
__device__ __forceinline__ float widen16(uint32_t h) {   // the low 16 bits
    if constexpr (TYPE == W4A16_FP16)
        return (float)__builtin_bit_cast(f16, (uint16_t)h);
    else
        return __builtin_bit_cast(float, h << 16);
}
template <int TYPE>
__device__ __forceinline__ uint32_t narrow16(float v) {   // rounded half to even
    if constexpr (TYPE == W4A16_FP16)
        return __builtin_bit_cast(uint16_t, (f16)v);
    else
        return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// 8 consecutive 16-bit values; vec: p is 16-byte aligned.
__device__ __forceinline__ u32x4 load8(const uint16_t* p, bool vec) {
    if (vec) return *reinterpret_cast<const u32x4*>(p);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return r;
}
template <int TYPE>
__device__ __forceinline__ void widen8(u32x4 v, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = widen16<TYPE>(v[i] & 0xFFFFu);
        x[2 * i + 1] = widen16<TYPE>(v[i] >> 16);
    }
}
template <int TYPE>
__device__ __forceinline__ u32x4 narrow8(const float (&x)[8]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = narrow16<TYPE>(x[2 * i]) | (narrow16<TYPE>(x[2 * i + 1]) << 16);
    return v;
}

// One rotated pair. No contraction: products and sums round to fp32 one by
// one, as separate torch operations do, so that codes of rotated keys agree.
__device__ __forceinline__ void rotate_pair(float& x1, float& x2, float c, float s) {
#pragma clang fp contract(off)
    const float a = x1 * c, b = x2 * s, d = x2 * c, e = x1 * s;
    x1 = a - b;
    x2 = d + e;
}

}  // namespace w4a16
