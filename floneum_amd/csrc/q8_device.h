// Device side of the 8-bit formats: nearest codes, and codes as 16-bit floats.
#pragma once
#include "device_utils.h"

namespace fhip {

constexpr float Q8_LEAST_SCALE = 0x1p-100f;

template <int FMT>
struct Q8Format;

// x / s to the nearest whole number, ties to even, for |x| <= 127 s (and what the scale's own rounding adds).  The product with the reciprocal is at most one off; what it leaves is
// exact (a multiple of half of s's last place, not above s) and says so.
template <>
struct Q8Format<FHIP_Q8_INT8> {
    static constexpr float LARGEST = 127.0f;
    static __device__ __forceinline__ uint32_t code(float x, float s, float inv) {
        float c = __builtin_rintf(x * inv);
        const float r = __builtin_fmaf(-c, s, x), h = 0.5f * s;
        const float away = __builtin_copysignf(1.0f, r);
        const bool odd = ((int)c & 1) != 0;
        if (__builtin_fabsf(r) > h || (__builtin_fabsf(r) == h && odd)) c += away;
        return (uint32_t)(int)c & 0xffu;
    }
    static __device__ __forceinline__ float value(uint32_t word, int byte) { return (float)((int)(word << (24 - 8 * byte)) >> 24); }
};

// The quotient is rounded to odd first (to the neighbour whose last bit is 1 where it is not an f32), from which the
// hardware's rounding to e4m3 is the rounding of the exact quotient: f32 has more than two bits beyond it.
template <>
struct Q8Format<FHIP_Q8_E4M3> {
    static constexpr float LARGEST = 448.0f;
    static __device__ __forceinline__ float quotient(float x, float s, float inv) {
        float y = x * inv;
        y = __builtin_fmaf(__builtin_fmaf(-y, s, x), inv, y);
        const float r = __builtin_fmaf(-y, s, x);
        uint32_t bits = __float_as_uint(y);
        if (r != 0.0f && (bits & 1u) == 0 && y != 0.0f) bits += (r > 0.0f) == (y > 0.0f) ? 1u : ~0u;
        return __uint_as_float(bits);
    }
    static __device__ __forceinline__ uint32_t code(float x, float s, float inv) {
        const float y = quotient(x, s, inv);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xffu;
    }
    static __device__ __forceinline__ float value(uint32_t word, int byte) {
        switch (byte) {
            case 0: return __builtin_amdgcn_cvt_f32_fp8((int)word, 0);
            case 1: return __builtin_amdgcn_cvt_f32_fp8((int)word, 1);
            case 2: return __builtin_amdgcn_cvt_f32_fp8((int)word, 2);
            default: return __builtin_amdgcn_cvt_f32_fp8((int)word, 3);
        }
    }
};

// Codes as half pairs, exactly.  INT8: a byte c, its sign bit turned and 0x64 put above it, is the half 1024 + 128 + c.
template <int FMT>
__device__ __forceinline__ half2_t q8_pair_low(uint32_t w);   // bytes 0 and 1 of w
template <int FMT>
__device__ __forceinline__ half2_t q8_pair_high(uint32_t w);  // bytes 2 and 3
__device__ __forceinline__ half2_t q8_unbias(uint32_t h) {
    const half2_t bias = {(half_t)1152.0f, (half_t)1152.0f};
    return __builtin_bit_cast(half2_t, h) - bias;
}
template <>
__device__ __forceinline__ half2_t q8_pair_low<FHIP_Q8_INT8>(uint32_t w) {
    return q8_unbias(__builtin_amdgcn_perm(w ^ 0x80808080u, 0x64646464u, 0x00050004u));
}
template <>
__device__ __forceinline__ half2_t q8_pair_high<FHIP_Q8_INT8>(uint32_t w) {
    return q8_unbias(__builtin_amdgcn_perm(w ^ 0x80808080u, 0x64646464u, 0x00070006u));
}
template <>
__device__ __forceinline__ half2_t q8_pair_low<FHIP_Q8_E4M3>(uint32_t w) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}
template <>
__device__ __forceinline__ half2_t q8_pair_high<FHIP_Q8_E4M3>(uint32_t w) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
}

}  // namespace fhip
