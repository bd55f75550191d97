// Device code that the attention kernels of the 8-bit cache share.
#pragma once
#include "q8.h"
#include "q8_device.h"

namespace fhip {

constexpr float Q8_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float xor16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 16) ? r[0] : r[1]);
}
__device__ __forceinline__ float xor32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float q8_load_any(const void *p, int64_t idx, int dtype) {
    if (dtype == FHIP_F32) return ((const float *)p)[idx];
    if (dtype == FHIP_F16) return (float)((const half_t *)p)[idx];
    return to_float(((const bf16_t *)p)[idx]);
}
__device__ __forceinline__ void q8_store_any(void *p, int64_t idx, int dtype, float v) {
    if (dtype == FHIP_F32) ((float *)p)[idx] = v;
    else if (dtype == FHIP_F16) ((half_t *)p)[idx] = (half_t)v;
    else ((bf16_t *)p)[idx] = from_float<bf16_t>(v);
}
// four consecutive dims of an output row
__device__ __forceinline__ void q8_store4_any(const Q8AttnParams &p, int64_t idx, float4_t v) {
    if (!p.out_vec) {
#pragma unroll
        for (int e = 0; e < 4; e++) q8_store_any(p.out, idx + e * p.os[3], p.out_dtype, v[e]);
    } else if (p.out_dtype == FHIP_F32) {
        *(float4_t *)((float *)p.out + idx) = v;
    } else {
        uint16_t bits[4];
#pragma unroll
        for (int e = 0; e < 4; e++) bits[e] = p.out_dtype == FHIP_F16 ? __builtin_bit_cast(uint16_t, (half_t)v[e]) : from_float<bf16_t>(v[e]).bits;
        *(uint2_t *)((uint16_t *)p.out + idx) = uint2_t{bits[0] | (uint32_t)bits[1] << 16, bits[2] | (uint32_t)bits[3] << 16};
    }
}

// Score and additive mask (both times log2 e).  A finite mask value hides nothing: what overflows in the log2 domain (the type's lowest value) counts as
// the least f32, and a row whose keys are all that far down weighs them alike, as f32 scores that vanish beside the mask do.
__device__ __forceinline__ float q8_with_mask(float s, float add) {
    const float t = s + add;
    return t < -3.402823466e38f ? -3.402823466e38f : t;
}

// The keys [lo, hi) that some row of row0 .. row1 sees, from the analytic mask and the lengths.
struct Q8Range {
    int lo, hi;
    int64_t pos0;  // position of query row 0
};
__device__ __forceinline__ Q8Range q8_visible(const Q8AttnParams &p, int b, int row0, int row1) {
    int64_t lo = 0, hi = p.Skv, pos0 = p.q_pos_offset + (p.q_positions ? p.q_positions[b] : 0);
    if (p.kv_lens) hi = min(hi, (int64_t)p.kv_lens[b]);
    if (p.causal) hi = min(hi, pos0 + row1 + 1);
    if (p.window > 0) lo = max(lo, pos0 + row0 - p.window + 1);
    hi = max(hi, (int64_t)0);
    Q8Range r;
    r.lo = (int)min(lo, hi), r.hi = (int)hi, r.pos0 = pos0;
    return r;
}

// Eight consecutive dims of a query row as they lie in memory: f32 (TERMS 2) or 16-bit ones.
template <int TERMS>
struct Q8Query8 {
    uint32_t w[4 * TERMS];
    // d0: the first of them; pieces beyond head_dim are read from the row's start
    __device__ __forceinline__ void load(const Q8AttnParams &p, int64_t base, int d0) {
        const int d = d0 < p.D ? d0 : 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if constexpr (TERMS == 2) {
                const uint4_t v = *(const uint4_t *)((const float *)p.q + base + d + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; e++) w[4 * i + e] = v[e];
            } else {
                const uint2_t v = *(const uint2_t *)((const uint16_t *)p.q + base + d + 4 * i);
                w[2 * i] = v[0], w[2 * i + 1] = v[1];
            }
        }
    }
    // the same of rows with any stride
    __device__ __forceinline__ void gather(const Q8AttnParams &p, int64_t base, int d0) {
        const int d = d0 < p.D ? d0 : 0;
        if constexpr (TERMS == 2) {
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = ((const uint32_t *)p.q)[base + (d + e) * p.qs[3]];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                w[e] = (uint32_t)((const uint16_t *)p.q)[base + (d + 2 * e) * p.qs[3]] |
                       (uint32_t)((const uint16_t *)p.q)[base + (d + 2 * e + 1) * p.qs[3]] << 16;
        }
    }
    // f16 queries as they are; a scale below 0 goes with them
    __device__ __forceinline__ half8_t halves(const Q8AttnParams &p, int d0) const {
        const uint32_t keep = d0 < p.D ? ~0u : 0u, turn = p.scale < 0.0f ? 0x80008000u : 0u;
        return __builtin_bit_cast(half8_t, uint4_t{(w[0] & keep) ^ turn, (w[1] & keep) ^ turn, (w[2] & keep) ^ turn, (w[3] & keep) ^ turn});
    }
    __device__ __forceinline__ void widen(const Q8AttnParams &p, int d0, float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (TERMS == 2) {
                x[e] = __uint_as_float(w[e]);
            } else {
                const uint32_t bits = e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
                x[e] = p.q_dtype == FHIP_F16 ? (float)__builtin_bit_cast(half_t, (uint16_t)bits) : __uint_as_float(bits << 16);
            }
            if (d0 >= p.D) x[e] = 0.0f;
        }
    }
};
// The power of two that brings a row's largest element to [2^14, 2^15); zeros, infinities and NaN stay as they are.
__device__ __forceinline__ int q8_query_shift(float top) { return top > 0.0f && top <= 3.402823466e38f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0; }
// An element as one term or two.  A scale of 0 or below goes with the queries: the one of the scores (q8_score_scale) is positive.
template <int TERMS>
__device__ __forceinline__ void q8_query_terms(const Q8AttnParams &p, float x, int shift, half_t &high, half_t &low) {
    const float v = __builtin_ldexpf(p.scale > 0.0f ? x : p.scale < 0.0f ? -x : 0.0f * x, shift);
    high = (half_t)v;
    if constexpr (TERMS == 2) low = (half_t)(v - (float)high);
}
// What takes a product of such a query with codes times their scale to the log2 domain, rounded once.  Never 0, which has no product with the
// -infinity of a hidden key, nor infinite, which has none with 0: a row that would need less than the least f32 has scores of next to nothing all the
// same.
__device__ __forceinline__ float q8_score_factor(const Q8AttnParams &p) { return p.scale != 0.0f ? __builtin_fabsf(p.scale) : 1.0f; }
__device__ __forceinline__ float q8_score_scale(const Q8AttnParams &p, int shift) {
    const float factor = q8_score_factor(p);
    const float g = __builtin_ldexpf(__builtin_amdgcn_frexp_mantf(factor) * Q8_LOG2E, __builtin_amdgcn_frexp_expf(factor) - shift);
    return fminf(fmaxf(g, 0x1p-149f), 3.402823466e38f);
}
// it is below 2 to this plus 1
__device__ __forceinline__ int q8_score_exponent(const Q8AttnParams &p, int shift) { return __builtin_amdgcn_frexp_expf(q8_score_factor(p)) - shift; }

}  // namespace fhip
