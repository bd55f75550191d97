// The 8-bit key / value cache: new rows coded as they are written (with the norm and the rotation in front of it), and rows read back.
// The wide cache's counterparts are in rope.hip and kv_cache.hip; the reference has neither (its cache holds the tensors' own type,
// fusor-ml/fusor/src/cache/kv_cache.rs:13-68).
#include <algorithm>

#include "q8.h"
#include "q8_device.h"

namespace fhip {

__device__ __forceinline__ float q8_load(const void *p, int64_t idx, int dtype) {
    if (dtype == FHIP_F32) return ((const float *)p)[idx];
    if (dtype == FHIP_F16) return (float)((const half_t *)p)[idx];
    return to_float(((const bf16_t *)p)[idx]);
}
__device__ __forceinline__ float4_t q8_load4(const void *p, int64_t idx, int dtype) {
    if (dtype == FHIP_F32) return *(const float4_t *)((const float *)p + idx);
    const uint2_t w = *(const uint2_t *)((const uint16_t *)p + idx);
    float4_t v;
    if (dtype == FHIP_F16) {
        const half2_t a = __builtin_bit_cast(half2_t, (uint32_t)w[0]), b = __builtin_bit_cast(half2_t, (uint32_t)w[1]);
        v = float4_t{(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
    } else {
        v = float4_t{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                     __uint_as_float(w[1] & 0xffff0000u)};
    }
    return v;
}
// rows of the rotation's tables, which begin at any f32
__device__ __forceinline__ float4_t q8_load_turn(const float *p) {
    typedef float float4_at4_t __attribute__((ext_vector_type(4), aligned(4)));
    const float4_at4_t v = *(const float4_at4_t *)p;
    return float4_t{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ float q8_round_through(float v, int dtype) {
    if (dtype == FHIP_F16) return (float)(half_t)v;
    if (dtype == FHIP_BF16) return to_float(from_float<bf16_t>(v));
    return v;
}
__device__ __forceinline__ void q8_store4(void *p, int64_t idx, int64_t stride, bool vec, int dtype, const float *v) {
    if (dtype == FHIP_F32) {
        if (vec) {
            *(float4_t *)((float *)p + idx) = float4_t{v[0], v[1], v[2], v[3]};
            return;
        }
        for (int e = 0; e < 4; e++) ((float *)p)[idx + e * stride] = v[e];
        return;
    }
    uint16_t bits[4];
    for (int e = 0; e < 4; e++)
        bits[e] = dtype == FHIP_F16 ? __builtin_bit_cast(uint16_t, (half_t)v[e]) : from_float<bf16_t>(v[e]).bits;
    if (vec) {
        *(uint2_t *)((uint16_t *)p + idx) = uint2_t{bits[0] | (uint32_t)bits[1] << 16, bits[2] | (uint32_t)bits[3] << 16};
        return;
    }
    for (int e = 0; e < 4; e++) ((uint16_t *)p)[idx + e * stride] = bits[e];
}

// eight elements: 16 bytes of a 16-bit type at once
__device__ __forceinline__ void q8_store8(void *p, int64_t idx, int64_t stride, bool vec, int dtype, const float *v) {
    if (!vec || dtype == FHIP_F32) {
        q8_store4(p, idx, stride, vec, dtype, v);
        q8_store4(p, idx + 4 * stride, stride, vec, dtype, v + 4);
        return;
    }
    typedef uint4_t __attribute__((aligned(8))) uint4_at8_t;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (dtype == FHIP_F16) w[e] = __builtin_bit_cast(uint32_t, half2_t{(half_t)v[2 * e], (half_t)v[2 * e + 1]});
        else w[e] = from_float<bf16_t>(v[2 * e]).bits | (uint32_t)from_float<bf16_t>(v[2 * e + 1]).bits << 16;
    }
    *(uint4_at8_t *)((uint16_t *)p + idx) = uint4_t{w[0], w[1], w[2], w[3]};
}

// the largest of LANES consecutive lanes' values, in all of them
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    auto step = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    x = step(x, (uint32_t)dpp_mov_i<DPP_QUAD_XOR1>((int)x));
    x = step(x, (uint32_t)dpp_mov_i<DPP_QUAD_XOR2>((int)x));
    x = step(x, (uint32_t)dpp_mov_i<DPP_ROW_HALF_MIRROR>((int)x));
    if constexpr (LANES >= 16) x = step(x, (uint32_t)dpp_mov_i<DPP_ROW_MIRROR>((int)x));
    if constexpr (LANES >= 32) x = step(x, (uint32_t)__shfl_xor((int)x, 16, 64));
    return x;
}

// four codes of values x at scale s
template <int FMT>
__device__ __forceinline__ uint32_t q8_codes4(const float *x, float s, float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) w |= Q8Format<FMT>::code(x[e], s, inv) << (8 * e);
    return w;
}
template <int FMT>
__device__ __forceinline__ uint32_t q8_recode4(uint32_t w, float before, float s, float inv) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = __fmul_rn(Q8Format<FMT>::value(w, e), before);
    return q8_codes4<FMT>(x, s, inv);
}

// RMS norm of the rows x[u] of a workgroup's groups, rounded to the source's type.  The squares, rounded before they are added, are added left to right
// by one lane per row (the order of fhip_norm_rope).
template <int LPR, int RPG>
__device__ __forceinline__ void q8_norm_rows(const Q8Rows &J, float (&x)[RPG][8], float *tile, float *rms, int D, int d0, int d1, bool lane_on, int group) {
    constexpr int GR = 256 / LPR, W = GR * RPG, PITCH = LPR * 8 + 4;
#pragma unroll
    for (int u = 0; u < RPG; u++) {
        float *t = tile + (u * GR + group) * PITCH;
        if (lane_on) {
            *(float4_t *)(t + d0) = float4_t{__fmul_rn(x[u][0], x[u][0]), __fmul_rn(x[u][1], x[u][1]), __fmul_rn(x[u][2], x[u][2]), __fmul_rn(x[u][3], x[u][3])};
            *(float4_t *)(t + d1) = float4_t{__fmul_rn(x[u][4], x[u][4]), __fmul_rn(x[u][5], x[u][5]), __fmul_rn(x[u][6], x[u][6]), __fmul_rn(x[u][7], x[u][7])};
        }
    }
    float w[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int d = (e < 4 ? d0 : d1 - 4) + e;
        w[e] = lane_on ? q8_load(J.norm_w, d, J.norm_dtype) : 0.0f;
        bias[e] = lane_on && J.norm_b ? q8_load(J.norm_b, d, J.norm_dtype) : 0.0f;
    }
    __syncthreads();
    if (threadIdx.x < W) {
        const float *t = tile + threadIdx.x * PITCH;
        float ss = 0.0f;
#pragma unroll 4
        for (int i = 0; i < D; i += 8) {
            const float4_t a = *(const float4_t *)(t + i), c = *(const float4_t *)(t + i + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) ss = __fadd_rn(ss, a[e]);
#pragma unroll
            for (int e = 0; e < 4; e++) ss = __fadd_rn(ss, c[e]);
        }
        rms[threadIdx.x] = sqrtf(__fadd_rn(__fdiv_rn(ss, (float)D), J.eps));
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < RPG; u++) {
        const float r = rms[u * GR + group];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float v = __fmul_rn(__fdiv_rn(x[u][e], r), w[e]);
            if (J.norm_b) v = __fadd_rn(v, bias[e]);
            x[u][e] = lane_on ? q8_round_through(v, J.src_dtype) : 0.0f;
        }
    }
}

// ---- rows on their own ------------------------------------------------------------------------------------------------------------------
// Every new row is the only one of its block that comes with the call (blocks of one token, or one new token per sequence): LPR lanes hold a row,
// eight elements each, the two pieces of four whose pairs the rotation turns.  Groups of lanes take RPG positions of a head each, consecutive groups
// the heads of those positions, which share their rows of the tables and, in a model's projections, lie together; the positions lie together in the
// cache.  Where a row joins earlier ones and raises the scale (of a block's k-th row one time in k), its lanes code those again, one after the other.
// Bound: memory for prompts, 53 us for q, k and v of 8192 f16 rows of 32 / 8 heads at 128 (188 MB, 3.5 TB/s; 41 us where the caches hold them): wavefronts
// wait for 74 % of their cycles, the vector units (an exact quotient and its codes) are busy for 55 %; one chain of latencies for a token (3.8 us for one
// sequence, 7 to 8 us with norms over 64 sequences).
__device__ __forceinline__ uint32_t q8_divided(uint32_t t, const uint32_t m[2]) { return m[0] ? __umulhi(t, m[0]) >> m[1] : t; }

struct Q8RowPlace {
    int64_t src, dst, codes, scale;
    int64_t pos;
    int place, older;  // of the row; earlier rows of its block
    bool fresh;
};

template <int FMT>
__device__ __forceinline__ void q8_write_row(const Q8Rows &J, const Q8RowPlace &r, const float (&x)[8], uint32_t top, int d0, int d1, int D, bool lane_on, int j) {
    float s = fmaxf(__fmul_rn(__uint_as_float(top), 1.0f / Q8Format<FMT>::LARGEST), Q8_LEAST_SCALE), before = 0.0f;
    if (r.older > 0) {
        before = J.out.scales[r.scale];
        s = fmaxf(s, before);
    }
    const bool lost = top >= 0x7f800000u || before != before;
    if (lost) s = __uint_as_float(0x7fc00000u);
    const float inv = 1.0f / s;
    uint8_t *const c = J.out.codes + r.codes;
    if (lane_on) {
        const uint32_t w0 = lost ? 0u : q8_codes4<FMT>(x, s, inv), w1 = lost ? 0u : q8_codes4<FMT>(x + 4, s, inv);
        if (J.mode == 0) {
            *(uint32_t *)(c + d0) = w0;
            *(uint32_t *)(c + d1) = w1;
        } else {
            *(uint2_t *)(c + d0) = uint2_t{w0, w1};
        }
    }
    if (r.older > 0 && !lost && s != before && lane_on) {
        for (int i = 1; i <= r.older; i++) {
            uint2_t *const o = (uint2_t *)(c - i * J.out.cs[2] + 8 * j);
            const uint2_t w = *o;
            *o = uint2_t{q8_recode4<FMT>(w[0], before, s, inv), q8_recode4<FMT>(w[1], before, s, inv)};
        }
    }
    if (j == 0) J.out.scales[r.scale] = s;
}

// NEAR: strides and places below 2^31, multiplied in 32 bits (one instruction instead of five, of a quarter of the rate)
template <bool NEAR>
__device__ __forceinline__ int64_t q8_times(uint32_t n, int64_t stride) {
    return NEAR ? (int64_t)(int32_t)n * (int32_t)stride : (int64_t)n * stride;
}

template <int LPR, int RPG, bool NORM, bool NEAR>
__global__ __launch_bounds__(256) void q8_append_rows_kernel(Q8AppendParams p) {
    request_arguments<Q8AppendParams>();
    constexpr int GR = 256 / LPR, W = GR * RPG, PITCH = LPR * 8 + 4;
    __shared__ __attribute__((aligned(16))) float tile[NORM ? W * PITCH : 4];
    __shared__ float rms[NORM ? W : 1];
    const int ji = (p.jobs > 1 && blockIdx.x >= p.first_wg[1] ? 1 : 0) + (p.jobs > 2 && blockIdx.x >= p.first_wg[2] ? 1 : 0);
    const Q8Rows &J = p.job[ji];
    const int D = p.D, half = D / 2;
    const int group = threadIdx.x / LPR, j = threadIdx.x % LPR;
    const bool lane_on = 8 * j < D;
    const int d0 = J.mode == 0 ? 4 * j : 8 * j, d1 = J.mode == 0 ? half + 4 * j : 8 * j + 4;
    const uint32_t idx = (blockIdx.x - p.first_wg[ji]) * (uint32_t)GR + group, at = min(idx, J.total - 1);
    const uint32_t bi = q8_divided(at, J.by_heads), h = at - bi * (uint32_t)J.heads, b = q8_divided(bi, J.by_rows), i0 = (bi - b * J.span) * (uint32_t)RPG;
    const int T = 1 << J.out.log2_block;
    const int64_t len = p.lens ? p.lens[b] : 0;
    const int count = p.counts ? min(p.counts[b], J.n) : J.n;

    Q8RowPlace r[RPG];
    float4_t xa[RPG], xb[RPG], tc[RPG], ts[RPG];
    const int64_t place0 = p.row + len + i0, pos0 = J.pos0 + len + i0;
    // rows outside the view or the tables, and those that the sequence does not bring, are left out
    int64_t most = min((int64_t)count - i0, J.out.rows - place0);
    if (p.cos) most = min(most, p.table_rows - pos0);
    const int left = idx < J.total && p.row + len >= 0 && (!p.cos || J.pos0 + len >= 0) ? (int)max(min(most, (int64_t)RPG), (int64_t)0) : 0;
    const int64_t src0 = q8_times<NEAR>(b, J.s[0]) + q8_times<NEAR>(h, J.s[1]) + q8_times<NEAR>(i0, J.s[2]);
    const int64_t dst0 = q8_times<NEAR>(b, J.d[0]) + q8_times<NEAR>(h, J.d[1]) + q8_times<NEAR>(i0, J.d[2]);
    const int64_t codes0 = q8_times<NEAR>(b, J.out.cs[0]) + q8_times<NEAR>(h, J.out.cs[1]) + q8_times<NEAR>((uint32_t)place0, J.out.cs[2]);
    const int64_t scale0 = q8_times<NEAR>(b, J.out.ss[0]) + q8_times<NEAR>(h, J.out.ss[1]);
#pragma unroll
    for (int u = 0; u < RPG; u++) {
        r[u].fresh = u < left;
        const int v = u < left ? u : 0;  // (a row that is left out is read as the first one, which is there)
        r[u].pos = left > 0 ? pos0 + v : 0;
        r[u].place = (int)place0 + v;
        r[u].older = min((J.out.first + r[u].place) & (T - 1), r[u].place);
        r[u].src = src0 + v * J.s[2];
        r[u].dst = dst0 + v * J.d[2];
        r[u].codes = codes0 + v * J.out.cs[2];
        r[u].scale = scale0 + ((J.out.first + r[u].place) >> J.out.log2_block);
        xa[u] = xb[u] = ts[u] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        tc[u] = float4_t{1.0f, 1.0f, 1.0f, 1.0f};
        if (lane_on) {
            if (J.vec) {
                xa[u] = q8_load4(J.src, r[u].src + d0, J.src_dtype), xb[u] = q8_load4(J.src, r[u].src + d1, J.src_dtype);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    xa[u][e] = q8_load(J.src, r[u].src + (d0 + e) * J.s[3], J.src_dtype);
                    xb[u][e] = q8_load(J.src, r[u].src + (d1 + e) * J.s[3], J.src_dtype);
                }
            }
            if (J.mode != 2) {
                tc[u] = q8_load_turn(p.cos + r[u].pos * half + 4 * j);
                ts[u] = q8_load_turn(p.sin + r[u].pos * half + 4 * j);
            }
        }
    }
    float x[RPG][8];
#pragma unroll
    for (int u = 0; u < RPG; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) x[u][e] = xa[u][e], x[u][4 + e] = xb[u][e];
    if constexpr (NORM) {
        if (J.norm_w) q8_norm_rows<LPR, RPG>(J, x, tile, rms, D, d0, d1, lane_on, group);
    }
#pragma unroll
    for (int u = 0; u < RPG; u++) {
        if (J.mode != 2) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int a = J.mode == 0 ? e : 2 * e, o = J.mode == 0 ? 4 + e : 2 * e + 1;
                const float lo = x[u][a], hi = x[u][o];
                x[u][a] = __fsub_rn(__fmul_rn(lo, tc[u][e]), __fmul_rn(hi, ts[u][e]));
                x[u][o] = __fadd_rn(__fmul_rn(hi, tc[u][e]), __fmul_rn(lo, ts[u][e]));
            }
        }
        if (J.is_q) {
            if (r[u].fresh && lane_on) {
                q8_store4(J.dst, r[u].dst + d0 * J.d[3], J.d[3], J.vec, J.dst_dtype, x[u]);
                q8_store4(J.dst, r[u].dst + d1 * J.d[3], J.d[3], J.vec, J.dst_dtype, x[u] + 4);
            }
            continue;
        }
        uint32_t top = 0;  // magnitudes as bits: in their order NaN and infinity are the largest
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[u][e]) & 0x7fffffffu);
        top = lanes_max<LPR>(top);
        if (!r[u].fresh) continue;
        if (p.format == FHIP_Q8_INT8) q8_write_row<FHIP_Q8_INT8>(J, r[u], x[u], top, d0, d1, D, lane_on, j);
        else q8_write_row<FHIP_Q8_E4M3>(J, r[u], x[u], top, d0, d1, D, lane_on, j);
    }
}

// ---- blocks of rows ---------------------------------------------------------------------------------------------------------------------
// A workgroup takes W consecutive row slots of one job; LPR lanes hold a row, eight elements each: the two pieces of four whose pairs
// the rotation turns.  Slots of a job run over (batch, head, place): with blocks of more than one token the places start at the
// block that the first new row falls into, so that a block lies in one workgroup, which alone reads its old scale, finds the new one and codes its
// rows, earlier ones included if the scale has grown.
// Measured with 8192 f16 rows from the caches (q, k and v, floor 38 us; rows alone take 41 and 44): 57, 58, 56 and 68 us into blocks of 8, 16, 32 and 64 at
// 128 dims, 32 / 8 heads; 58, 55, 69 and 121 at 256, 16 / 4 heads, where a lane holds up to eight rows and registers leave two wavefronts per SIMD.
template <int LPR, int RPG, bool NORM>
__global__ __launch_bounds__(256) void q8_append_kernel(Q8AppendParams p) {
    constexpr int GR = 256 / LPR, W = GR * RPG, PITCH = LPR * 8 + 4;
    __shared__ uint32_t row_top[W];
    __shared__ __attribute__((aligned(16))) float tile[NORM ? W * PITCH : 4];
    __shared__ float rms[NORM ? W : 1];
    const int ji = (p.jobs > 1 && blockIdx.x >= p.first_wg[1] ? 1 : 0) + (p.jobs > 2 && blockIdx.x >= p.first_wg[2] ? 1 : 0);
    const Q8Rows &J = p.job[ji];
    const int D = p.D, half = D / 2, lt = J.is_q ? 0 : J.out.log2_block, T = 1 << lt;
    const int group = threadIdx.x / LPR, j = threadIdx.x % LPR;
    const bool lane_on = 8 * j < D;
    const int d0 = J.mode == 0 ? 4 * j : 8 * j, d1 = J.mode == 0 ? half + 4 * j : 8 * j + 4;
    const uint32_t slot0 = (blockIdx.x - p.first_wg[ji]) * (uint32_t)W;

    float x[RPG][8];
    int64_t place[RPG], cbase[RPG], sbase[RPG];
    bool fresh[RPG], block_new[RPG], block_old[RPG], older[RPG];
    float before[RPG];
    int64_t pos[RPG];
    int64_t src[RPG], dst[RPG];
#pragma unroll
    for (int u = 0; u < RPG; u++) {
        const uint32_t idx = slot0 + u * GR + group;
        const bool on = idx < J.total;
        const uint32_t bh = on ? idx / J.span : 0, i = on ? idx - bh * J.span : 0;
        const uint32_t b = bh / (uint32_t)J.heads, h = bh - b * (uint32_t)J.heads;
        const int64_t len = p.lens ? p.lens[b] : 0, start = p.row + len;
        int64_t cnt = p.counts ? min(max((int64_t)p.counts[b], (int64_t)0), (int64_t)J.n) : J.n;
        if (p.cos) {  // positions that the tables hold (values are left out with their keys)
            if (J.pos0 + len < 0) cnt = 0;
            cnt = min(cnt, p.table_rows - (J.pos0 + len));
        }
        // where the rows go; q's are left out with the keys of the same step
        if (start < 0) cnt = 0;
        cnt = min(cnt, J.out.rows - start);
        cnt = max(cnt, (int64_t)0);
        const int64_t base = lt ? ((J.out.first + start) >> lt << lt) - J.out.first : start;
        place[u] = base + i;
        fresh[u] = on && place[u] >= start && place[u] < start + cnt;
        const int64_t block_at = place[u] - (lt ? (int64_t)(i & (T - 1)) : 0);
        block_new[u] = on && block_at < start + cnt && block_at + T > start && cnt > 0;
        block_old[u] = block_new[u] && block_at < start && start > 0;
        older[u] = block_old[u] && place[u] >= 0 && place[u] < start;
        pos[u] = J.pos0 + len + (place[u] - start);
        src[u] = (int64_t)b * J.s[0] + (int64_t)h * J.s[1] + (place[u] - start) * J.s[2];
        dst[u] = (int64_t)b * J.d[0] + (int64_t)h * J.d[1] + (place[u] - start) * J.d[2];
        cbase[u] = (int64_t)b * J.out.cs[0] + (int64_t)h * J.out.cs[1] + place[u] * J.out.cs[2];
        sbase[u] = (int64_t)b * J.out.ss[0] + (int64_t)h * J.out.ss[1] + ((J.out.first + block_at) >> lt);
#pragma unroll
        for (int e = 0; e < 8; e++) x[u][e] = 0.0f;
        before[u] = block_old[u] ? J.out.scales[sbase[u]] : 0.0f;
        if (fresh[u] && lane_on) {
            if (J.vec) {
                const float4_t a = q8_load4(J.src, src[u] + d0, J.src_dtype), c = q8_load4(J.src, src[u] + d1, J.src_dtype);
#pragma unroll
                for (int e = 0; e < 4; e++) x[u][e] = a[e], x[u][4 + e] = c[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[u][e] = q8_load(J.src, src[u] + (d0 + e) * J.s[3], J.src_dtype);
                    x[u][4 + e] = q8_load(J.src, src[u] + (d1 + e) * J.s[3], J.src_dtype);
                }
            }
        }
    }
    if constexpr (NORM) {
        if (J.norm_w) {
            q8_norm_rows<LPR, RPG>(J, x, tile, rms, D, d0, d1, lane_on, group);
#pragma unroll
            for (int u = 0; u < RPG; u++)
                if (!fresh[u])
#pragma unroll
                    for (int e = 0; e < 8; e++) x[u][e] = 0.0f;
        }
    }
    if (J.mode != 2) {
#pragma unroll
        for (int u = 0; u < RPG; u++) {
            if (!fresh[u] || !lane_on) continue;
            const float4_t c = q8_load_turn(p.cos + pos[u] * half + 4 * j), s = q8_load_turn(p.sin + pos[u] * half + 4 * j);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int a = J.mode == 0 ? e : 2 * e, o = J.mode == 0 ? 4 + e : 2 * e + 1;
                const float lo = x[u][a], hi = x[u][o];
                x[u][a] = __fsub_rn(__fmul_rn(lo, c[e]), __fmul_rn(hi, s[e]));
                x[u][o] = __fadd_rn(__fmul_rn(hi, c[e]), __fmul_rn(lo, s[e]));
            }
        }
    }
    if (J.is_q) {
#pragma unroll
        for (int u = 0; u < RPG; u++) {
            if (!fresh[u] || !lane_on) continue;
            q8_store4(J.dst, dst[u] + d0 * J.d[3], J.d[3], J.vec, J.dst_dtype, x[u]);
            q8_store4(J.dst, dst[u] + d1 * J.d[3], J.d[3], J.vec, J.dst_dtype, x[u] + 4);
        }
        return;
    }
    // magnitudes as bits: in their order NaN and infinity are the largest
    uint32_t top[RPG];
#pragma unroll
    for (int u = 0; u < RPG; u++) {
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) t = max(t, __float_as_uint(x[u][e]) & 0x7fffffffu);
        top[u] = lanes_max<LPR>(t);
    }
    if (lt) {
#pragma unroll
        for (int u = 0; u < RPG; u++)
            if (j == 0) row_top[u * GR + group] = top[u];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < RPG; u++) {
            const int at = (u * GR + group) & ~(T - 1);
            uint32_t t = 0;
            for (int e = j; e < T; e += LPR) t = max(t, row_top[at + e]);
            top[u] = lanes_max<LPR>(t);
        }
    }
    const bool int8 = p.format == FHIP_Q8_INT8;
#pragma unroll
    for (int u = 0; u < RPG; u++) {
        if (!block_new[u]) continue;
        float s = fmaxf(__fmul_rn(__uint_as_float(top[u]), int8 ? 1.0f / Q8Format<FHIP_Q8_INT8>::LARGEST : 1.0f / Q8Format<FHIP_Q8_E4M3>::LARGEST), Q8_LEAST_SCALE);
        if (block_old[u]) s = fmaxf(s, before[u]);
        const bool lost = top[u] >= 0x7f800000u || before[u] != before[u];
        if (lost) s = __uint_as_float(0x7fc00000u);
        const float inv = 1.0f / s;
        uint8_t *const c = J.out.codes + cbase[u];
        if (lane_on && fresh[u]) {
            uint32_t w0 = 0, w1 = 0;
            if (!lost) {
                w0 = int8 ? q8_codes4<FHIP_Q8_INT8>(x[u], s, inv) : q8_codes4<FHIP_Q8_E4M3>(x[u], s, inv);
                w1 = int8 ? q8_codes4<FHIP_Q8_INT8>(x[u] + 4, s, inv) : q8_codes4<FHIP_Q8_E4M3>(x[u] + 4, s, inv);
            }
            *(uint32_t *)(c + d0) = w0;
            *(uint32_t *)(c + d1) = w1;
        } else if (lane_on && older[u] && !lost && s != before[u]) {
            const uint32_t w0 = *(const uint32_t *)(c + d0), w1 = *(const uint32_t *)(c + d1);
            *(uint32_t *)(c + d0) = int8 ? q8_recode4<FHIP_Q8_INT8>(w0, before[u], s, inv) : q8_recode4<FHIP_Q8_E4M3>(w0, before[u], s, inv);
            *(uint32_t *)(c + d1) = int8 ? q8_recode4<FHIP_Q8_INT8>(w1, before[u], s, inv) : q8_recode4<FHIP_Q8_E4M3>(w1, before[u], s, inv);
        }
        if (j == 0 && (((u * GR + group) & (T - 1)) == 0)) J.out.scales[sbase[u]] = s;
    }
}

// slots: of a job per workgroup.  0: more than a launch may have (2^32 lanes)
static uint32_t append_workgroups(Q8AppendParams &p, uint32_t slots) {
    uint32_t wgs = 0;
    for (int i = 0; i < p.jobs; i++) {
        p.first_wg[i] = wgs;
        wgs += (p.job[i].total + slots - 1) / slots;
    }
    if (wgs < (1u << 24)) return wgs;
    set_error("q8_append: more rows than a launch has lanes for");
    return 0;
}
// t / d for t < 2^31 as the high half of t * m[0], shifted down by m[1] (m[0] = 0: d is 1): with 2^l >= d the factor ceil(2^(31 + l) / d) is off by less
// than one in 2^l / d, which is too little to reach the next quotient (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994)
static void divisor(uint32_t d, uint32_t m[2]) {
    m[0] = m[1] = 0;
    if (d <= 1) return;
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) l++;
    m[0] = (uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d);
    m[1] = l - 1;
}
template <int LPR, int RPG>
static int launch_rows(Q8AppendParams &p, bool normed, hipStream_t stream) {
    for (int i = 0; i < p.jobs; i++) {  // a slot is RPG positions of a head
        Q8Rows &j = p.job[i];
        const uint32_t sequences = j.total / ((uint32_t)j.heads * j.span);
        j.span = ((uint32_t)j.n + RPG - 1) / RPG;
        j.total = sequences * (uint32_t)j.heads * j.span;
        divisor((uint32_t)j.heads, j.by_heads);
        divisor(j.span, j.by_rows);
    }
    bool near = true;
    for (int i = 0; i < p.jobs; i++) {
        const Q8Rows &j = p.job[i];
        auto far = [](int64_t x) { return x >= INT32_MAX || x <= INT32_MIN; };
        for (int d = 0; d < 3; d++) near = near && !far(j.s[d]) && !far(j.d[d]) && !far(j.out.cs[d]);
        near = near && !far(j.out.ss[0]) && !far(j.out.ss[1]);
    }
    const dim3 grid(append_workgroups(p, 256 / LPR));
    if (grid.x == 0) return FHIP_ERR_UNSUPPORTED;
    if (normed && near) hipLaunchKernelGGL((q8_append_rows_kernel<LPR, RPG, true, true>), grid, dim3(256), 0, stream, p);
    else if (normed) hipLaunchKernelGGL((q8_append_rows_kernel<LPR, RPG, true, false>), grid, dim3(256), 0, stream, p);
    else if (near) hipLaunchKernelGGL((q8_append_rows_kernel<LPR, RPG, false, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((q8_append_rows_kernel<LPR, RPG, false, false>), grid, dim3(256), 0, stream, p);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}
template <int LPR, int RPG>
static int launch_blocks(Q8AppendParams &p, bool normed, hipStream_t stream) {
    const dim3 grid(append_workgroups(p, 256 / LPR * RPG));
    if (grid.x == 0) return FHIP_ERR_UNSUPPORTED;
    if (normed) hipLaunchKernelGGL((q8_append_kernel<LPR, RPG, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((q8_append_kernel<LPR, RPG, false>), grid, dim3(256), 0, stream, p);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}
template <int LPR>
static int launch_append_lpr(Q8AppendParams &p, int max_block, bool rows_alone, bool normed, hipStream_t stream) {
    constexpr int GR = 256 / LPR;
    if (rows_alone) {
        uint64_t rows = 0;
        for (int i = 0; i < p.jobs; i++) rows += p.job[i].total;
        // two positions per group of lanes where that still gives every CU eight workgroups (us, q, k and v of 8192 f16 rows of 32/8 heads at 128, with
        // one, two and four: 57, 52 and 72)
        if (rows >= (uint64_t)GR * 2 * 2048) return launch_rows<LPR, 2>(p, normed, stream);
        return launch_rows<LPR, 1>(p, normed, stream);
    }
    if (max_block <= GR) return launch_blocks<LPR, 1>(p, normed, stream);
    if (max_block <= 2 * GR) return launch_blocks<LPR, 2>(p, normed, stream);
    if constexpr (LPR > 8) {  // 64 tokens on groups of 16 or 32 lanes
        if (max_block <= 4 * GR) return launch_blocks<LPR, 4>(p, normed, stream);
        if constexpr (LPR > 16) return launch_blocks<LPR, 8>(p, normed, stream);
    }
    return FHIP_ERR_UNSUPPORTED;  // (no such block)
}
int launch_q8_append(Q8AppendParams &p, int max_block, bool rows_alone, bool normed, hipStream_t stream) {
    if (p.D <= 64) return launch_append_lpr<8>(p, max_block, rows_alone, normed, stream);
    if (p.D <= 128) return launch_append_lpr<16>(p, max_block, rows_alone, normed, stream);
    return launch_append_lpr<32>(p, max_block, rows_alone, normed, stream);
}

// ---- reading back -----------------------------------------------------------------------------------------------------------------------
// Eight codes per lane and piece, UNROLL pieces requested before the first is stored, one rounding of the product.  Bound by bytes: 36 us for 67 M
// elements of e4m3 to bf16 (201 MB, 5.6 TB/s).
template <int FMT, int UNROLL>
__global__ __launch_bounds__(256) void q8_dequantize_kernel(Q8ReadParams p, Q8ReadDivisors div, uint32_t total) {
    request_arguments<Q8ReadParams>();
    const uint32_t pieces = (uint32_t)p.D / 8, at0 = blockIdx.x * (256u * UNROLL) + threadIdx.x;
    uint2_t w[UNROLL];
    float s[UNROLL];
    int64_t out[UNROLL];
    bool there[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
        const uint32_t at = at0 + 256 * u, t = min(at, total - 1);
        const uint32_t r = q8_divided(t, div.pieces), piece = t - r * pieces, bh = q8_divided(r, div.rows), i = r - bh * (uint32_t)p.n,
                       b = q8_divided(bh, div.heads), h = bh - b * (uint32_t)p.H;
        const int64_t place = p.row + (p.lens ? p.lens[b] : 0) + i;
        there[u] = at < total && place >= 0 && place < p.x.rows;
        const int64_t from = there[u] ? place : 0;
        s[u] = p.x.scales[(int64_t)b * p.x.ss[0] + (int64_t)h * p.x.ss[1] + ((p.x.first + from) >> p.x.log2_block)];
        w[u] = *(const uint2_t *)(p.x.codes + (int64_t)b * p.x.cs[0] + (int64_t)h * p.x.cs[1] + from * p.x.cs[2] + 8 * piece);
        out[u] = (int64_t)b * p.os[0] + (int64_t)h * p.os[1] + (int64_t)i * p.os[2] + (int64_t)(8 * piece) * p.os[3];
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
        if (!there[u]) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __fmul_rn(Q8Format<FMT>::value(w[u][e >> 2], e & 3), s[u]);
        q8_store8(p.out, out[u], p.os[3], p.vec, p.out_dtype, v);
    }
}

int launch_q8_dequantize(const Q8ReadParams &p, hipStream_t stream) {
    // parts of at most 2^30 pieces: of the batch, or of one sequence's rows
    const uint64_t per_row = (uint64_t)p.H * (p.D / 8), most_rows = std::max<uint64_t>(1, (1u << 30) / per_row);
    const int rows = (int)std::min<uint64_t>(p.n, most_rows), sequences = (int)std::max<uint64_t>(1, std::min<uint64_t>(p.B, most_rows / rows));
    const int64_t bytes = p.out_dtype == FHIP_F32 ? 4 : 2;
    for (int64_t b = 0; b < p.B; b += sequences)
        for (int64_t i = 0; i < p.n; i += rows) {
            Q8ReadParams q = p;
            q.B = (int)std::min<int64_t>(sequences, p.B - b);
            q.n = (int)std::min<int64_t>(rows, p.n - i);
            q.x.codes += b * p.x.cs[0];
            q.x.scales += b * p.x.ss[0];
            q.out = (char *)p.out + (b * p.os[0] + i * p.os[2]) * bytes;
            q.row += i;
            if (p.lens) q.lens += b;
            Q8ReadDivisors div;
            divisor((uint32_t)q.D / 8, div.pieces);
            divisor((uint32_t)q.n, div.rows);
            divisor((uint32_t)q.H, div.heads);
            const uint32_t total = (uint32_t)(per_row * q.n * q.B);
            // four pieces a lane where that leaves every CU four workgroups (8192 f16 rows of 8 heads at 128: 7.4 us, with one 9.6; 32 times that: 36 and 51)
            const bool many = total >= 4u * 256 * 1024, int8 = q.format == FHIP_Q8_INT8;
            const dim3 grid((total + (many ? 1023 : 255)) / (many ? 1024 : 256));
            if (many && int8) hipLaunchKernelGGL((q8_dequantize_kernel<FHIP_Q8_INT8, 4>), grid, dim3(256), 0, stream, q, div, total);
            else if (many) hipLaunchKernelGGL((q8_dequantize_kernel<FHIP_Q8_E4M3, 4>), grid, dim3(256), 0, stream, q, div, total);
            else if (int8) hipLaunchKernelGGL((q8_dequantize_kernel<FHIP_Q8_INT8, 1>), grid, dim3(256), 0, stream, q, div, total);
            else hipLaunchKernelGGL((q8_dequantize_kernel<FHIP_Q8_E4M3, 1>), grid, dim3(256), 0, stream, q, div, total);
            FHIP_HIP_CHECK(hipGetLastError());
        }
    return FHIP_OK;
}

}  // namespace fhip
