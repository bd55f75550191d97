// The 8-bit key / value cache: new rows coded as they are written (with the norm and the rotation in front of it), and rows read back.
// The wide cache's counterparts are in rope.hip and kv_cache.hip; the reference has neither (its cache holds the tensors' own type,
// fusor-ml/fusor/src/cache/kv_cache.rs:13-68).
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

// A workgroup takes W consecutive row slots of one job; LPR lanes hold a row, eight elements each: the two pieces of four whose pairs
// the rotation turns.  Slots of a job run over (batch, head, place): with blocks of more than one token the places start at the
// block that the first new row falls into, so that a block lies in one workgroup, which alone reads its old scale, finds the new one and codes its
// rows, earlier ones included if the scale has grown.
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
            // squares, rounded before they are added left to right by one lane per row (the order of fhip_norm_rope)
#pragma unroll
            for (int u = 0; u < RPG; u++) {
                float *t = tile + (u * GR + group) * PITCH;
                if (lane_on) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        t[d0 + e] = __fmul_rn(x[u][e], x[u][e]);
                        t[d1 + e] = __fmul_rn(x[u][4 + e], x[u][4 + e]);
                    }
                }
            }
            __syncthreads();
            if (threadIdx.x < W) {
                const float *t = tile + threadIdx.x * PITCH;
                float ss = 0.0f;
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
            float w[8], bias[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = (e < 4 ? d0 : d1 - 4) + e;
                w[e] = lane_on ? q8_load(J.norm_w, d, J.norm_dtype) : 0.0f;
                bias[e] = lane_on && J.norm_b ? q8_load(J.norm_b, d, J.norm_dtype) : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < RPG; u++) {
                const float r = rms[u * GR + group];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float v = __fmul_rn(__fdiv_rn(x[u][e], r), w[e]);
                    if (J.norm_b) v = __fadd_rn(v, bias[e]);
                    x[u][e] = lane_on && fresh[u] ? q8_round_through(v, J.src_dtype) : 0.0f;
                }
            }
        }
    }
    if (J.mode != 2) {
#pragma unroll
        for (int u = 0; u < RPG; u++) {
            if (!fresh[u] || !lane_on) continue;
            const float4_t c = *(const float4_t *)(p.cos + pos[u] * half + 4 * j), s = *(const float4_t *)(p.sin + pos[u] * half + 4 * j);
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

template <int LPR, int RPG>
static int launch_append_rpg(Q8AppendParams &p, bool normed, hipStream_t stream) {
    constexpr uint32_t W = 256 / LPR * RPG;
    uint32_t wgs = 0;
    for (int i = 0; i < p.jobs; i++) {
        p.first_wg[i] = wgs;
        wgs += (p.job[i].total + W - 1) / W;
    }
    if (normed) hipLaunchKernelGGL((q8_append_kernel<LPR, RPG, true>), dim3(wgs), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((q8_append_kernel<LPR, RPG, false>), dim3(wgs), dim3(256), 0, stream, p);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}
template <int LPR>
static int launch_append_lpr(Q8AppendParams &p, int max_block, bool normed, hipStream_t stream) {
    constexpr int GR = 256 / LPR;
    if (max_block <= GR) return launch_append_rpg<LPR, 1>(p, normed, stream);
    if (max_block <= 2 * GR) return launch_append_rpg<LPR, 2>(p, normed, stream);
    if constexpr (LPR > 8)
        if (max_block <= 4 * GR) return launch_append_rpg<LPR, 4>(p, normed, stream);
    if constexpr (LPR > 16) return launch_append_rpg<LPR, 8>(p, normed, stream);
    set_error("q8 append: block of %d tokens", max_block);
    return FHIP_ERR_INVALID_ARG;
}
int launch_q8_append(Q8AppendParams &p, int max_block, bool normed, hipStream_t stream) {
    if (p.D <= 64) return launch_append_lpr<8>(p, max_block, normed, stream);
    if (p.D <= 128) return launch_append_lpr<16>(p, max_block, normed, stream);
    return launch_append_lpr<32>(p, max_block, normed, stream);
}

// Eight codes per lane and step.
template <int FMT>
__global__ __launch_bounds__(256) void q8_dequantize_kernel(Q8ReadParams p, uint32_t pieces, uint64_t total) {
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256) {
        const uint32_t piece = (uint32_t)(at % pieces);
        uint64_t t = at / pieces;
        const uint32_t i = (uint32_t)(t % (uint32_t)p.n);
        t /= (uint32_t)p.n;
        const uint32_t h = (uint32_t)(t % (uint32_t)p.H), b = (uint32_t)(t / (uint32_t)p.H);
        const int64_t place = p.row + (p.lens ? p.lens[b] : 0) + i;
        if (place < 0 || place >= p.x.rows) continue;
        const float s = p.x.scales[(int64_t)b * p.x.ss[0] + (int64_t)h * p.x.ss[1] + ((p.x.first + place) >> p.x.log2_block)];
        const uint2_t w = *(const uint2_t *)(p.x.codes + (int64_t)b * p.x.cs[0] + (int64_t)h * p.x.cs[1] + place * p.x.cs[2] + 8 * piece);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __fmul_rn(Q8Format<FMT>::value(w[e >> 2], e & 3), s);
        const int64_t o = (int64_t)b * p.os[0] + (int64_t)h * p.os[1] + (int64_t)i * p.os[2] + (int64_t)(8 * piece) * p.os[3];
        q8_store4(p.out, o, p.os[3], p.vec, p.out_dtype, v);
        q8_store4(p.out, o + 4 * p.os[3], p.os[3], p.vec, p.out_dtype, v + 4);
    }
}

int launch_q8_dequantize(const Q8ReadParams &p, hipStream_t stream) {
    const uint32_t pieces = (uint32_t)p.D / 8;
    const uint64_t total = (uint64_t)p.B * p.H * p.n * pieces;
    if (total == 0) return FHIP_OK;
    const uint64_t blocks = (total + 255) / 256;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    if (p.format == FHIP_Q8_INT8) hipLaunchKernelGGL(q8_dequantize_kernel<FHIP_Q8_INT8>, grid, dim3(256), 0, stream, p, pieces, total);
    else hipLaunchKernelGGL(q8_dequantize_kernel<FHIP_Q8_E4M3>, grid, dim3(256), 0, stream, p, pieces, total);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

}  // namespace fhip
