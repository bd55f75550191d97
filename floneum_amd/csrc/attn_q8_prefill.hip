// Attention over the 8-bit cache for many query rows: tiles of 64 keys, widened to f16 once per workgroup on their way into LDS.
//
// A workgroup of WAVES wavefronts serves 32 * WAVES columns ((query row, head of the group) pairs of one KV head: heads of a group share the
// tile, and a causal mask cuts columns of few rows); a wavefront has 32 of them on v_mfma_f32_32x32x16_f16:
//   S^T[key][column] = K Q^T     K in LDS by rows, Q in registers
//   O^T[dim][column] += V^T P^T  V in LDS transposed, eight keys of a dim to 16 bytes, in the order in which the scores' registers hold the keys
// so that probabilities go from the scores' registers to the operand's without leaving their lane.  A lane holds 16 keys of each half of the tile;
// their scales lie in one register of 16 lanes (a DPP row) and are broadcast by the multiplication that uses them.
//
// Numbers are brought to f16 as in the kernel for few rows (attn_q8_decode.hip): codes exactly, a column's q scaled by a power of two, one term for
// 16-bit queries and two for f32.  The values' scales go with the probabilities, brought below 2^15 by a power of two E that follows the largest
// scale met: w_j = p_j vs_j 2^(15 - E), out = 2^(E - 15) sum w_j c_j / sum p_j.
#include <algorithm>
#include <utility>

#include "q8.h"
#include "q8_attention.h"
#include "q8_device.h"

namespace fhip {

constexpr int Q8_TILE = 64;

template <int N, typename F, int... I>
__device__ __forceinline__ void q8_each(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void q8_each(F &&f) {
    q8_each<N>(f, std::make_integer_sequence<int, N>{});
}
// x of lane N of the own row of 16 lanes
template <int N>
__device__ __forceinline__ float row_lane(float x) {
    return dpp_mov<0x150 + N>(x);
}
__device__ __forceinline__ half8_t q8_widen8_pairs(half2_t a, half2_t b, half2_t c, half2_t d) {
    return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Waits: `WAVES_PER_SIMD` wavefronts share a SIMD's registers.
template <int DV, int TERMS, int FMT, int WAVES, bool MASK>
__global__ __launch_bounds__(64 * WAVES, DV <= 128 ? 2 : 1) void q8_prefill_kernel(Q8AttnParams p) {
    request_arguments<Q8AttnParams>();
    constexpr int COLS = 32 * WAVES, STEPS = DV / 16, DT = DV / 32, UNITS = DV / 16, CHUNKS = DV / 8;
    // LDS, 16-byte chunks: K [key][chunk of 8 dims], V [dim][chunk of 8 keys]; the chunk is turned by the row so that 16 rows' pieces lie in
    // different banks
    __shared__ __attribute__((aligned(16))) half_t lds_k[2][Q8_TILE * DV];
    __shared__ __attribute__((aligned(16))) half_t lds_v[2][Q8_TILE * DV];
    auto k_at = [](int key, int chunk) { return (key * CHUNKS + (chunk ^ (DV % 128 == 0 ? key & 15 : (key >> 1) & 7))) * 8; };
    auto v_at = [](int dim, int chunk) { return (dim * 8 + (chunk ^ (((dim >> 1) ^ (dim >> 4)) & 7))) * 8; };

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
    const int NC = p.G * p.Sq, units = p.B * p.Hkv;
    // consecutive workgroups take different KV heads, so that the workgroups of one (with units a multiple of the XCDs) share an XCD's L2; the
    // columns that see most keys first
    const int blocks = (NC + COLS - 1) / COLS;
    const uint32_t id = blockIdx.x;
    const int bg = (int)(id % units);
    const uint32_t rest = id / units;
    const int split = (int)(rest % p.nsplit), cb = blocks - 1 - (int)(rest / p.nsplit);
    const int kvh = bg % p.Hkv, b = bg / p.Hkv;
    const int c0 = cb * COLS, c1 = min(c0 + COLS, NC) - 1;

    const Q8Range vis = q8_visible(p, b, c0 / p.G, c1 / p.G);
    const int len = vis.hi - vis.lo;
    const int share = (max(p.min_chunk, (int)(((uint32_t)len + p.nsplit - 1) / (uint32_t)p.nsplit)) + 63) / 64 * 64;
    const int64_t lo64 = vis.lo + (int64_t)split * share;
    const int lo = (int)min(lo64, (int64_t)vis.hi), hi = (int)min((int64_t)vis.hi, lo64 + share);

    const int c = min(c0 + wave * 32 + n, NC - 1);
    const int row = c / p.G, head = kvh * p.G + c % p.G;
    half8_t q[TERMS][STEPS];
    float colscale;
    {  // lane half h holds dims 16 i + 8 h .. + 7 of step i
        const int64_t base = (int64_t)b * p.qs[0] + (int64_t)head * p.qs[1] + (int64_t)row * p.qs[2];
        Q8Query8<TERMS> raw[STEPS];
        if (p.q_vec) {
#pragma unroll
            for (int i = 0; i < STEPS; i++) raw[i].load(p, base, 16 * i + 8 * h);
        } else {
#pragma unroll
            for (int i = 0; i < STEPS; i++) raw[i].gather(p, base, 16 * i + 8 * h);
        }
        if (TERMS == 1 && p.q_dtype == FHIP_F16 && p.scale != 0.0f) {  // as they are
#pragma unroll
            for (int i = 0; i < STEPS; i++) q[0][i] = raw[i].halves(p, 16 * i + 8 * h);
            colscale = q8_score_scale(p, 0);
        } else {
            float x[STEPS][8], top = 0.0f;
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                raw[i].widen(p, 16 * i + 8 * h, x[i]);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[i][e]));
            }
            const int shift = q8_query_shift(fmaxf(top, xor32(top)));
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    half_t high, low;
                    q8_query_terms<TERMS>(p, x[i][e], shift, high, low);
                    q[0][i][e] = high;
                    if constexpr (TERMS == 2) q[1][i][e] = low;
                }
            colscale = q8_score_scale(p, shift);
        }
    }
    const int64_t at = vis.pos0 + row;
    const int limit = (int)(p.causal ? max((int64_t)0, min((int64_t)hi, at + 1)) : hi);
    const int start = (int)(p.window > 0 ? min((int64_t)hi, max((int64_t)0, at - p.window + 1)) : 0);

    const int64_t mask_row = (p.mask_kind == FHIP_MASK_QK ? row : b) * p.ms0;
    float16_t acc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[t][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int E = -200;

    const uint8_t *const kbase = p.k.codes + (int64_t)b * p.k.cs[0] + (int64_t)kvh * p.k.cs[1];
    const uint8_t *const vbase = p.v.codes + (int64_t)b * p.v.cs[0] + (int64_t)kvh * p.v.cs[1];
    const float *const kscale = p.k.scales + (int64_t)b * p.k.ss[0] + (int64_t)kvh * p.k.ss[1];
    const float *const vscale = p.v.scales + (int64_t)b * p.v.ss[0] + (int64_t)kvh * p.v.ss[1];
    const int pitch = (p.D + 15) & ~15, krow = (int)p.k.cs[2], vrow = (int)p.v.cs[2];

    // staging: 256 lanes move a tile's keys and 256 its values (the same ones in workgroups of four wavefronts)
    constexpr int KN = 4 * DV / 256 > 0 ? 4 * DV / 256 : 1, VN = (2 * DV + 255) / 256;
    const int sid = threadIdx.x & 255;
    const bool moves_k = WAVES == 4 || wave >= 4, moves_v = WAVES == 4 || wave < 4;
    uint4_t ksrc[KN];
    uint32_t vsrc[VN][8];
    // Rows beyond the share are loaded as its last one (what lies there may be anything, 8-bit NaN among it); pieces beyond a row from its start:
    // q is 0 there, and such dims of v are not written.
    auto load_tile = [&](int k0) {
        const int last = hi - 1 - k0;
        if (moves_k) {
            const uint8_t *const r = kbase + (int64_t)k0 * krow;
#pragma unroll
            for (int i = 0; i < KN; i++) {
                const int u = sid + 256 * i, key = u / UNITS, off = 16 * (u % UNITS);
                ksrc[i] = *(const uint4_t *)(r + (uint32_t)(min(key, last) * krow + (off < pitch ? off : 0)));
            }
        }
        if (moves_v) {
            const uint8_t *const r = vbase + (int64_t)k0 * vrow;
#pragma unroll
            for (int i = 0; i < VN; i++) {
                const int u = sid + 256 * i;
                if (2 * DV % 256 != 0 && u >= 2 * DV) continue;
                const int kg = u / (DV / 4), off = 4 * (u % (DV / 4)), base = 16 * (kg >> 1) + 4 * (kg & 1);
                const uint32_t o = off < pitch ? off : 0;
#pragma unroll
                for (int e = 0; e < 8; e++) vsrc[i][e] = *(const uint32_t *)(r + (uint32_t)(min(base + (e & 3) + 8 * (e >> 2), last) * vrow + o));
            }
        }
    };
    auto store_tile = [&](int buf) {
        if (moves_k) {
#pragma unroll
            for (int i = 0; i < KN; i++) {
                const int u = sid + 256 * i, key = u / UNITS, chunk = 2 * (u % UNITS);
#pragma unroll
                for (int e = 0; e < 2; e++)
                    *(half8_t *)&lds_k[buf][k_at(key, chunk + e)] =
                        q8_widen8_pairs(q8_pair_low<FMT>(ksrc[i][2 * e]), q8_pair_high<FMT>(ksrc[i][2 * e]), q8_pair_low<FMT>(ksrc[i][2 * e + 1]),
                                        q8_pair_high<FMT>(ksrc[i][2 * e + 1]));
            }
        }
        if (moves_v) {
#pragma unroll
            for (int i = 0; i < VN; i++) {
                const int u = sid + 256 * i;
                if (2 * DV % 256 != 0 && u >= 2 * DV) continue;
                const int kg = u / (DV / 4), dim = 4 * (u % (DV / 4));
                half2_t x[4][4];  // [dim][pair of keys]
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t a = vsrc[i][2 * e], c2 = vsrc[i][2 * e + 1];
                    const uint32_t t01 = __builtin_amdgcn_perm(c2, a, 0x05010400u), t23 = __builtin_amdgcn_perm(c2, a, 0x07030602u);
                    x[0][e] = q8_pair_low<FMT>(t01), x[1][e] = q8_pair_high<FMT>(t01);
                    x[2][e] = q8_pair_low<FMT>(t23), x[3][e] = q8_pair_high<FMT>(t23);
                }
#pragma unroll
                for (int t = 0; t < 4; t++) *(half8_t *)&lds_v[buf][v_at(dim + t, kg)] = q8_widen8_pairs(x[t][0], x[t][1], x[t][2], x[t][3]);
            }
        }
    };
    // the scales of the lane's keys, one of 16 per lane of a row: key 32 u + 8 (i / 4) + 4 h + i % 4 in lane i
    float ks[2], vs[2];
    auto load_scales = [&](int k0) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int key = min(k0 + 32 * u + 8 * ((lane >> 2) & 3) + 4 * h + (lane & 3), hi - 1);
            ks[u] = kscale[(p.k.first + key) >> p.k.log2_block];
            vs[u] = vscale[(p.v.first + key) >> p.v.log2_block];
        }
    };

    if (lo < hi) {
        load_tile(lo);
        load_scales(lo);
        store_tile(0);
    }
    lds_barrier();
    int buf = 0;
    for (int k0 = lo; k0 < hi; k0 += Q8_TILE, buf ^= 1) {
        const bool more = k0 + Q8_TILE < hi;
        if (more) load_tile(k0 + Q8_TILE);
        float kf[2], vf[2];
        int e = E;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            // NaN among the values' scales goes by way of the scores, where rows that a mask hides are taken out
            const bool lost = vs[u] != vs[u];
            kf[u] = lost ? vs[u] : ks[u], vf[u] = lost ? 0.0f : vs[u];
            e = max(e, vf[u] > 0.0f ? __builtin_amdgcn_frexp_expf(vf[u]) : -200);
        }
        e = wave_reduce_i(e, [](int x, int y) { return x > y ? x : y; });
        float grown = 1.0f;
        if (e > E) grown = __builtin_ldexpf(1.0f, max(E - e, -1000)), E = e;
#pragma unroll
        for (int u = 0; u < 2; u++) vf[u] = __builtin_ldexpf(vf[u], 15 - E);
        if (more) load_scales(k0 + Q8_TILE);

        float16_t s[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[u][r] = 0.0f;
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                const half8_t a = *(const half8_t *)&lds_k[buf][k_at(32 * u + n, 2 * i + h)];
#pragma unroll
                for (int x = TERMS - 1; x >= 0; x--) s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q[x][i], s[u], 0, 0, 0);
            }
        }
        // times the keys' scales; with a mask in the log2 domain, else before the column's scale (which is positive)
        float top = -INFINITY;
        if constexpr (MASK) {
#pragma unroll
            for (int u = 0; u < 2; u++)
                q8_each<16>([&](auto i) {
                    constexpr int r = decltype(i)::value;
                    const int key = k0 + 32 * u + 8 * (r / 4) + 4 * h + r % 4;
                    float add = -INFINITY;
                    if (key < limit) add = q8_load_any(p.mask, mask_row + key * p.ms1, p.q_dtype);
                    const float t = q8_with_mask(row_lane<r>(kf[u]) * s[u][r] * colscale, add * Q8_LOG2E);
                    s[u][r] = add == -INFINITY ? -INFINITY : t;
                });
        } else {
#pragma unroll
            for (int u = 0; u < 2; u++)
                q8_each<16>([&](auto i) {
                    constexpr int r = decltype(i)::value;
                    s[u][r] = row_lane<r>(kf[u]) * s[u][r];
                });
            if (__builtin_amdgcn_ballot_w64(k0 + Q8_TILE > limit || k0 < start) != 0) {
#pragma unroll
                for (int u = 0; u < 2; u++)
                    q8_each<16>([&](auto i) {
                        constexpr int r = decltype(i)::value;
                        const int key = 32 * u + 8 * (r / 4) + r % 4;
                        if (key >= limit - k0 - 4 * h || key < start - k0 - 4 * h) s[u][r] = -INFINITY;
                    });
            }
        }
        const float g = MASK ? 1.0f : colscale;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[u][r]);
        top = fmaxf(top, xor32(top)) * g;
        top = fmaxf(m, top);
        const float ref = top == -INFINITY ? 0.0f : top;
        if (__builtin_amdgcn_ballot_w64(top > m || grown != 1.0f) != 0) {
            const float shrink = __builtin_amdgcn_exp2f(m - ref);
            m = top;
            l *= shrink;
#pragma unroll
            for (int t = 0; t < DT; t++) acc[t] *= shrink * grown;
        }
        half8_t pw[TERMS][4];
#pragma unroll
        for (int u = 0; u < 2; u++)
            q8_each<16>([&](auto i) {
                constexpr int r = decltype(i)::value;
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], g, -ref));
                l += x;
                float w = row_lane<r>(vf[u]) * x;
                if constexpr (TERMS == 2) asm("" : "+v"(w));  // (both terms from the same rounded w: the product is not contracted into them)
                const half_t high = (half_t)w;
                pw[0][2 * u + r / 8][r % 8] = high;
                if constexpr (TERMS == 2) pw[1][2 * u + r / 8][r % 8] = (half_t)(w - (float)high);
            });
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const half8_t a = *(const half8_t *)&lds_v[buf][v_at(32 * t + n, 2 * j + h)];
#pragma unroll
                for (int x = TERMS - 1; x >= 0; x--) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pw[x][j], acc[t], 0, 0, 0);
            }
        if (more) store_tile(buf ^ 1);
        lds_barrier();
    }
    l += xor32(l);
    if (c0 + wave * 32 + n >= NC) return;
    const float up = __builtin_ldexpf(1.0f, max(E, -140) - 15);
    const int64_t o = (int64_t)b * p.os[0] + (int64_t)head * p.os[1] + (int64_t)row * p.os[2];
    const int64_t part = ((int64_t)bg * p.nsplit + split) * NC + c;
    // (sum / l) 2^(E - 15): the quotient first, which stays in range
    const float inv = p.nsplit > 1 ? 1.0f : 1.0f / l;
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * t + 2 * r + 4 * h;
            if (d >= p.D) continue;
            float4_t v = {acc[t][r], acc[t][r + 1], acc[t][r + 2], acc[t][r + 3]};
            if (p.nsplit > 1) {
                *(float4_t *)(p.partials + part * DV + d) = v * up;
            } else {
                v = v * inv * up;
                q8_store4_any(p, o + d * p.os[3], v);
            }
        }
    if (p.nsplit > 1 && h == 0) {
        float *const ml = p.partials + (int64_t)p.B * p.Hkv * p.nsplit * NC * DV + part * 2;
        ml[0] = m, ml[1] = l;
    }
}

static int q8_padded_dim(int D) { return (D + 63) / 64 * 64; }

Q8AttnPlan q8_prefill_plan(const Q8AttnParams &p) {
    Q8AttnPlan plan;
    plan.prefill = true;
    const int64_t NC = (int64_t)p.G * p.Sq, units = (int64_t)p.B * p.Hkv;
    const int dv = q8_padded_dim(p.D);
    // workgroups of eight wavefronts where they fill the chip, of four otherwise
    plan.waves = dv <= 128 && !p.mask && units * ((NC + 255) / 256) >= p.cus ? 8 : 4;
    const int cols = 32 * plan.waves;
    const int64_t groups = units * ((NC + cols - 1) / cols);
    const int64_t target = (plan.waves == 8 || dv > 128 ? 1 : 2) * (int64_t)p.cus;
    int64_t seen = p.Skv;
    if (p.window > 0) seen = std::min<int64_t>(seen, p.window + p.Sq - 1);
    plan.min_chunk = 256;
    int64_t ns = std::min(target / std::max<int64_t>(groups, 1), (seen + plan.min_chunk - 1) / plan.min_chunk);
    plan.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(ns, 256));
    plan.bytes = plan.nsplit > 1 ? (size_t)units * plan.nsplit * NC * (dv + 2) * sizeof(float) : 0;
    return plan;
}

template <int DV, int TERMS, int FMT, int WAVES, bool MASK>
static int launch_prefill_waves(const Q8AttnParams &p, hipStream_t stream) {
    const int64_t NC = (int64_t)p.G * p.Sq, blocks = (NC + 32 * WAVES - 1) / (32 * WAVES);
    hipLaunchKernelGGL((q8_prefill_kernel<DV, TERMS, FMT, WAVES, MASK>), dim3((unsigned)((int64_t)p.B * p.Hkv * blocks * p.nsplit)), dim3(64 * WAVES), 0,
                       stream, p);
    FHIP_HIP_CHECK(hipGetLastError());
    return p.nsplit > 1 ? launch_q8_merge(p, stream) : FHIP_OK;
}
template <int DV, int TERMS, int FMT>
static int launch_prefill_dims(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream) {
    if (p.mask) return launch_prefill_waves<DV, TERMS, FMT, 4, true>(p, stream);
    if constexpr (DV <= 128)
        if (plan.waves == 8) return launch_prefill_waves<DV, TERMS, FMT, 8, false>(p, stream);
    return launch_prefill_waves<DV, TERMS, FMT, 4, false>(p, stream);
}
template <int DV>
static int launch_prefill_types(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream) {
    if (p.q_dtype == FHIP_F32)
        return p.format == FHIP_Q8_INT8 ? launch_prefill_dims<DV, 2, FHIP_Q8_INT8>(p, plan, stream)
                                        : launch_prefill_dims<DV, 2, FHIP_Q8_E4M3>(p, plan, stream);
    return p.format == FHIP_Q8_INT8 ? launch_prefill_dims<DV, 1, FHIP_Q8_INT8>(p, plan, stream)
                                    : launch_prefill_dims<DV, 1, FHIP_Q8_E4M3>(p, plan, stream);
}
int launch_q8_prefill(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream) {
    switch (q8_padded_dim(p.D)) {
        case 64: return launch_prefill_types<64>(p, plan, stream);
        case 128: return launch_prefill_types<128>(p, plan, stream);
        case 192: return launch_prefill_types<192>(p, plan, stream);
        default: return launch_prefill_types<256>(p, plan, stream);
    }
}

}  // namespace fhip
