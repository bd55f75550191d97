// Attention over the 8-bit cache for few query rows: every code is read from memory once and straight into the registers that feed the
// matrix cores; no LDS in the loop.
//
// A workgroup of four wavefronts serves 16 columns ((query row, head of the group) pairs of one KV head) over one share of
// the keys; a wavefront takes 32 keys a step.  S^T[key][column] = K Q^T and O^T[dim][column] += V^T P^T on v_mfma_f32_16x16x32_f16.
// Lane (n = lane % 16, g = lane / 16):
//   K operand  lane n of 16-key tile u holds key 8 (n / 4) + 4 u + n % 4, dims 64 s + 16 g .. + 15: one 16-byte load is two
//              operands, 64 consecutive bytes per row; the order of the dims does not matter as Q is laid out the same
//   scores     arrive in lane (column n, g), register r of tile u: key 8 g + 4 u + r, so that a lane has keys 8 g .. 8 g + 7
//   V operand  lane n holds head_dim / 16 consecutive dims of those same eight keys (4, 8 or 16 bytes a row: whole rows per 16 lanes);
//              the transposition to eight keys of one dim is byte permutes, which the widening needs anyway
// so probabilities go from the scores' registers to the operand's without leaving their lane.
//
// Codes are whole f16 numbers, so the products are exact up to the f32 accumulation.  A column's q is scaled by a power of two
// to f16's upper range: f16 and bf16 queries fit one term exactly (to 2^-29 of the row's largest element), f32 ones take two (22 bits).
// The value scale vs_j, in [2^(e_j - 1), 2^e_j), goes with the probability, which the sum of the weights takes without it: with the running maxima
// M of s_j and X of s_j - M + e_j,
//   p_j = 2^(s_j - M),  w_j = p_j vs_j 2^(15 - X) <= 2^15,  out = 2^(X - 15) sum w_j c_j / sum p_j
// which holds whatever the scales' range (a first token with values of almost nothing, rows of zeros beside large ones: X >= -99, the exponent of the
// least scale).  w is rounded to 11 bits (relative 2^-12, to 2^-29 of the largest) for 16-bit tensors, whose output is rounded as much once more (error
// against 64 bits 2.9e-4 in f16 where f32 weights leave 2.1e-4, 1.7e-3 either way in bf16), and taken as two terms for f32 (2.9e-7).
//
// Bound by the bytes of codes and scales where there are many: 156 us for 16 ragged sequences of up to 16384 keys, 32 heads of 96 (e4m3, 5.2 TB/s),
// 33.6 us with the joining for 16 of 4096, 8 KV heads of 128 (134 MB).  One sequence is bound by a chain of latencies: 10 us for 4096 keys, 8 of the
// main kernel and 3 of the joining where each stands alone (one kernel whose last workgroup joins the shares took 97 us: the order it needs
// between XCDs writes back and drops their L2).  Two steps of keys in flight without a branch, against one behind one: 58 -> 35 us for the 16
// sequences, with the joining by lanes side by side; non-temporal loads: no change.
#include <algorithm>

#include "q8.h"
#include "q8_attention.h"
#include "q8_device.h"

namespace fhip {

typedef float float2_at8_t __attribute__((ext_vector_type(2)));

template <int DV>
struct Q8Dims {
    static constexpr int VW = DV / 64;   // 32-bit words of V per lane and key
    static constexpr int KS = DV / 64;   // 16-byte pieces of K per lane and key
    static constexpr int TILES = DV / 16;
    // dim of row m of output tile 4 w + t
    static __device__ __forceinline__ int dim(int m, int w, int t) {
        if constexpr (DV == 64) return 4 * m + t;
        else if constexpr (DV == 128) return 8 * m + 4 * w + t;
        else if constexpr (DV == 192) return w < 2 ? 8 * m + 4 * w + t : 128 + 4 * m + t;
        else return 16 * m + 4 * w + t;
    }
};

__device__ __forceinline__ float quads_max(float x) {
    x = fmaxf(x, xor16(x));
    return fmaxf(x, xor32(x));
}
__device__ __forceinline__ float quads_sum(float x) {
    x += xor16(x);
    return x + xor32(x);
}
template <int DV, int TERMS, int FMT, bool MASK, bool BLOCKS>
__global__ __launch_bounds__(256, DV == 64 ? 3 : 2) void q8_decode_kernel(Q8AttnParams p) {
    request_arguments<Q8AttnParams>();
    using Dims = Q8Dims<DV>;
    constexpr int VW = Dims::VW, KS = Dims::KS, TILES = Dims::TILES, COLS = 16, NBUF = DV <= 128 ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float lds_acc[4][16][DV + 4];
    __shared__ float lds_m[4][COLS], lds_fit[4][COLS], lds_l[4][COLS];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int NC = p.G * p.Sq, blocks = (NC + COLS - 1) / COLS;
    const int split = blockIdx.x;
    const uint32_t unit = blockIdx.y + blockIdx.z * gridDim.y;
    const int bg = blocks == 1 ? unit : unit / blocks, cb = unit - bg * blocks, b = (uint32_t)bg / (uint32_t)p.Hkv, kvh = bg - b * p.Hkv;
    if (b >= p.B) return;
    const int c0 = cb * COLS, c1 = min(c0 + COLS, NC) - 1;

    const Q8Range vis = q8_visible(p, b, c0 / p.G, c1 / p.G);
    // this share of the keys
    const int len = vis.hi - vis.lo;
    const int chunk = (max(p.min_chunk, (int)(((uint32_t)len + p.nsplit - 1) / (uint32_t)p.nsplit)) + 127) / 128 * 128;
    const int64_t lo64 = vis.lo + (int64_t)split * chunk;
    const int lo = (int)min(lo64, (int64_t)vis.hi), hi = (int)min((int64_t)vis.hi, lo64 + chunk);

    float4_t acc[TILES];
    // the largest score so far (never -infinity), the largest of scores less that plus the exponents of the values' scales, 2^(15 - fit), the weights' sum
    float m = -3.402823466e38f, fit = -100.0f, lift = 0x1p115f, l = 0.0f;
#pragma unroll
    for (int t = 0; t < TILES; t++) acc[t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

    const uint8_t *const kbase = p.k.codes + (int64_t)b * p.k.cs[0] + (int64_t)kvh * p.k.cs[1];
    const uint8_t *const vbase = p.v.codes + (int64_t)b * p.v.cs[0] + (int64_t)kvh * p.v.cs[1];
    const float *const kscale = p.k.scales + (int64_t)b * p.k.ss[0] + (int64_t)kvh * p.k.ss[1];
    const float *const vscale = p.v.scales + (int64_t)b * p.v.ss[0] + (int64_t)kvh * p.v.ss[1];
    const int pitch = (p.D + 15) & ~15;
    const int krow = (int)p.k.cs[2], vrow = (int)p.v.cs[2];  // below 2^26
    // byte offsets of the lane's pieces in a row; pieces beyond the row are loaded from its start: q is 0 there, such dims of v are not written
    const int klast = 64 * (KS - 1) + 16 * g < pitch ? 64 * (KS - 1) + 16 * g : 0;
    const int voff = (VW == 3 ? 8 : 4 * VW) * n < pitch ? (VW == 3 ? 8 : 4 * VW) * n : 0, vlast = 128 + 4 * n < pitch ? 128 + 4 * n : 0;
    const int kkey = 8 * (n >> 2) + (n & 3), vkey = 8 * g;  // the lane's first key of a step

    // queries: column c is row c / G, head c % G of the group
    half8_t q[TERMS][KS][2];
    float colscale;
    bool tiny, vast;  // a column's factor that alone would end beyond f32's normal range: 2^64 of it, or 2^-64, go with the keys' scales
    int limit, start;  // keys [start, limit) of the column
    int row;
    // What a wavefront holds of a step's keys.  Steps are loaded NBUF ahead, without a branch (behind one the compiler would wait for all
    // loads): the last step of a share starts 32 keys before its end and leaves out those of the step before, and steps beyond it load that
    // one again.  A tensor has at least 32 rows here.
    struct Step {
        uint4_t kc[2][KS];
        uint32_t vc[8][VW];
        float ks[8], vs[8];
    };
    const uint32_t klane = (uint32_t)(kkey * krow), vlane = (uint32_t)(vkey * vrow);
    auto first_key = [&](int k0) { return max(0, min(k0, hi - 32)); };
    auto load_k = [&](Step &x, int k0) {
        const uint8_t *r = kbase + (int64_t)first_key(k0) * krow;
#pragma unroll
        for (int u = 0; u < 2; u++, r += 4 * krow)
#pragma unroll
            for (int s = 0; s < KS; s++)
                x.kc[u][s] = *(const uint4_t *)((r + (klane + (s == KS - 1 ? klast : 64 * s + 16 * g))));
    };
    auto load_v = [&](Step &x, int k0) {
        const uint8_t *r = vbase + (int64_t)first_key(k0) * vrow;
#pragma unroll
        for (int i = 0; i < 8; i++, r += vrow) {
            if constexpr (VW == 1) {
                x.vc[i][0] = *(const uint32_t *)((r + (vlane + voff)));
            } else if constexpr (VW == 4) {
                const uint4_t w = *(const uint4_t *)((r + (vlane + voff)));
#pragma unroll
                for (int e = 0; e < 4; e++) x.vc[i][e] = w[e];
            } else {
                const uint2_t w = *(const uint2_t *)((r + (vlane + voff)));
                x.vc[i][0] = w[0], x.vc[i][1] = w[1];
                if constexpr (VW == 3) x.vc[i][2] = *(const uint32_t *)((r + (vlane + vlast)));
            }
        }
    };
    // scales of the lane's eight keys: one each, or with blocks of eight and more two at most
    auto load_scale8 = [&](float (&out)[8], const float *s, const Q8View &v, int k0) {
        const int at = v.first + first_key(k0) + vkey;
        if constexpr (BLOCKS) {
            out[0] = s[at >> v.log2_block], out[7] = s[(at + 7) >> v.log2_block];
        } else {
            typedef float float4_at4_t __attribute__((ext_vector_type(4), aligned(4)));
            const float4_at4_t a = *(const float4_at4_t *)(s + at), c = *(const float4_at4_t *)(s + at + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) out[i] = a[i], out[4 + i] = c[i];
        }
    };
    auto spread_scale8 = [&](float (&x)[8], const Q8View &v, int k0) {
        if constexpr (BLOCKS) {
            const int T = 1 << v.log2_block, phase = (v.first + first_key(k0) + vkey) & (T - 1);
            const float a = x[0], c = x[7];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = phase + i < T ? a : c;
        }
    };
    auto load_scales = [&](Step &x, int k0) {
        load_scale8(x.ks, kscale, p.k, k0);
        load_scale8(x.vs, vscale, p.v, k0);
    };

    // the step at k0, and the loads of the step that takes its registers next
    auto step = [&](Step &x, int k0) {
        const int at = first_key(k0), next = k0 + NBUF * 128;
        spread_scale8(x.ks, p.k, k0);
        spread_scale8(x.vs, p.v, k0);
        float exf[8], vs[8], ks[8];  // (exf: e_j)
        uint32_t top_scale = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) ks[i] = x.ks[i], vs[i] = x.vs[i], top_scale = max(top_scale, __float_as_uint(vs[i]));
        // What is no number among the values' scales (infinity and, as bits, all beyond it) goes by way of the scores, where rows that a mask hides are taken out
        if (__builtin_amdgcn_ballot_w64(tiny || vast || top_scale >= 0x7f800000u) != 0) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (tiny || vast) ks[i] *= tiny ? 0x1p-64f : 0x1p64f;
                if (__float_as_uint(vs[i]) >= 0x7f800000u) ks[i] = __uint_as_float(0x7fc00000u), vs[i] = 0.0f;
            }
        }
        // scores
        float sc[8];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float4_t s4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int a = 0; a < 2; a++) {
                    half8_t kf;
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const uint32_t word = x.kc[u][s][2 * a + w];
                        const half2_t y = q8_pair_low<FMT>(word), z = q8_pair_high<FMT>(word);
                        kf[4 * w] = y[0], kf[4 * w + 1] = y[1], kf[4 * w + 2] = z[0], kf[4 * w + 3] = z[1];
                    }
#pragma unroll
                    for (int t = TERMS - 1; t >= 0; t--)
                        s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[t][s][a], s4, 0, 0, 0);
                }
#pragma unroll
            for (int r = 0; r < 4; r++) sc[4 * u + r] = s4[r];
        }
        load_k(x, next);
#pragma unroll
        for (int i = 0; i < 8; i++) exf[i] = (float)__builtin_amdgcn_frexp_expf(fmaxf(vs[i], Q8_LEAST_SCALE));
        half8_t pw[TERMS];
        {
            float top = -INFINITY;
            if constexpr (!MASK) {
#pragma unroll
                for (int i = 0; i < 8; i++) sc[i] *= ks[i] * colscale;
                // the step reaches beyond what some column sees
                if (__builtin_amdgcn_ballot_w64(at + 32 > limit || at < start || at < k0) != 0) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int key = at + vkey + i;
                        if (key >= limit || key < start || key < k0) sc[i] = -INFINITY;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = at + vkey + i;
                    float add = -INFINITY;
                    if (key < limit && key >= k0)
                        add = q8_load_any(p.mask, (p.mask_kind == FHIP_MASK_QK ? row : b) * p.ms0 + key * p.ms1, p.q_dtype);
                    const float s = q8_with_mask(sc[i] * (ks[i] * colscale), add * Q8_LOG2E);
                    sc[i] = add == -INFINITY ? -INFINITY : s;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, sc[i]);
            top = fmaxf(m, quads_max(top));
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                sc[i] -= top;
                most = fmaxf(most, sc[i] + exf[i]);
            }
            most = fmaxf(fmaxf(fit + (m - top), -100.0f), quads_max(most));
            if (__builtin_amdgcn_ballot_w64(top > m || most > fit) != 0) {
                const float f = __builtin_amdgcn_exp2f((m - top) + (fit - most));
                l *= __builtin_amdgcn_exp2f(m - top);
                m = top, fit = most;
                lift = __builtin_amdgcn_exp2f(15.0f - fit);
#pragma unroll
                for (int t = 0; t < TILES; t++) acc[t] *= f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float e = __builtin_amdgcn_exp2f(sc[i]);
                l += e;
                float w = e * vs[i] * lift;
                if constexpr (TERMS == 2) asm("" : "+v"(w));  // (both terms from the same rounded w: the product is not contracted into them)
                const half_t hi16 = (half_t)w;
                pw[0][i] = hi16;
                if constexpr (TERMS == 2) pw[1][i] = (half_t)(w - (float)hi16);
            }
        }
        load_scales(x, next);
        // rows that are no keys of this step's may hold anything, 8-bit NaN among it
        if (at < k0 || at + 32 > hi) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (at + vkey + i < k0 || at + vkey + i >= hi)
#pragma unroll
                    for (int w = 0; w < VW; w++) x.vc[i][w] = 0;
        }
        // values: byte t of the eight keys' words w is dim(n, w, t)
#pragma unroll
        for (int w = 0; w < VW; w++) {
            half8_t vf[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t a = x.vc[2 * i][w], c = x.vc[2 * i + 1][w];
                const uint32_t t01 = __builtin_amdgcn_perm(c, a, 0x05010400u), t23 = __builtin_amdgcn_perm(c, a, 0x07030602u);
                const half2_t h0 = q8_pair_low<FMT>(t01), h1 = q8_pair_high<FMT>(t01), h2 = q8_pair_low<FMT>(t23), h3 = q8_pair_high<FMT>(t23);
                vf[0][2 * i] = h0[0], vf[0][2 * i + 1] = h0[1];
                vf[1][2 * i] = h1[0], vf[1][2 * i + 1] = h1[1];
                vf[2][2 * i] = h2[0], vf[2][2 * i + 1] = h2[1];
                vf[3][2 * i] = h3[0], vf[3][2 * i + 1] = h3[1];
            }
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int y = TERMS - 1; y >= 0; y--)
                    acc[4 * w + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[t], pw[y], acc[4 * w + t], 0, 0, 0);
        }
        load_v(x, next);
    };

    Q8Query8<TERMS> raw[KS][2];
    {
        const int c = min(c0 + n, NC - 1);
        row = c / p.G;
        const int64_t base = (int64_t)b * p.qs[0] + (int64_t)(kvh * p.G + c - row * p.G) * p.qs[1] + (int64_t)row * p.qs[2];
        if (p.q_vec) {
#pragma unroll
            for (int s = 0; s < 2 * KS; s++) raw[s >> 1][s & 1].load(p, base, 64 * (s >> 1) + 16 * g + 8 * (s & 1));
        } else {
#pragma unroll
            for (int s = 0; s < 2 * KS; s++) raw[s >> 1][s & 1].gather(p, base, 64 * (s >> 1) + 16 * g + 8 * (s & 1));
        }
    }
    Step steps[NBUF];
    int k0 = lo + 32 * wave;
    if (k0 < hi) {
#pragma unroll
        for (int i = 0; i < NBUF; i++) {
            load_k(steps[i], k0 + 128 * i);
            load_scales(steps[i], k0 + 128 * i);
            load_v(steps[i], k0 + 128 * i);
        }
    }
    {
        int shift = 0;
        if (TERMS == 1 && p.q_dtype == FHIP_F16 && p.scale != 0.0f) {  // as they are
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int a = 0; a < 2; a++) q[0][s][a] = raw[s][a].halves(p, 64 * s + 16 * g + 8 * a);
        } else {
            float x[KS][2][8], top = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int a = 0; a < 2; a++) {
                    raw[s][a].widen(p, 64 * s + 16 * g + 8 * a, x[s][a]);
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[s][a][e]));
                }
            shift = q8_query_shift(quads_max(top));
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int a = 0; a < 2; a++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        half_t high, low;
                        q8_query_terms<TERMS>(p, x[s][a][e], shift, high, low);
                        q[0][s][a][e] = high;
                        if constexpr (TERMS == 2) q[1][s][a][e] = low;
                    }
        }
        const int exponent = q8_score_exponent(p, shift);
        tiny = exponent < -75, vast = exponent > 100;
        colscale = q8_score_scale(p, shift - (tiny ? 64 : vast ? -64 : 0));
        const int64_t at = vis.pos0 + row;
        limit = (int)(p.causal ? max((int64_t)0, min((int64_t)hi, at + 1)) : hi);
        start = (int)(p.window > 0 ? min((int64_t)hi, max((int64_t)0, at - p.window + 1)) : 0);
    }

    while (k0 < hi) {
#pragma unroll
        for (int i = 0; i < NBUF; i++) {
            step(steps[i], k0);
            k0 += 128;
            if (i + 1 < NBUF && k0 >= hi) break;
        }
    }

    // the four wavefronts' states
    l = quads_sum(l);
    if (g == 0) lds_m[wave][n] = m, lds_fit[wave][n] = fit, lds_l[wave][n] = l;
    {
        lds_barrier();  // (the loads of steps beyond the last one may still be on their way)
#pragma unroll
        for (int w = 0; w < VW; w++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float4_t v = {acc[4 * w][r], acc[4 * w + 1][r], acc[4 * w + 2][r], acc[4 * w + 3][r]};
                *(float4_t *)&lds_acc[wave][n][Dims::dim(4 * g + r, w, 0)] = v;
            }
        lds_barrier();
        const int col = threadIdx.x >> 4, sub = threadIdx.x & 15, c = c0 + col;
        if (c < NC) {
            float M = -INFINITY, most = -INFINITY, L = 0.0f, f[4];
#pragma unroll
            for (int x = 0; x < 4; x++) M = fmaxf(M, lds_m[x][col]);
#pragma unroll
            for (int x = 0; x < 4; x++) {
                f[x] = lds_m[x][col] - M;
                L += lds_l[x][col] * __builtin_amdgcn_exp2f(f[x]);
                f[x] += lds_fit[x][col];
                most = fmaxf(most, f[x]);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) f[x] = __builtin_amdgcn_exp2f(f[x] - most);
            const int at = c / p.G;
            const int64_t o = (int64_t)b * p.os[0] + (int64_t)(kvh * p.G + c - at * p.G) * p.os[1] + (int64_t)at * p.os[2];
            const int64_t share = ((int64_t)bg * p.nsplit + split) * NC + c;
            // (of a share without a key that the column sees: zeros, which count for nothing)
            const float inv = p.nsplit > 1 && L == 0.0f ? 0.0f : 1.0f / L, up = __builtin_amdgcn_exp2f(most - 15.0f);
            for (int d = 4 * sub; d < p.D; d += 64) {
                float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < 4; x++) v += *(const float4_t *)&lds_acc[x][col][d] * f[x];
                v = v * inv * up;
                if (p.nsplit > 1) {
                    *(float4_t *)(p.partials + share * DV + d) = v;
                } else {
                    q8_store4_any(p, o + d * p.os[3], v);
                }
            }
            if (p.nsplit > 1 && sub == 0) {
                float *const ml = p.partials + (int64_t)p.B * p.Hkv * p.nsplit * NC * DV + share * 2;
                ml[0] = M, ml[1] = L;
            }
        }
    }
}

// Joins the shares of a (batch, kv head, column), which are means of their keys' values (sums of values near f32's end would pass it), by their parts of
// the weights' sum: groups of lanes, four dims a lane, add up every GROUPS-th share.  Bound by one memory latency after another, so up to 64 shares are
// requested at once: a lane's shares, and by every wavefront the shares' maxima and sums, one a lane, whose parts it keeps to itself.
template <int DV, bool FEW>
__global__ __launch_bounds__(256) void q8_merge_kernel(Q8AttnParams p) {
    request_arguments<Q8AttnParams>();
    constexpr int LPG = DV == 192 ? 64 : DV / 4, GROUPS = 256 / LPG, MOST = 64 / GROUPS;
    __shared__ float weight[FEW ? 4 * 64 : Q8_MAX_SHARES], red[8];
    __shared__ __attribute__((aligned(16))) float sums[GROUPS][4 * LPG];
    const int NC = p.G * p.Sq, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t at = blockIdx.x, bg = at / (uint32_t)NC;
    const int c = (int)(at - bg * NC);
    const float *const ml = p.partials + (int64_t)p.B * p.Hkv * p.nsplit * NC * DV;
    const int64_t first = (int64_t)bg * p.nsplit * NC + c, step = (int64_t)NC * DV;
    const int group = tid / LPG, d = 4 * (tid % LPG);
    const float *const part = p.partials + first * DV + (d < p.D ? d : 0);
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    // parts of the sum are counted in 16 times the power of two above the number of keys (weights of the many-row kernel reach 16), so that no sum of means
    // times parts is larger than a mean; their own sum, which takes two reductions more, is needed at the end only
    const float down = __builtin_ldexpf(1.0f, __builtin_clz(p.Skv) - 36);
    float L;
    if constexpr (FEW) {
        const float2_at8_t own = *(const float2_at8_t *)(ml + 2 * (first + (int64_t)min(lane, p.nsplit - 1) * NC));
        float4_t x[MOST];
#pragma unroll
        for (int i = 0; i < MOST; i++) x[i] = *(const float4_t *)(part + min(group + i * GROUPS, p.nsplit - 1) * step);
        const float M = wave_max(own[0]), ref = M == -INFINITY ? 0.0f : M;
        const float f = lane < p.nsplit ? own[1] * down * __builtin_amdgcn_exp2f(own[0] - ref) : 0.0f;
        weight[64 * wave + lane] = f;
        L = wave_sum(f);
        wave_lds_sync();
#pragma unroll
        for (int i = 0; i < MOST; i++)
            if (group + i * GROUPS < p.nsplit) v += x[i] * weight[64 * wave + group + i * GROUPS];
    } else {
        float m[Q8_MAX_SHARES / 256], l[Q8_MAX_SHARES / 256], M = -INFINITY;
#pragma unroll
        for (int i = 0; i < Q8_MAX_SHARES / 256; i++) {
            const int s = tid + 256 * i;
            m[i] = -INFINITY, l[i] = 0.0f;
            if (s < p.nsplit) m[i] = ml[2 * (first + (int64_t)s * NC)], l[i] = ml[2 * (first + (int64_t)s * NC) + 1];
            M = fmaxf(M, m[i]);
        }
        M = wave_max(M);
        if (lane == 0) red[wave] = M;
        __syncthreads();
        M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float ref = M == -INFINITY ? 0.0f : M;
        L = 0.0f;
#pragma unroll
        for (int i = 0; i < Q8_MAX_SHARES / 256; i++) {
            const float f = l[i] * down * __builtin_amdgcn_exp2f(m[i] - ref);
            if (tid + 256 * i < p.nsplit) weight[tid + 256 * i] = f;
            L += f;
        }
        L = wave_sum(L);
        if (lane == 0) red[4 + wave] = L;
        __syncthreads();
        L = (red[4] + red[5]) + (red[6] + red[7]);
#pragma unroll 4
        for (int s = group; s < p.nsplit; s += GROUPS) v += *(const float4_t *)(part + s * step) * weight[s];
    }
    *(float4_t *)&sums[group][d] = v;
    __syncthreads();
    if (tid >= LPG || d >= p.D) return;
#pragma unroll
    for (int g = 1; g < GROUPS; g++) v += *(const float4_t *)&sums[g][d];
    const int b = (int)(bg / p.Hkv), row = c / p.G, head = (int)(bg - b * p.Hkv) * p.G + c - row * p.G;
    q8_store4_any(p, (int64_t)b * p.os[0] + (int64_t)head * p.os[1] + (int64_t)row * p.os[2] + d * p.os[3], v * (1.0f / L));
}

static int q8_padded_dim(int D) { return (D + 63) / 64 * 64; }

template <int DV>
static void launch_merge_dims(const Q8AttnParams &p, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)p.B * p.H * p.Sq));
    if (p.nsplit <= 64) hipLaunchKernelGGL((q8_merge_kernel<DV, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((q8_merge_kernel<DV, false>), grid, dim3(256), 0, stream, p);
}
int launch_q8_merge(const Q8AttnParams &p, hipStream_t stream) {
    switch (q8_padded_dim(p.D)) {
        case 64: launch_merge_dims<64>(p, stream); break;
        case 128: launch_merge_dims<128>(p, stream); break;
        case 192: launch_merge_dims<192>(p, stream); break;
        default: launch_merge_dims<256>(p, stream);
    }
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

Q8AttnPlan q8_decode_plan(const Q8AttnParams &p) {
    Q8AttnPlan plan;
    const int NC = p.G * p.Sq;
    plan.prefill = false;
    plan.waves = 4;
    const int64_t units = (int64_t)p.B * p.Hkv * ((NC + 15) / 16);
    int64_t seen = p.Skv;
    if (p.window > 0) seen = std::min<int64_t>(seen, p.window + p.Sq - 1);
    // As many workgroups as the chip holds at once (us, for one, two, three and four per CU, recorded calls: 16 sequences of 4096 keys, 32/8 heads at 128,
    // f16, 28, 30, 34, 32; 3 of 14000 29, 28, 26, 28; 8 of 4001, 16/4 at 256, 22, 22, 32, 32); four times as many shorter shares where the sequences have
    // lengths of their own, which the host does not know: the long ones are spread (us, 16 of 128 to 16384 keys, 32/32 heads at 96: shares for 2, 4, 8 and
    // 16 workgroups per CU 209, 189, 175 and 188).
    const int64_t target = (p.kv_lens || p.q_positions ? 8 : 2) * (int64_t)p.cus;
    plan.min_chunk = 128;
    int64_t ns = std::min((target + units - 1) / units, (seen + 127) / 128);
    ns = std::max<int64_t>(1, std::min<int64_t>(ns, Q8_MAX_SHARES));
    plan.nsplit = (int)ns;
    plan.bytes = ns > 1 ? (size_t)p.B * p.Hkv * ns * NC * (q8_padded_dim(p.D) + 2) * sizeof(float) : 0;
    return plan;
}

template <int DV, int TERMS, int FMT>
static int launch_decode_dims(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream) {
    const int NC = p.G * p.Sq;
    const int64_t units = (int64_t)p.B * p.Hkv * ((NC + 15) / 16);
    const int64_t y = std::min<int64_t>(units, 32768), z = (units + y - 1) / y;
    const dim3 grid(p.nsplit, (unsigned)y, (unsigned)z);
    const bool blocks = p.k.log2_block > 0;
    if (p.mask && blocks) hipLaunchKernelGGL((q8_decode_kernel<DV, TERMS, FMT, true, true>), grid, dim3(256), 0, stream, p);
    else if (p.mask) hipLaunchKernelGGL((q8_decode_kernel<DV, TERMS, FMT, true, false>), grid, dim3(256), 0, stream, p);
    else if (blocks) hipLaunchKernelGGL((q8_decode_kernel<DV, TERMS, FMT, false, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((q8_decode_kernel<DV, TERMS, FMT, false, false>), grid, dim3(256), 0, stream, p);
    FHIP_HIP_CHECK(hipGetLastError());
    return p.nsplit > 1 ? launch_q8_merge(p, stream) : FHIP_OK;
}
template <int DV>
static int launch_decode_types(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream) {
    if (p.q_dtype == FHIP_F32)
        return p.format == FHIP_Q8_INT8 ? launch_decode_dims<DV, 2, FHIP_Q8_INT8>(p, plan, stream)
                                        : launch_decode_dims<DV, 2, FHIP_Q8_E4M3>(p, plan, stream);
    return p.format == FHIP_Q8_INT8 ? launch_decode_dims<DV, 1, FHIP_Q8_INT8>(p, plan, stream)
                                    : launch_decode_dims<DV, 1, FHIP_Q8_E4M3>(p, plan, stream);
}
int launch_q8_decode(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream) {
    switch (q8_padded_dim(p.D)) {
        case 64: return launch_decode_types<64>(p, plan, stream);
        case 128: return launch_decode_types<128>(p, plan, stream);
        case 192: return launch_decode_types<192>(p, plan, stream);
        default: return launch_decode_types<256>(p, plan, stream);
    }
}

}  // namespace fhip
