// Attention over the 8-bit cache for few query rows: every code is read from memory once and straight into the registers that feed the
// matrix cores; no LDS in the loop.
//
// A workgroup of four wavefronts serves CB blocks of 16 columns ((query row, head of the group) pairs of one KV head) over one share of
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
// The value scale vs_j, in [2^(e_j - 1), 2^e_j), goes with the probability: with the running maximum M of s_j + e_j,
//   p_j = 2^(s_j + e_j - M + 15) 2^-e_j,  w_j = p_j vs_j <= 2^15,  out = sum w_j c_j / sum p_j
// which holds whatever the scales' range (a first token with values of almost nothing).  w is rounded to 11 bits (relative 2^-12, to 2^-29 of the largest) for 16-bit tensors and
// taken as two terms for f32.
#include <algorithm>

#include "q8.h"
#include "q8_attention.h"
#include "q8_device.h"

namespace fhip {

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
template <int DV, int TERMS, int FMT, int CB>
__global__ __launch_bounds__(256, DV <= 128 ? 3 : 2) void q8_decode_kernel(Q8AttnParams p) {
    using Dims = Q8Dims<DV>;
    constexpr int VW = Dims::VW, KS = Dims::KS, TILES = Dims::TILES, COLS = 16 * CB;
    __shared__ __attribute__((aligned(16))) float lds_acc[4][16][DV + 4];
    __shared__ float lds_m[4][COLS], lds_l[4][COLS];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int NC = p.G * p.Sq, blocks = (NC + COLS - 1) / COLS;
    const int split = blockIdx.x;
    const uint32_t unit = blockIdx.y + blockIdx.z * gridDim.y;
    const int cb = unit % blocks;
    const int bg = unit / blocks, kvh = bg % p.Hkv, b = bg / p.Hkv;
    if (b >= p.B) return;
    const int c0 = cb * COLS, c1 = min(c0 + COLS, NC) - 1;

    const Q8Range vis = q8_visible(p, b, c0 / p.G, c1 / p.G);
    // this share of the keys
    const int len = vis.hi - vis.lo;
    const int chunk = (max(p.min_chunk, (int)(((int64_t)len + p.nsplit - 1) / p.nsplit)) + 127) / 128 * 128;
    const int64_t lo64 = vis.lo + (int64_t)split * chunk;
    const int lo = (int)min(lo64, (int64_t)vis.hi), hi = (int)min((int64_t)vis.hi, lo64 + chunk);

    // queries: column c is row c / G, head c % G of the group
    half8_t q[CB][TERMS][KS][2];
    float colscale[CB];
    int limit[CB], start[CB];  // keys [start, limit) of the column
    int row[CB];
#pragma unroll
    for (int cbk = 0; cbk < CB; cbk++) {
        const int c = min(c0 + cbk * 16 + n, NC - 1);
        row[cbk] = c / p.G;
        const int head = kvh * p.G + c % p.G;
        const int64_t base = (int64_t)b * p.qs[0] + (int64_t)head * p.qs[1] + (int64_t)row[cbk] * p.qs[2];
        float x[KS][16], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int d = 64 * s + 16 * g + e;
                x[s][e] = d < p.D ? q8_load_any(p.q, base + d * p.qs[3], p.q_dtype) : 0.0f;
                top = fmaxf(top, __builtin_fabsf(x[s][e]));
            }
        top = quads_max(top);
        // the largest element to [2^14, 2^15); zeros, infinities and NaN stay as they are
        const int shift = top > 0.0f && top <= 3.402823466e38f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float v = __builtin_ldexpf(x[s][e], shift);
                const half_t high = (half_t)v;
                q[cbk][0][s][e >> 3][e & 7] = high;
                if constexpr (TERMS == 2) q[cbk][1][s][e >> 3][e & 7] = (half_t)(v - (float)high);
            }
        colscale[cbk] = __builtin_ldexpf(p.scale * Q8_LOG2E, -shift);
        const int64_t at = vis.pos0 + row[cbk];
        limit[cbk] = (int)(p.causal ? max((int64_t)0, min((int64_t)hi, at + 1)) : hi);
        start[cbk] = (int)(p.window > 0 ? min((int64_t)hi, max((int64_t)0, at - p.window + 1)) : 0);
    }

    float4_t acc[CB][TILES];
    float m[CB], l[CB];
#pragma unroll
    for (int cbk = 0; cbk < CB; cbk++) {
        m[cbk] = -INFINITY, l[cbk] = 0.0f;
#pragma unroll
        for (int t = 0; t < TILES; t++) acc[cbk][t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

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

    uint4_t kc[2][KS];
    uint32_t vc[8][VW];
    float ks[8], vs[8];
    auto load_k_rows = [&](int u, const uint8_t *r, int at) {
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int off = s == KS - 1 ? klast : 64 * s + 16 * g;
            kc[u][s] = __builtin_nontemporal_load((const uint4_t *)(r + (uint32_t)(at + off)));
        }
    };
    auto load_v_rows = [&](int i, const uint8_t *r, int at) {
        if constexpr (VW == 1) {
            vc[i][0] = __builtin_nontemporal_load((const uint32_t *)(r + (uint32_t)(at + voff)));
        } else if constexpr (VW == 4) {
            const uint4_t w = __builtin_nontemporal_load((const uint4_t *)(r + (uint32_t)(at + voff)));
#pragma unroll
            for (int e = 0; e < 4; e++) vc[i][e] = w[e];
        } else {
            const uint2_t w = __builtin_nontemporal_load((const uint2_t *)(r + (uint32_t)(at + voff)));
            vc[i][0] = w[0], vc[i][1] = w[1];
            if constexpr (VW == 3) vc[i][2] = __builtin_nontemporal_load((const uint32_t *)(r + (uint32_t)(at + vlast)));
        }
    };
    // Keys beyond the share are loaded as its last one: what lies there may be anything, 8-bit NaN among it.
    auto load_k = [&](int k0) {
        const uint8_t *const r = kbase + (int64_t)k0 * krow;
        if (k0 + 32 <= hi) {
#pragma unroll
            for (int u = 0; u < 2; u++) load_k_rows(u, r + 4 * u * krow, kkey * krow);
        } else {
#pragma unroll
            for (int u = 0; u < 2; u++) load_k_rows(u, r, min(kkey + 4 * u, hi - 1 - k0) * krow);
        }
    };
    auto load_v = [&](int k0) {
        const uint8_t *const r = vbase + (int64_t)k0 * vrow;
        if (k0 + 32 <= hi) {
#pragma unroll
            for (int i = 0; i < 8; i++) load_v_rows(i, r + i * vrow, vkey * vrow);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) load_v_rows(i, r, min(vkey + i, hi - 1 - k0) * vrow);
        }
    };
    // scales of the lane's eight keys
    auto load_scales = [&](float (&out)[8], const float *s, const Q8View &v, int k0) {
        if (v.log2_block == 0) {
            if (k0 + 32 <= hi) {
                typedef float float4_at4_t __attribute__((ext_vector_type(4), aligned(4)));
                const float4_at4_t a = *(const float4_at4_t *)(s + k0 + vkey), c = *(const float4_at4_t *)(s + k0 + vkey + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) out[i] = a[i], out[4 + i] = c[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) out[i] = s[min(k0 + vkey + i, hi - 1)];
            }
        } else {  // blocks of 8 keys or more: two at most
            const int at = v.first + k0 + vkey, last = v.first + hi - 1, T = 1 << v.log2_block;
            const float a = s[min(at, last) >> v.log2_block], c = s[min(at + 7, last) >> v.log2_block];
            const int phase = at & (T - 1);
#pragma unroll
            for (int i = 0; i < 8; i++) out[i] = phase + i < T ? a : c;
        }
    };

    int k0 = lo + 32 * wave;
    if (k0 < hi) load_k(k0);
    for (; k0 < hi; k0 += 128) {
        load_scales(ks, kscale, p.k, k0);
        load_scales(vs, vscale, p.v, k0);
        load_v(k0);
        // NaN among the values' scales goes by way of the scores, where rows that a mask hides are taken out
        bool lost = false;
#pragma unroll
        for (int i = 0; i < 8; i += 2) lost = lost || __builtin_isunordered(vs[i], vs[i + 1]);
        if (__builtin_amdgcn_ballot_w64(lost) != 0) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (vs[i] != vs[i]) ks[i] = vs[i], vs[i] = 1.0f;
        }
        // scores
        float sc[CB][8];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float4_t s4[CB];
#pragma unroll
            for (int cbk = 0; cbk < CB; cbk++) s4[cbk] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int a = 0; a < 2; a++) {
                    half8_t kf;
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const uint32_t word = kc[u][s][2 * a + w];
                        const half2_t x = q8_pair_low<FMT>(word), y = q8_pair_high<FMT>(word);
                        kf[4 * w] = x[0], kf[4 * w + 1] = x[1], kf[4 * w + 2] = y[0], kf[4 * w + 3] = y[1];
                    }
#pragma unroll
                    for (int cbk = 0; cbk < CB; cbk++) {
#pragma unroll
                        for (int x = TERMS - 1; x >= 0; x--)
                            s4[cbk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[cbk][x][s][a], s4[cbk], 0, 0, 0);
                    }
                }
#pragma unroll
            for (int cbk = 0; cbk < CB; cbk++)
#pragma unroll
                for (int r = 0; r < 4; r++) sc[cbk][4 * u + r] = s4[cbk][r];
        }
        if (k0 + 128 < hi) load_k(k0 + 128);
        float exf[8], back[8];  // e_j, 2^-e_j
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int e = __builtin_amdgcn_frexp_expf(fmaxf(vs[i], Q8_LEAST_SCALE));
            exf[i] = (float)e;
            back[i] = __builtin_ldexpf(1.0f, -e);
        }
        half8_t pw[CB][TERMS];
#pragma unroll
        for (int cbk = 0; cbk < CB; cbk++) {
            float top = -INFINITY;
            if (p.mask == nullptr) {
#pragma unroll
                for (int i = 0; i < 8; i++) sc[cbk][i] = __builtin_fmaf(sc[cbk][i], ks[i] * colscale[cbk], exf[i]);
                // the step reaches beyond what some column sees
                if (__builtin_amdgcn_ballot_w64(k0 + 32 > limit[cbk] || k0 < start[cbk]) != 0) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int key = k0 + vkey + i;
                        if (key >= limit[cbk] || key < start[cbk]) sc[cbk][i] = -INFINITY;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = k0 + vkey + i;
                    float add = -INFINITY;
                    if (key < limit[cbk])
                        add = q8_load_any(p.mask, (p.mask_kind == FHIP_MASK_QK ? row[cbk] : b) * p.ms0 + key * p.ms1, p.q_dtype);
                    const float s = q8_with_mask(sc[cbk][i] * (ks[i] * colscale[cbk]), add * Q8_LOG2E);
                    sc[cbk][i] = add == -INFINITY ? -INFINITY : s + exf[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, sc[cbk][i]);
            top = fmaxf(m[cbk], quads_max(top));
            const float ref = top == -INFINITY ? 0.0f : top - 15.0f;
            if (__builtin_amdgcn_ballot_w64(top > m[cbk]) != 0) {
                const float f = __builtin_amdgcn_exp2f(m[cbk] - (top == -INFINITY ? 0.0f : top));
                m[cbk] = top;
                l[cbk] *= f;
#pragma unroll
                for (int t = 0; t < TILES; t++) acc[cbk][t] *= f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float e = __builtin_amdgcn_exp2f(sc[cbk][i] - ref) * back[i];
                l[cbk] += e;
                float w = e * vs[i];
                if constexpr (TERMS == 2) asm("" : "+v"(w));  // (both terms from the same rounded w: the product is not contracted into them)
                const half_t hi16 = (half_t)w;
                pw[cbk][0][i] = hi16;
                if constexpr (TERMS == 2) pw[cbk][1][i] = (half_t)(w - (float)hi16);
            }
        }
        // values: byte t of the eight keys' words w is dim(n, w, t)
#pragma unroll
        for (int w = 0; w < VW; w++) {
            half8_t vf[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t a = vc[2 * i][w], c = vc[2 * i + 1][w];
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
                for (int cbk = 0; cbk < CB; cbk++) {
                    float4_t &a = acc[cbk][4 * w + t];
#pragma unroll
                    for (int x = TERMS - 1; x >= 0; x--)
                        a = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[t], pw[cbk][x], a, 0, 0, 0);
                }
        }
    }

    // the four wavefronts' states, one column block at a time
#pragma unroll
    for (int cbk = 0; cbk < CB; cbk++) {
        l[cbk] = quads_sum(l[cbk]);
        if (g == 0) lds_m[wave][cbk * 16 + n] = m[cbk], lds_l[wave][cbk * 16 + n] = l[cbk];
    }
#pragma unroll
    for (int cbk = 0; cbk < CB; cbk++) {
        __syncthreads();
#pragma unroll
        for (int w = 0; w < VW; w++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float4_t v = {acc[cbk][4 * w][r], acc[cbk][4 * w + 1][r], acc[cbk][4 * w + 2][r], acc[cbk][4 * w + 3][r]};
                *(float4_t *)&lds_acc[wave][n][Dims::dim(4 * g + r, w, 0)] = v;
            }
        __syncthreads();
        const int col = threadIdx.x >> 4, sub = threadIdx.x & 15, c = c0 + cbk * 16 + col;
        if (c < NC) {
            float M = -INFINITY, L = 0.0f, f[4];
#pragma unroll
            for (int x = 0; x < 4; x++) M = fmaxf(M, lds_m[x][cbk * 16 + col]);
            const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                f[x] = __builtin_amdgcn_exp2f(lds_m[x][cbk * 16 + col] - ref);
                L += lds_l[x][cbk * 16 + col] * f[x];
            }
            const int head = kvh * p.G + c % p.G;
            const int64_t o = (int64_t)b * p.os[0] + (int64_t)head * p.os[1] + (int64_t)(c / p.G) * p.os[2];
            const int64_t share = ((int64_t)bg * p.nsplit + split) * NC + c;
            for (int d = 4 * sub; d < p.D; d += 64) {
                float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < 4; x++) v += *(const float4_t *)&lds_acc[x][col][d] * f[x];
                if (p.nsplit > 1) {
                    *(float4_t *)(p.partials + share * DV + d) = v;
                } else {
                    q8_store4_any(p, o + d * p.os[3], v / L);
                }
            }
            if (p.nsplit > 1 && sub == 0) {
                float *const ml = p.partials + (int64_t)p.B * p.Hkv * p.nsplit * NC * DV + share * 2;
                ml[0] = M, ml[1] = L;
            }
        }
    }
}

// Joins the shares: a wavefront per (batch, kv head, column), four dims a lane.
template <int DV>
__global__ __launch_bounds__(64) void q8_merge_kernel(Q8AttnParams p) {
    const int NC = p.G * p.Sq, lane = threadIdx.x;
    const int64_t at = blockIdx.x;
    const int c = (int)(at % NC);
    const int64_t bg = at / NC;
    const float *const ml = p.partials + (int64_t)p.B * p.Hkv * p.nsplit * NC * DV;
    float M = -INFINITY;
    for (int s = 0; s < p.nsplit; s++) M = fmaxf(M, ml[((bg * p.nsplit + s) * NC + c) * 2]);
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < p.nsplit; s++) {
        const int64_t i = (bg * p.nsplit + s) * NC + c;
        const float sm = ml[2 * i];
        if (sm == -INFINITY) continue;  // (NaN goes on)
        const float f = __builtin_amdgcn_exp2f(sm - ref);
        L += ml[2 * i + 1] * f;
        if (4 * lane < p.D) v += *(const float4_t *)(p.partials + i * DV + 4 * lane) * f;
    }
    if (4 * lane >= p.D) return;
    const int b = (int)(bg / p.Hkv), head = (int)(bg % p.Hkv) * p.G + c % p.G;
    const int64_t o = (int64_t)b * p.os[0] + (int64_t)head * p.os[1] + (int64_t)(c / p.G) * p.os[2];
    q8_store4_any(p, o + 4 * lane * p.os[3], v / L);
}

static int q8_padded_dim(int D) { return (D + 63) / 64 * 64; }

int launch_q8_merge(const Q8AttnParams &p, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)p.B * p.H * p.Sq));
    switch (q8_padded_dim(p.D)) {
        case 64: hipLaunchKernelGGL(q8_merge_kernel<64>, grid, dim3(64), 0, stream, p); break;
        case 128: hipLaunchKernelGGL(q8_merge_kernel<128>, grid, dim3(64), 0, stream, p); break;
        case 192: hipLaunchKernelGGL(q8_merge_kernel<192>, grid, dim3(64), 0, stream, p); break;
        default: hipLaunchKernelGGL(q8_merge_kernel<256>, grid, dim3(64), 0, stream, p);
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
    const int64_t target = 3 * (int64_t)p.cus;
    plan.min_chunk = 128;
    int64_t ns = std::min((target + units - 1) / units, (seen + 127) / 128);
    ns = std::max<int64_t>(1, std::min<int64_t>(ns, 1024));
    plan.nsplit = (int)ns;
    plan.bytes = ns > 1 ? (size_t)p.B * p.Hkv * ns * NC * (q8_padded_dim(p.D) + 2) * sizeof(float) : 0;
    return plan;
}

template <int DV, int TERMS, int FMT>
static int launch_decode_dims(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream) {
    const int NC = p.G * p.Sq;
    const int64_t units = (int64_t)p.B * p.Hkv * ((NC + 15) / 16);
    const int64_t y = std::min<int64_t>(units, 32768), z = (units + y - 1) / y;
    hipLaunchKernelGGL((q8_decode_kernel<DV, TERMS, FMT, 1>), dim3(p.nsplit, (unsigned)y, (unsigned)z), dim3(256), 0, stream, p);
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
