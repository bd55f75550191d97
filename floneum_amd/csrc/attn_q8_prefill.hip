// Attention over the 8-bit cache for many query rows: tiles of 64 keys, widened to f16 once per workgroup on their way into LDS.
//
// A workgroup of WAVES wavefronts serves 32 * WAVES columns ((query row, head of the group) pairs of one KV head: heads of a group share the
// tile, and a causal mask cuts columns of few rows); a wavefront has 32 of them on v_mfma_f32_32x32x16_f16:
//   S^T[key][column] = K Q^T     K in LDS by rows, Q in registers
//   O^T[dim][column] += V^T P^T  V in LDS transposed, eight keys of a dim to 16 bytes, in the order in which the scores' registers hold the keys
// so that probabilities go from the scores' registers to the operand's without leaving their lane.  A lane holds 16 keys of each half of the tile;
// their scales lie in one register of 16 lanes (a DPP row) and are broadcast by the multiplication that uses them.
//
// A tile costs a wavefront of 128 dims 32 products of 32 cycles and about 330 vector instructions, 32 of them exp2.  Both units are kept busy by one
// wavefront: the next tile's scores are multiplied while this one's weights are made, this tile's values while the next one's scores are scaled and
// the tile after them is widened into LDS.  The order is written down step by step (sched_barrier): left to itself the compiler puts the products
// of a tile behind each other, each waiting for its piece of LDS (695 us against 660 for the prompt below).
// Measured: 620 to 660 us, box to box, for a causal prompt of 8192 f16 rows, 32 / 8 heads of 128, int8 (830 to 890 TFLOP/s of visible pairs; the
// matrix units are busy for 37 % of the cycles, the vector units for 57 %); 156 us for 4 chunks of 512 bf16 rows over a window of 4096, e4m3; 68 us for
// 129 f32 rows on 8003 keys, whose queries of two terms fill the registers.  Mask tensors walk all keys and spill at 128 dims: 299 us for 2048 f16 rows
// under a causal one, against 75 under the analytic mask.
//
// Numbers are brought to f16 as in the kernel for few rows (attn_q8_decode.hip): codes exactly, a column's q scaled by a power of two, one term for
// 16-bit queries and two for f32.  The values' scales go with the probabilities, brought below 2^15 by a power of two E that follows the largest
// scale met: w_j = p_j vs_j 2^(15 - E), out = 2^(E - 15) sum w_j c_j / sum p_j.  16-bit tensors' w is rounded to 11 bits, one term: the output's own rounding
// is as large (error against 64 bits 2.9e-4 in f16 where f32 weights leave 2.0e-4, 1.7e-3 either way in bf16), and a second term would double the
// values' products.
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

template <int DV, int TERMS, int FMT, int WAVES, bool MASK>
__global__ __launch_bounds__(64 * WAVES, DV <= 128 ? 2 : 1) void q8_prefill_kernel(Q8AttnParams p) {
    request_arguments<Q8AttnParams>();
    // 16-bit queries: a column's reference is at most 2^SLACK behind its maximum, so that sums shrink once in many tiles (666 -> 649 us for a prompt
    // of 8192); half a step of the smallest weights is 2^-35 of the largest scale.  f32 takes none of it.
    constexpr int SLACK = TERMS == 1 ? 4 : 0;
    // pieces of LDS in flight: two ahead of their products, one for f32, whose registers are full (71 us against 73)
    constexpr int RG = TERMS == 1 ? 3 : 2;
    constexpr int COLS = 32 * WAVES, STEPS = DV / 16, DT = DV / 32, UNITS = DV / 16;
    // LDS: K [key][dim], V [dim][key]; a row's last 16 bytes are left over, so that 16 rows' pieces lie in different banks and every piece is at a
    // constant distance from the lane's first
    constexpr int KP = DV + 8, VP = Q8_TILE + 8;
    __shared__ __attribute__((aligned(16))) half_t lds_k[2][Q8_TILE * KP];
    __shared__ __attribute__((aligned(16))) half_t lds_v[2][DV * VP];

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
    int shift = 0;
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
        } else {
            float x[STEPS][8], top = 0.0f;
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                raw[i].widen(p, 16 * i + 8 * h, x[i]);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[i][e]));
            }
            shift = q8_query_shift(fmaxf(top, xor32(top)));
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    half_t high, low;
                    q8_query_terms<TERMS>(p, x[i][e], shift, high, low);
                    q[0][i][e] = high;
                    if constexpr (TERMS == 2) q[1][i][e] = low;
                }
        }
    }
    // Products of codes and queries, below 2^33, are multiplied by the keys' scales (2^-100 to 2^121) first and by the column's factor afterwards: 2^-26 of it
    // goes with the former, so that no product of finite numbers passes f32's range, or as much as the wavefront's largest factor leaves room for
    const int ahead = min(26, 126 - __builtin_amdgcn_readfirstlane(wave_reduce_i(q8_score_exponent(p, shift), [](int x, int y) { return x > y ? x : y; })));
    const float colscale = q8_score_scale(p, shift - ahead), down = __builtin_ldexpf(1.0f, -ahead);
    const int64_t at = vis.pos0 + row;
    const int limit = (int)(p.causal ? max((int64_t)0, min((int64_t)hi, at + 1)) : hi);
    const int start = (int)(p.window > 0 ? min((int64_t)hi, max((int64_t)0, at - p.window + 1)) : 0);

    const int64_t mask_row = (p.mask_kind == FHIP_MASK_QK ? row : b) * p.ms0;
    float16_t acc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[t][r] = 0.0f;
    // the column's reference, from which its weights are counted (never -infinity: a row without a key has no weights, but no difference of infinities
    // either), their sum, and the largest exponent of the values' scales (of the wavefront)
    float m = -3.402823466e38f, l = 0.0f;
    int E = -200;

    const uint8_t *const kbase = p.k.codes + (int64_t)b * p.k.cs[0] + (int64_t)kvh * p.k.cs[1];
    const uint8_t *const vbase = p.v.codes + (int64_t)b * p.v.cs[0] + (int64_t)kvh * p.v.cs[1];
    const float *const kscale = p.k.scales + (int64_t)b * p.k.ss[0] + (int64_t)kvh * p.k.ss[1];
    const float *const vscale = p.v.scales + (int64_t)b * p.v.ss[0] + (int64_t)kvh * p.v.ss[1];
    const int pitch = (p.D + 15) & ~15;
    const uint32_t krow = (uint32_t)p.k.cs[2], vrow = (uint32_t)p.v.cs[2];

    // Staging: pieces of 16 bytes of the keys, 4 keys x 4 dims of the values.  Where a tile has fewer of them than there are lanes, the first half
    // of the lanes moves keys, the second values.
    constexpr int LANES = 64 * WAVES, PIECES = 4 * DV, KN = (PIECES + LANES - 1) / LANES;
    const bool moves_k = PIECES >= LANES || wave < WAVES / 2, moves_v = PIECES >= LANES || wave >= WAVES / 2;
    const int sid = PIECES >= LANES ? threadIdx.x : threadIdx.x % PIECES;
    // of the values a wavefront takes 8 groups of keys by 8 of dims, which meet few banks
    auto value_group = [](int u) { return 8 * ((u >> 6) & 1) + (u >> 3 & 7); };
    auto value_dims = [](int u) { return 8 * (u >> 7) + (u & 7); };
    uint4_t ksrc[KN];
    uint32_t vsrc[KN][4];
    // Rows beyond the share are loaded as its last one (what lies there may be anything, 8-bit NaN among it); pieces beyond a row from its start:
    // q is 0 there, and such dims of v are not written.
    auto load_keys = [&](int at) {
        const int k0 = min(at, hi - 1);
        const uint32_t last = min(hi - 1 - k0, Q8_TILE - 1);
        if (!moves_k) return;
        const uint8_t *const r = kbase + (int64_t)k0 * krow;
#pragma unroll
        for (int i = 0; i < KN; i++) {
            const int u = sid + LANES * i, off = 16 * (u % UNITS);
            ksrc[i] = *(const uint4_t *)(r + (min((uint32_t)(u / UNITS) * krow, last * krow) + (off < pitch ? off : 0)));
        }
    };
    auto load_values = [&](int at) {
        const int k0 = min(at, hi - 1);
        const uint32_t last = min(hi - 1 - k0, Q8_TILE - 1);
        if (!moves_v) return;
        const uint8_t *const r = vbase + (int64_t)k0 * vrow;
#pragma unroll
        for (int i = 0; i < KN; i++) {
            const int u = sid + LANES * i, off = 4 * value_dims(u);
            const uint32_t o = off < pitch ? off : 0, at0 = 4 * value_group(u) * vrow;
#pragma unroll
            for (int e = 0; e < 4; e++) vsrc[i][e] = *(const uint32_t *)(r + (min(at0 + e * vrow, last * vrow) + o));
        }
    };
    auto store_keys = [&](int buf) {
        if (!moves_k) return;
#pragma unroll
        for (int i = 0; i < KN; i++) {
            const int u = sid + LANES * i, key = u / UNITS, chunk = 2 * (u % UNITS);
#pragma unroll
            for (int e = 0; e < 2; e++)
                *(half8_t *)&lds_k[buf][key * KP + 8 * (chunk + e)] =
                    q8_widen8_pairs(q8_pair_low<FMT>(ksrc[i][2 * e]), q8_pair_high<FMT>(ksrc[i][2 * e]), q8_pair_low<FMT>(ksrc[i][2 * e + 1]),
                                    q8_pair_high<FMT>(ksrc[i][2 * e + 1]));
        }
    };
    auto store_values = [&](int buf) {
        if (!moves_v) return;
#pragma unroll
        for (int i = 0; i < KN; i++) {
            const int u = sid + LANES * i, g = value_group(u), dim = 4 * value_dims(u), chunk = 2 * (g >> 2) + (g & 1), part = (g >> 1) & 1;
            half2_t x[4][2];  // [dim][pair of keys]
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t a = vsrc[i][2 * e], c2 = vsrc[i][2 * e + 1];
                const uint32_t t01 = __builtin_amdgcn_perm(c2, a, 0x05010400u), t23 = __builtin_amdgcn_perm(c2, a, 0x07030602u);
                x[0][e] = q8_pair_low<FMT>(t01), x[1][e] = q8_pair_high<FMT>(t01);
                x[2][e] = q8_pair_low<FMT>(t23), x[3][e] = q8_pair_high<FMT>(t23);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) *(half4_t *)&lds_v[buf][(dim + t) * VP + 8 * chunk + 4 * part] = half4_t{x[t][0][0], x[t][0][1], x[t][1][0], x[t][1][1]};
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

    // A tile's steps: its scores; scores times the keys' scales, masked, and their largest; weights; values.  Matrix products of a tile are STEPS2
    // pieces read from LDS, of the keys (S) and again of the values (V).
    constexpr int STEPS2 = DV / 8;
    float16_t s[2], next[2];
    half8_t piece[RG];
    float kf[2], vf[2], nf[2];  // scales of the keys and values of the next tile (nf), and of this one's values (vf)
    float top;
    int e = E;
    auto read_key = [&](int buf, auto ic) {
        constexpr int i = decltype(ic)::value;
        piece[i % RG] = *(const half8_t *)&lds_k[buf][(32 * (i % 2) + n) * KP + 8 * (i / 2 * 2 + h)];
    };
    auto read_value = [&](int buf, auto ic) {
        constexpr int i = decltype(ic)::value;
        piece[(STEPS2 + i) % RG] = *(const half8_t *)&lds_v[buf][(32 * (i % DT) + n) * VP + 8 * (i / DT * 2 + h)];
    };
    auto score = [&](auto ic) {
        constexpr int i = decltype(ic)::value, u = i % 2;
        if constexpr (i < 2)
#pragma unroll
            for (int r = 0; r < 16; r++) next[u][r] = 0.0f;
#pragma unroll
        for (int x = TERMS - 1; x >= 0; x--) next[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(piece[i % RG], q[x][i / 2], next[u], 0, 0, 0);
    };
    auto take_scales = [&]() {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            // what is no number among the values' scales goes by way of the scores, where rows that a mask hides are taken out
            kf[u] = __builtin_fmaf(vs[u], 0.0f, ks[u] * down), nf[u] = vs[u] < INFINITY ? vs[u] : 0.0f;
            e = max(e, nf[u] > 0.0f ? __builtin_amdgcn_frexp_expf(nf[u]) : -200);
        }
    };
    // score i (of 32) times its key's scale; with a mask in the log2 domain, else before the column's scale (which is positive)
    auto scaled = [&](int k0, auto ic) {
        constexpr int i = decltype(ic)::value, u = i / 16, r = i % 16;
        const int key = 32 * u + 8 * (r / 4) + r % 4;
        float t = row_lane<r>(kf[u]) * next[u][r];
        if constexpr (MASK) {
            float add = -INFINITY;
            if (key < limit - k0 - 4 * h) add = q8_load_any(p.mask, mask_row + (k0 + key + 4 * h) * p.ms1, p.q_dtype);
            t = add == -INFINITY ? -INFINITY : q8_with_mask(t * colscale, add * Q8_LOG2E);
        }
        s[u][r] = t;
    };
    // what the column does not see, and the largest score
    auto largest = [&](int k0) {
        if (!MASK && __builtin_amdgcn_ballot_w64(k0 + Q8_TILE > limit || k0 < start) != 0) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = 32 * u + 8 * (r / 4) + r % 4;
                    if (key >= limit - k0 - 4 * h || key < start - k0 - 4 * h) s[u][r] = -INFINITY;
                }
        }
        top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[u][r]);
    };
    const float g = MASK ? 1.0f : colscale;
    half8_t pw[TERMS][4];
    auto weight = [&](auto ic) {
        constexpr int i = decltype(ic)::value, u = i / 16, r = i % 16;
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], g, -m));
        l += x;
        float w = row_lane<r>(vf[u]) * x;
        if constexpr (TERMS == 2) asm("" : "+v"(w));  // (both terms from the same rounded w: the product is not contracted into them)
        const half_t high = (half_t)w;
        pw[0][2 * u + r / 8][r % 8] = high;
        if constexpr (TERMS == 2) pw[1][2 * u + r / 8][r % 8] = (half_t)(w - (float)high);
    };
    auto value = [&](auto ic) {
        constexpr int i = decltype(ic)::value, t = i % DT;
#pragma unroll
        for (int x = TERMS - 1; x >= 0; x--) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(piece[(STEPS2 + i) % RG], pw[x][i / DT], acc[t], 0, 0, 0);
    };
    // the part of 32 numbers that goes with step `i` of STEPS2
    auto portion = [&](auto ic, auto &&f) {
        constexpr int i = decltype(ic)::value, from = 32 * i / STEPS2, to = 32 * (i + 1) / STEPS2;
        q8_each<to - from>([&](auto j) { f(std::integral_constant<int, from + decltype(j)::value>()); });
    };
#define IC(n) std::integral_constant<int, n>()

    if (lo < hi) {
        load_keys(lo);
        load_values(lo);
        load_scales(lo);
        store_keys(0);
        store_values(0);
        take_scales();
        load_keys(lo + Q8_TILE);
        load_values(lo + Q8_TILE);
        load_scales(lo + Q8_TILE);
        lds_barrier();
        q8_each<STEPS2>([&](auto i) {
            read_key(0, i);
            score(i);
        });
        store_keys(1);
        load_keys(lo + 2 * Q8_TILE);
        q8_each<32>([&](auto i) { scaled(lo, i); });
        lds_barrier();
    }
    // the maximum and the scales' largest exponent follow; what was added so far shrinks with them
    auto settle = [&](int k0) {
        largest(k0);
        float grown = 1.0f;
        if (__builtin_amdgcn_ballot_w64(e > E) != 0) {
            e = __builtin_amdgcn_readfirstlane(wave_reduce_i(e, [](int x, int y) { return x > y ? x : y; }));
            grown = __builtin_ldexpf(1.0f, max(E - e, -1000)), E = e;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) vf[u] = __builtin_ldexpf(nf[u], 15 - SLACK - E);
        top = fmaxf(m, fmaxf(top, xor32(top)) * g);
        if (__builtin_amdgcn_ballot_w64(top > m + SLACK || grown != 1.0f) != 0) {
            const float shrink = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= shrink;
#pragma unroll
            for (int t = 0; t < DT; t++) acc[t] *= shrink * grown;
        }
    };
    int buf = 0, k0 = lo;
    for (; k0 + Q8_TILE < hi; k0 += Q8_TILE, buf ^= 1) {
        read_key(buf ^ 1, IC(0));
        if constexpr (RG == 3) read_key(buf ^ 1, IC(1));
        settle(k0);
        // the next tile's scores beside this one's weights
        q8_each<STEPS2>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            __builtin_amdgcn_sched_barrier(0);
            score(ic);
            if constexpr (i + RG - 1 < STEPS2) read_key(buf ^ 1, IC(i + RG - 1));
            else read_value(buf, IC(i + RG - 1 - STEPS2));
            portion(ic, weight);
        });
        // this tile's values beside the scaling of the next one's scores and the staging
        q8_each<STEPS2>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            __builtin_amdgcn_sched_barrier(0);
            value(ic);
            if constexpr (i + RG - 1 < STEPS2) read_value(buf, IC(i + RG - 1));
            if constexpr (i == 0) take_scales();
            if constexpr (!MASK) portion(ic, [&](auto j) { scaled(k0 + Q8_TILE, j); });
            if constexpr (i == 1) load_scales(k0 + 2 * Q8_TILE);
            if constexpr (i == 2) store_keys(buf);
            if constexpr (i == STEPS2 / 2 - 1) load_keys(k0 + 3 * Q8_TILE);
            if constexpr (i == STEPS2 / 2) store_values(buf ^ 1);
            if constexpr (i == STEPS2 - 2) load_values(k0 + 2 * Q8_TILE);
        });
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MASK) q8_each<32>([&](auto j) { scaled(k0 + Q8_TILE, j); });
        lds_barrier();
    }
    if (k0 < hi) {
        settle(k0);
        q8_each<32>(weight);
        q8_each<STEPS2>([&](auto i) {
            read_value(buf, i);
            value(i);
        });
    }
#undef IC
    l += xor32(l);
    if (c0 + wave * 32 + n >= NC) return;
    const float up = __builtin_ldexpf(1.0f, max(E, -140) - 15 + SLACK);
    const int64_t o = (int64_t)b * p.os[0] + (int64_t)head * p.os[1] + (int64_t)row * p.os[2];
    const int64_t part = ((int64_t)bg * p.nsplit + split) * NC + c;
    // (sum / l) 2^(E - 15): the quotient first, which stays in range (of a share without a key that the column sees: zeros, which count for nothing)
    const float inv = p.nsplit > 1 && l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * t + 2 * r + 4 * h;
            if (d >= p.D) continue;
            float4_t v = {acc[t][r], acc[t][r + 1], acc[t][r + 2], acc[t][r + 3]};
            v = v * inv * up;
            if (p.nsplit > 1) {
                *(float4_t *)(p.partials + part * DV + d) = v;
            } else {
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
    // Workgroups of eight wavefronts where they fill the chip, of four otherwise: a tile that is widened once serves twice the columns (us, eight and
    // four, f16, recorded calls: causal prompt of 8192 rows, 32/8 heads at 128, 621 and 654; 4 chunks of 512 on 4607 keys 173 and 188; 8 sequences of 65 rows on
    // 300, 32/32 heads, 19 and 36; below one round: 1000 causal rows 66 and 62, 1500 of 32/32 heads 58 and 49).  Where it does not pay: causal prompts of about
    // one round of workgroups, whose last rows set the time (2048 rows 74 and 65, 2300 83 and 74).
    plan.waves = dv <= 128 && !p.mask && units * ((NC + 255) / 256) >= p.cus ? 8 : 4;
    const int cols = 32 * plan.waves;
    const int64_t groups = units * ((NC + cols - 1) / cols);
    // as many workgroups as the chip holds at once (us, for one, two and three per CU, 129 causal rows on 8003 keys: 32/8 heads at 128, f16 52, 46, 50, f32 82, 69,
    // 80; 16/4 at 256, which a CU holds one of, 57, 66, 84; 200 on 4000 at 64 22, 24, 24)
    const int64_t target = (plan.waves == 8 || dv > 128 ? 1 : 2) * (int64_t)p.cus;
    int64_t seen = p.Skv;
    if (p.window > 0) seen = std::min<int64_t>(seen, p.window + p.Sq - 1);
    // (us, for shares of 64, 128, 256 and 512 keys at least, f16 at 128: 16 rows on 3000 keys, 32/8 heads, 18, 15, 16, 22, 40 on 1000 17, 16, 18, 24; calls of few
    // workgroups would take shorter ones, 64 rows on 500 keys of 4/2 heads at 64 10, 11, 13, 16)
    plan.min_chunk = 256;
    int64_t ns = std::min(target / std::max<int64_t>(groups, 1), (seen + plan.min_chunk - 1) / plan.min_chunk);
    plan.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(ns, 256));
    plan.bytes = plan.nsplit > 1 ? (size_t)units * plan.nsplit * NC * (dv + 2) * sizeof(float) : 0;
    return plan;
}

template <int DV, int TERMS, int FMT, int WAVES, bool MASK>
static int launch_prefill_waves(const Q8AttnParams &p, hipStream_t stream) {
    const int64_t NC = (int64_t)p.G * p.Sq, blocks = (NC + 32 * WAVES - 1) / (32 * WAVES);
    const int64_t workgroups = (int64_t)p.B * p.Hkv * blocks * p.nsplit;
    if (workgroups * 64 * WAVES > UINT32_MAX) {
        set_error("q8_attention: more query rows than a launch has lanes for");
        return FHIP_ERR_UNSUPPORTED;
    }
    hipLaunchKernelGGL((q8_prefill_kernel<DV, TERMS, FMT, WAVES, MASK>), dim3((unsigned)workgroups), dim3(64 * WAVES), 0, stream, p);
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
