// Attention over a context in two parts for few query rows: every visible key and value is read once per column block, straight from memory
// into registers and from there through LDS to the matrix cores; what lies outside the columns' windows is not touched.
//
// Columns are (query row, head of the group) pairs that share a KV head.  A workgroup of four wavefronts serves 16 or 32 of them over one share of one
// part's visible keys, which are numbered without the gap between first tokens and window, a tile of 32 (f32, and above head_dim 128: 16) per wavefront
// and step:
//   own keys   columns of one sequence
//   prefix     columns of all sequences, so that the prefix is read once for the batch
// Both go in one launch, the prefix's workgroups first.
//   S^T[key][column] = K Q^T           v_mfma_f32_16x16x32 of the tensors' type, f32: v_mfma_f32_16x16x4_f32
//   p = exp2(s * scale * log2 e - m)   m the column's running maximum, l the running sum, O rescaled when some maximum moves
//   O^T[dim][column] += V^T P^T        P rounded to the tensors' type (f32: as it is), V^T by transposing LDS reads
// A column's state lives in the four lanes with its number modulo 16; wavefronts are joined in LDS, shares by context_merge_kernel.
//
// Bound, and measured with inputs larger than the caches:
//   many keys of their own   memory: 64 sequences of 4096 f16 keys of 32/8 heads at 128 stream 6.3 TB/s, 16 ragged ones 5.2, every byte once
//   a prefix                 the caches: 32 sequences on 8192 shared and up to 1024 own keys 31.6 us; memory reads 109 MB, each byte once, the column blocks take in 205:
//                            7.5 TB/s over the launch's 27.5 us, 10 while its one round of workgroups is whole (they live three quarters of it in the mean)
//   f32 columns              16 sequences on 4096 shared and 1500 own keys under a window 53 us: two rounds of workgroups, about 700 with keys on 512 places.  The
//                            matrix instructions hold a SIMD for 13 us of it, vector ones for 8; a wavefront waits 42 % of its time to issue and 31 % for memory and LDS
//   one sequence             two launches that depend on each other, a chain of latencies each: 1028 visible f32 keys 7.0 and 3.2 us
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "context_device.h"

namespace fhip {

constexpr int CR_WAVES = 4;
constexpr int CR_STREAMED = 2;         // past the caches: own keys, which are read once (16 ragged sequences, 259 MB: 51.0 us, 57.4 without); a prefix is
                                       // read once per block of columns (32 sequences on 8192 keys: 31.9 us, 35.4 streamed)
constexpr uint64_t CR_FAR = 1 << 25;   // bytes between rows up to which a tile's offsets stay in 31 bits
typedef uint32_t uint2r_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) char *lds_t;
#define CR_LDS(type, at) ((__attribute__((address_space(3))) type *)(at))

template <typename T>
struct RowsMma;
template <>
struct RowsMma<half_t> {
    typedef half8_t vec8;
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pack2(float x, float y) {
        const half2_t h = {(half_t)x, (half_t)y};
        return __builtin_bit_cast(uint32_t, h);
    }
};
template <>
struct RowsMma<bf16_t> {
    typedef bf16x8_t vec8;
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pack2(float x, float y) {
        typedef __bf16 bf16x2r_t __attribute__((ext_vector_type(2)));
        const bf16x2r_t h = {(__bf16)x, (__bf16)y};
        return __builtin_bit_cast(uint32_t, h);
    }
};

// max / sum over the four lanes of a column
__device__ __forceinline__ float column_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// bits of keys that some column of the 16 lanes sees
__device__ __forceinline__ uint32_t any_column(uint32_t x) {
    x |= (uint32_t)dpp_mov_i<DPP_QUAD_XOR1>((int)x);
    x |= (uint32_t)dpp_mov_i<DPP_QUAD_XOR2>((int)x);
    x |= (uint32_t)dpp_mov_i<DPP_ROW_HALF_MIRROR>((int)x);
    return x | (uint32_t)dpp_mov_i<DPP_ROW_MIRROR>((int)x);
}
// 16 lanes clear a row of BYTES in LDS
template <int BYTES>
__device__ __forceinline__ void clear_row(lds_t row, int lane) {
#pragma unroll
    for (int at = 0; at < BYTES; at += 256)
        if (at + 16 * lane < BYTES) *CR_LDS(uint4_t, row + at + 16 * lane) = uint4_t{0, 0, 0, 0};
}

// where a column's row of q, of the result and of the partials is
struct ColumnAt {
    int b, h, row;
};
__device__ __forceinline__ ColumnAt column_at(const ContextParams &p, int b, int g, int column) {
    const uint32_t each = (uint32_t)(p.G * p.Sq);
    if (b < 0) b = (int)((uint32_t)column / each), column -= b * (int)each;
    const int head = p.Sq == 1 ? column : (int)((uint32_t)column / (uint32_t)p.Sq);
    return {b, g * p.G + head, column - head * p.Sq};
}

// a workgroup's part of the call
struct RowsWork {
    bool none;
    bool prefix;
    int b, g;         // b < 0: columns of all sequences
    int c0, columns;  // first column, columns in use
    int slot, split, nsplit, chunk;
};
__device__ __forceinline__ RowsWork rows_work(const ContextParams &p, const ContextRows &rows) {
    const bool second = (int)blockIdx.x >= rows.second;
    const ContextRowsJob &job = rows.job[second];
    const uint32_t w = blockIdx.x - (second ? (uint32_t)rows.second : 0u), blocks = (uint32_t)job.blocks, nsplit = (uint32_t)job.nsplit;
    // workgroups are dealt to the 8 XCDs in turn: the column blocks that read the same keys share one, and its L2
    const uint32_t share = blocks == 1 ? w : w / (8 * blocks) * 8 + w % 8, block = blocks == 1 ? 0 : w / 8 % blocks;
    const uint32_t unit = nsplit == 1 ? share : share / nsplit;
    RowsWork r;
    r.none = unit >= (uint32_t)job.units;
    // (where sequences are short only the first shares have keys: they are spread over the XCDs as well)
    r.split = nsplit == 1 ? 0 : (int)((share - unit * nsplit + unit) % nsplit);
    r.slot = job.slot0 + r.split;
    r.nsplit = job.nsplit, r.chunk = job.chunk;
    r.prefix = job.prefix;
    const uint32_t b = unit / (uint32_t)p.Hkv;
    r.g = (int)(unit - b * p.Hkv);
    r.b = r.prefix ? -1 : (int)b;
    const int all = (r.prefix ? p.B : 1) * p.G * p.Sq;
    r.c0 = (int)block * rows.columns;
    r.columns = min(rows.columns, all - r.c0);
    return r;
}

// A share without keys: its sums are zero.
__device__ __forceinline__ void park_nothing(const ContextParams &p, const RowsWork &w) {
    if ((int)threadIdx.x >= w.columns) return;
    const ColumnAt at = column_at(p, w.b, w.g, w.c0 + threadIdx.x);
    float *ws = p.partials + ((((int64_t)at.b * p.H + at.h) * p.Sq + at.row) * p.slots + w.slot) * p.pf_pitch;
    ws[p.D] = -INFINITY;
    ws[p.D + 1] = 0.0f;
}

// Four dims of a column's result, or of its share.
template <typename T>
__device__ __forceinline__ void write_column(const ContextParams &p, const RowsWork &w, int column, int d, float m, float l, float4_t o) {
    const ColumnAt at = column_at(p, w.b, w.g, column);
    if (p.slots > 1) {
        float *ws = p.partials + ((((int64_t)at.b * p.H + at.h) * p.Sq + at.row) * p.slots + w.slot) * p.pf_pitch;
        *(float4_t *)(ws + d) = o;
        if (d == 0) ws[p.D] = m, ws[p.D + 1] = l;
        return;
    }
    const int64_t to = at.b * p.os[0] + at.h * p.os[1] + at.row * p.os[2] + d * p.os[3];
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] /= l;  // no visible key: 0 / 0 = NaN
    const bool f32 = sizeof(T) == 4 || p.out_f32;
    char *const out = (char *)p.out + to * (f32 ? 4 : 2);
    if (p.os[3] == 1 && ((uintptr_t)out & (f32 ? 15 : 7)) == 0) {
        if (f32) {
            *(float4_t *)out = o;
        } else if constexpr (sizeof(T) == 2) {
            const T four[4] = {from_float<T>(o[0]), from_float<T>(o[1]), from_float<T>(o[2]), from_float<T>(o[3])};
            uint2r_t bits;
            __builtin_memcpy(&bits, four, 8);
            *(uint2r_t *)out = bits;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (f32) ((float *)p.out)[to + e * p.os[3]] = o[e];
            else ((T *)p.out)[to + e * p.os[3]] = from_float<T>(o[e]);
        }
    }
}

// A wavefront's columns and their state.  Above head_dim 128 tiles of 16 keys leave room for a second workgroup on the CU (half of a second product's
// contraction is then zero: 32 sequences of up to 1024 keys of 16/4 heads at 192 take 17.6 us instead of 23.1).  DP: head_dim rounded up to a multiple of 32; Q is zero in the dims behind head_dim, and such dims of the result
// are not written.
// Rows that no column sees may hold anything, NaN among it, which 0 x NaN would bring into the result: in tiles with such rows their values are
// cleared in LDS.
template <typename T, int DP, int CB>
struct Columns {
    typedef typename RowsMma<T>::vec8 vec8;
    static constexpr int KEYS = DP > 128 ? 16 : 32, TB = KEYS / 16, E = 4 * TB;
    static constexpr int KP = DP * 2 + 16, VP = DP * 2 + 32;  // row pitches in LDS: 4 and 8 banks apart
    static constexpr int KB = DP / 32, NB = DP / 16;
    vec8 q[CB][KB];
    float4_t o[CB][NB];
    float m[CB], l[CB];
    ContextRow seen[CB];

    // Q^T operand: column j, dims 32 kb + 8 q4 .. + 7
    __device__ __forceinline__ void load_q(const ContextParams &p, int cb, const ColumnAt &at, bool used, int q4) {
        const uint16_t *from = (const uint16_t *)p.q + at.b * p.qs[0] + at.h * p.qs[1] + at.row * p.qs[2];
        const bool whole = p.qs[3] == 1 && ((uintptr_t)from & 15) == 0;
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            const int dim = 32 * kb + 8 * q4;
            uint4_t raw = {0, 0, 0, 0};
            if (used && dim < p.D) {
                if (whole) {
                    raw = *(const uint4_t *)(from + dim);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) raw[e >> 1] |= (uint32_t)from[(dim + e) * p.qs[3]] << ((e & 1) * 16);
                }
            }
            q[cb][kb] = __builtin_bit_cast(vec8, raw);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int cb = 0; cb < CB; cb++) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++) o[cb][nb] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            m[cb] = -INFINITY, l[cb] = 0.0f;
        }
    }
    // The tile of visible keys base .. in LDS; whole: every column sees all of it.
    __device__ __forceinline__ void step(lds_t k, lds_t v, int base, int end, int first, int gap, bool whole, float scale2, int lane) {
        const int j = lane & 15, q4 = lane >> 4;
        float4_t s[CB][TB];
#pragma unroll
        for (int t = 0; t < TB; t++) {
#pragma unroll
            for (int cb = 0; cb < CB; cb++) s[cb][t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                const uint4_t raw = *CR_LDS(uint4_t, k + (16 * t + j) * KP + (32 * kb + 8 * q4) * 2);
#pragma unroll
                for (int cb = 0; cb < CB; cb++) s[cb][t] = RowsMma<T>::mfma(__builtin_bit_cast(vec8, raw), q[cb][kb], s[cb][t]);
            }
        }
        vec8 weights[CB];
        uint32_t used = 0;  // the lane's keys that some column sees
#pragma unroll
        for (int cb = 0; cb < CB; cb++) {
            // element (t, r) is visible key base + 16 t + 4 q4 + r
            float x[E];
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = s[cb][e >> 2][e & 3] * scale2;
            if (!whole) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int n = base + 16 * (e >> 2) + 4 * q4 + (e & 3), key = n + (n >= first ? gap : 0);
                    const bool sees = n < end && key < seen[cb].hi && (key >= seen[cb].lo || key < seen[cb].first);
                    x[e] = sees ? x[e] : -INFINITY;
                    used |= sees ? 1u << e : 0u;
                }
            }
            float top = x[0];
#pragma unroll
            for (int e = 1; e < E; e++) top = fmaxf(top, x[e]);
            top = fmaxf(m[cb], column_max(top));
            if (__builtin_amdgcn_ballot_w64(top > m[cb]) != 0) {
                const float moved = __builtin_amdgcn_exp2f(m[cb] - (top == -INFINITY ? 0.0f : top));
                m[cb] = top;
                l[cb] *= moved;
#pragma unroll
                for (int nb = 0; nb < NB; nb++) o[cb][nb] *= moved;
            }
            const float reference = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                x[e] = __builtin_amdgcn_exp2f(x[e] - reference);
                sum += x[e];
            }
            l[cb] += sum;
            // P^T operand: slot (q4, e) is key 4 q4 + e, or 16 + 4 q4 + e - 4 from e = 4 on (of 16 keys: zero)
            uint4_t packed = {RowsMma<T>::pack2(x[0], x[1]), RowsMma<T>::pack2(x[2], x[3]), 0, 0};
            if constexpr (TB == 2) packed[2] = RowsMma<T>::pack2(x[4], x[5]), packed[3] = RowsMma<T>::pack2(x[6], x[7]);
            weights[cb] = __builtin_bit_cast(vec8, packed);
        }
        if (!whole) {
            used = any_column(used);
#pragma unroll
            for (int e = 0; e < E; e++)
                if (!(used >> e & 1)) clear_row<DP * 2>(v + (16 * (e >> 2) + 4 * q4 + (e & 3)) * VP, j);
            wave_lds_sync();
        }
        // the transposing load hands lane i of 16 V[row .. row + 3][dim + i]
        const lds_t v_at = v + (4 * q4 + (j >> 2)) * VP + 8 * (j & 3);
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const short4_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(CR_LDS(short4_t, v_at + nb * 32));
            uint2r_t u0 = __builtin_bit_cast(uint2r_t, a0), u1 = {0, 0};
            if constexpr (TB == 2) u1 = __builtin_bit_cast(uint2r_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(CR_LDS(short4_t, v_at + 16 * VP + nb * 32)));
            const vec8 values = __builtin_bit_cast(vec8, uint4_t{u0[0], u0[1], u1[0], u1[1]});
#pragma unroll
            for (int cb = 0; cb < CB; cb++) o[cb][nb] = RowsMma<T>::mfma(values, weights[cb], o[cb][nb]);
        }
    }
    // dims of column 16 cb + j to `to`, [DP], then the reference and the sum
    __device__ __forceinline__ void park(float *to, int cb, int q4) {
        const float sum = column_sum(l[cb]);
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int r = 0; r < 4; r++) to[16 * nb + 4 * q4 + r] = o[cb][nb][r];
        if (q4 == 0) to[DP] = m[cb], to[DP + 1] = sum;
    }
};

// The same for f32 tensors: 16 keys per tile.  Contraction slot (c, i, q4) of K Q^T is dim 16 c + 4 q4 + i, so that one 16-byte read of a row feeds
// four matrix steps; slot (i, q4) of V^T P^T is key 4 q4 + i, whose weight the lane already holds, and row n of output block (nb, e) is dim
// 16 VW nb + VW n + e, so that one read of a row feeds VW steps.  The tile's share of O forms on its own and is added once (one rounding at the
// size of the sum).
template <int DP>
struct Columns<float, DP, 1> {
    static constexpr int KEYS = 16;
    static constexpr int KP = DP * 4 + 16, VP = KP;
    static constexpr int KC = DP / 16, VW = DP % 64 == 0 ? 4 : 2, NB = DP / (16 * VW);
    typedef float vrow_t __attribute__((ext_vector_type(VW)));
    float4_t q[KC];
    float4_t o[NB][VW];
    float m, l;
    ContextRow seen[1];

    // Q^T operand: column j, dims 16 c + 4 q4 .. + 3
    __device__ __forceinline__ void load_q(const ContextParams &p, int cb, const ColumnAt &at, bool used, int q4) {
        const float *from = (const float *)p.q + at.b * p.qs[0] + at.h * p.qs[1] + at.row * p.qs[2];
        const bool whole = p.qs[3] == 1 && ((uintptr_t)from & 15) == 0;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const int dim = 16 * c + 4 * q4;
            q[c] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (used && dim < p.D) {
                if (whole) {
                    q[c] = *(const float4_t *)(from + dim);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) q[c][e] = from[(dim + e) * p.qs[3]];
                }
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < VW; e++) o[nb][e] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY, l = 0.0f;
    }
    __device__ __forceinline__ void step(lds_t k, lds_t v, int base, int end, int first, int gap, bool whole, float scale2, int lane) {
        const int j = lane & 15, q4 = lane >> 4;
        // (in four sums: a single one would add up four times the roundings)
        float4_t sums[4];
#pragma unroll
        for (int i = 0; i < 4; i++) sums[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const float4_t a = *CR_LDS(float4_t, k + j * KP + (16 * c + 4 * q4) * 4);
#pragma unroll
            for (int i = 0; i < 4; i++) sums[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], q[c][i], sums[i], 0, 0, 0);
        }
        const float4_t s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        float x[4];
        bool hidden[4] = {false, false, false, false};
        uint32_t used = 0;
        // element r is visible key base + 4 q4 + r
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = s[r] * scale2;
        if (!whole) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int n = base + 4 * q4 + r, key = n + (n >= first ? gap : 0);
                const bool sees = n < end && key < seen[0].hi && (key >= seen[0].lo || key < seen[0].first);
                x[r] = sees ? x[r] : -INFINITY;
                hidden[r] = !sees;
                used |= sees ? 1u << r : 0u;
            }
        }
        const float top = fmaxf(m, column_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))));
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
            const float moved = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
            m = top;
            l *= moved;
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int e = 0; e < VW; e++) o[nb][e] *= moved;
        }
        const float reference = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            // (one rounding, at the size of the difference; a hidden key's stays -infinity)
            const float d = __builtin_fmaf(s[r], scale2, -reference);
            x[r] = __builtin_amdgcn_exp2f(hidden[r] ? -INFINITY : d);
            sum += x[r];
        }
        l += sum;
        if (!whole) {
            used = any_column(used);
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (!(used >> r & 1)) clear_row<DP * 4>(v + (4 * q4 + r) * VP, j);
            wave_lds_sync();
        }
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            vrow_t a[4];
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = *CR_LDS(vrow_t, v + (4 * q4 + i) * VP + (16 * VW * nb + VW * j) * 4);
#pragma unroll
            for (int e = 0; e < VW; e++) {
                float4_t share = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 4; i++) share = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][e], x[i], share, 0, 0, 0);
                o[nb][e] += share;
            }
        }
    }
    __device__ __forceinline__ void park(float *to, int cb, int q4) {
        const float sum = column_sum(l);
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < VW; e++)
#pragma unroll
                for (int r = 0; r < 4; r++) to[16 * VW * nb + VW * (4 * q4 + r) + e] = o[nb][e][r];
        if (q4 == 0) to[DP] = m, to[DP + 1] = sum;
    }
};

// CB: blocks of 16 columns
template <typename T, int DP, int CB>
__global__ __launch_bounds__(64 * CR_WAVES, DP > 128 && sizeof(T) == 4 ? 1 : 2) void context_rows_kernel(ContextParams p, ContextRows rows) {
    request_arguments<ContextParams, ContextRows>();
    typedef Columns<T, DP, CB> C;
    constexpr int KEYS = C::KEYS, COLS = 16 * CB, ES = sizeof(T), STEP = CR_WAVES * KEYS;
    constexpr int PER = 16 / ES, CPR = DP / PER, LOADS = KEYS * CPR / 64;  // elements of a 16-byte piece, pieces of a row, loads per lane and tensor
    constexpr bool RUNS = 64 % CPR == 0;  // a load takes whole rows
    constexpr int WAVE_BYTES = KEYS * (C::KP + C::VP), STATE = DP + 2, STATE_BYTES = CR_WAVES * COLS * STATE * 4;
    __shared__ __attribute__((aligned(16))) char smem[CR_WAVES * WAVE_BYTES > STATE_BYTES ? CR_WAVES * WAVE_BYTES : STATE_BYTES];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, j = lane & 15, q4 = lane >> 4;
    const lds_t k_tile = (lds_t)smem + wave * WAVE_BYTES, v_tile = k_tile + KEYS * C::KP;
    const RowsWork w = rows_work(p, rows);
    if (w.none) return;

    // the lane's columns and what they see
    C columns;
    ContextSpan span = {0, 0, p.P};  // (of a prefix without a window: not asked of the sequences' positions, which are a memory latency away)
#pragma unroll
    for (int cb = 0; cb < CB; cb++) {
        const ColumnAt at = column_at(p, w.b, w.g, w.c0 + min(j + 16 * cb, w.columns - 1));
        columns.load_q(p, cb, at, j + 16 * cb < w.columns, q4);
        columns.seen[cb] = context_row(p, at.b, at.row).of(p, w.prefix);
        if (!(w.prefix && p.window == 0)) {
            const ContextSpan s = context_span(columns.seen[cb]);
            if (cb == 0) {
                span = s;
            } else {
                const int lo = s.keys() == 0 ? span.lo : span.keys() == 0 ? s.lo : min(span.lo, s.lo);
                span.hi = max(span.hi, s.hi), span.first = max(span.first, s.first), span.lo = max(lo, span.first);
            }
        }
    }
    // Shares of `chunk` keys, or where these do not hold all of them of the length that does, in whole steps.  (In 32 bits without a sign: the last share may begin
    // behind 2^31 keys.)
    const int first = span.first, gap = span.gap();
    const uint32_t keys = (uint32_t)span.keys();
    uint32_t chunk = (uint32_t)w.chunk;
    if (keys > chunk * (uint32_t)w.nsplit) chunk = ((keys + w.nsplit - 1) / w.nsplit + STEP - 1) / STEP * STEP;
    const int v_lo = (int)min(w.split * chunk, keys), v_hi = (int)min(w.split * chunk + chunk, keys);
    if (v_lo >= v_hi && p.slots > 1) {
        park_nothing(p, w);
        return;
    }
    bool alike = true;
#pragma unroll
    for (int cb = 0; cb < CB; cb++)
        alike = alike && columns.seen[cb].first >= first && columns.seen[cb].lo <= span.lo && columns.seen[cb].hi >= span.hi;
    alike = __builtin_amdgcn_ballot_w64(!alike) == 0;  // every column sees the whole share
    columns.clear();

    const T *const k = w.prefix ? (const T *)p.pk + w.g * p.pks[0] : (const T *)p.k + w.b * p.ks[0] + w.g * p.ks[1];
    const T *const v = w.prefix ? (const T *)p.pv + w.g * p.pvs[0] : (const T *)p.v + w.b * p.vs[0] + w.g * p.vs[1];
    const int64_t k_row = (w.prefix ? p.pks[1] : p.ks[2]) * ES, v_row = (w.prefix ? p.pvs[1] : p.vs[2]) * ES;  // bytes

    // The tile behind the one in LDS is on its way in registers.  A tile's rows are a buffer that starts at its first and ends with the share's last key:
    // what lies behind reads as zero, without a clamp or an address per lane.  Rows that a load does not
    // divide evenly, rows far apart and the one tile within which the first tokens end have an address per lane, with the last key again behind
    // it.  (With addresses alone 64 f32 columns on 2048 keys at head_dim 128 take 25.4 us instead of 22.9.)
    const int row = lane / CPR, col = lane % CPR;
    const bool inside = col * PER < p.D, far = (uint64_t)k_row > CR_FAR || (uint64_t)v_row > CR_FAR;
    const uint32_t k_at = inside ? row * (uint32_t)k_row + col * 16 : 0x7ffffff0u, v_at = inside ? row * (uint32_t)v_row + col * 16 : 0x7ffffff0u;
    constexpr int ROWS = 64 / CPR;  // of a load
    uint4_t kst[LOADS], vst[LOADS];
    auto load_tile = [&](int base) __attribute__((always_inline)) {
        if (!RUNS || far || (base < first && base + KEYS > first)) {
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const int piece = lane + 64 * u, x = min(base + piece / CPR, v_hi - 1), dim = piece % CPR * PER < p.D ? piece % CPR * PER : 0;
                const int64_t key = x + (x >= first ? gap : 0);
                kst[u] = __builtin_nontemporal_load((const uint4_t *)((const char *)(k + dim) + key * k_row));
                vst[u] = __builtin_nontemporal_load((const uint4_t *)((const char *)(v + dim) + key * v_row));
            }
        } else {
            const int64_t key = base + (base >= first ? gap : 0);
            const int left = min(v_hi - base, KEYS) - 1;
            auto rows_from = [&](const T *from, int64_t bytes) __attribute__((always_inline)) {
                const uint64_t at = (uint64_t)((const char *)from + key * bytes);
                const uint32_t low = __builtin_amdgcn_readfirstlane((int)(uint32_t)at), high = __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32));
                return __builtin_amdgcn_make_buffer_rsrc((void *)((uint64_t)high << 32 | low), 0, __builtin_amdgcn_readfirstlane(left * (int)bytes + p.D * ES),
                                                         0x00020000);
            };
            const auto k_rows = rows_from(k, k_row), v_rows = rows_from(v, v_row);
            auto pieces = [&](auto aux) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < LOADS; u++) {
                    kst[u] = __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(k_rows, k_at + u * ROWS * (uint32_t)k_row, 0, decltype(aux)::value));
                    vst[u] = __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(v_rows, v_at + u * ROWS * (uint32_t)v_row, 0, decltype(aux)::value));
                }
            };
            if (w.prefix) pieces(std::integral_constant<int, 0>{});
            else pieces(std::integral_constant<int, CR_STREAMED>{});
        }
    };
    const float scale2 = p.scale * CONTEXT_LOG2E;
    int base = v_lo + wave * KEYS;
    if (base < v_hi) load_tile(base);
    for (; base < v_hi; base += STEP) {
        // Pieces of K behind head_dim meet zeros of Q, and 0 x inf is NaN.  (Cleared here and not where they are loaded, which would wait for the load: 16 f32
        // sequences of 2005 visible keys at head_dim 136 42.6 us instead of 37.5.)
        if (p.D < DP) {
            asm volatile("");  // a branch
#pragma unroll
            for (int u = 0; u < LOADS; u++)
                if ((lane + 64 * u) % CPR * PER >= p.D) kst[u] = uint4_t{0, 0, 0, 0};
        }
        wave_lds_sync();  // the previous tile's reads precede these writes
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            const int piece = lane + 64 * u;
            *CR_LDS(uint4_t, k_tile + piece / CPR * C::KP + piece % CPR * 16) = kst[u];
            *CR_LDS(uint4_t, v_tile + piece / CPR * C::VP + piece % CPR * 16) = vst[u];
        }
        wave_lds_sync();
        if (base + STEP < v_hi) load_tile(base + STEP);
        columns.step(k_tile, v_tile, base, v_hi, first, gap, alike && base + KEYS <= v_hi, scale2, lane);
    }

    __syncthreads();  // the states take the tiles' place
    float *const states = (float *)smem;
#pragma unroll
    for (int cb = 0; cb < CB; cb++) columns.park(states + (wave * COLS + j + 16 * cb) * STATE, cb, q4);
    __syncthreads();
    const int pieces = p.D / 4;
    for (int i = threadIdx.x; i < w.columns * pieces; i += 64 * CR_WAVES) {
        const int column = i / pieces, d = 4 * (i - column * pieces);
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int x = 0; x < CR_WAVES; x++) m = fmaxf(m, states[(x * COLS + column) * STATE + DP]);
        const float reference = m == -INFINITY ? 0.0f : m;
        float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < CR_WAVES; x++) {
            const float *src = states + (x * COLS + column) * STATE;
            const float weight = __builtin_amdgcn_exp2f(src[DP] - reference);
            l += weight * src[DP + 1];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] += weight * src[d + e];
        }
        write_column<T>(p, w, w.c0 + column, d, m, l, o);
    }
}

// ---- shares ---------------------------------------------------------------------------------------------------------------------------
// LANES lanes take a row's dims, four each.  Where rows are few, GROUPS groups of them take parts of a row's shares, and the first folds the
// groups' states through LDS.
template <typename T, int LANES, int GROUPS>
__global__ __launch_bounds__(GROUPS > 1 ? LANES * GROUPS : 256) void context_merge_kernel(ContextParams p, int out_vec) {
    request_arguments<ContextParams, int>();
    constexpr int ROWS = GROUPS > 1 ? 1 : 256 / LANES, U = 8;
    __shared__ __attribute__((aligned(16))) float parts[GROUPS][GROUPS > 1 ? 4 * LANES : 4];
    __shared__ float states[GROUPS][2];
    const uint32_t row = GROUPS > 1 ? blockIdx.x : (blockIdx.y * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / LANES;
    if (GROUPS == 1 && row >= (uint32_t)(p.B * p.H * p.Sq)) return;
    const int group = GROUPS > 1 ? threadIdx.x / LANES : 0, D = p.D, lane_dim = 4 * (threadIdx.x % LANES), dim = lane_dim < D ? lane_dim : 0;
    const float *const from = p.partials + (int64_t)row * p.slots * p.pf_pitch;
    const int each = (p.slots + GROUPS - 1) / GROUPS, begin = group * each, end = min(p.slots, begin + each);
    float m = -INFINITY, l = 0.0f;
    float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = begin; s0 < end; s0 += U) {
        float ms[U], ls[U];
        float4_t os[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float *src = from + (int64_t)min(s0 + u, end - 1) * p.pf_pitch;
            const float2 ml = *(const float2 *)(src + D);
            os[u] = *(const float4_t *)(src + dim);
            ms[u] = s0 + u < end ? ml.x : -INFINITY;
            ls[u] = s0 + u < end ? ml.y : 0.0f;
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < U; u++) top = fmaxf(top, ms[u]);
        const float reference = top == -INFINITY ? 0.0f : top, moved = __builtin_amdgcn_exp2f(m - reference);
        l *= moved;
        o *= moved;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float weight = __builtin_amdgcn_exp2f(ms[u] - reference);
            l += weight * ls[u];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] += ms[u] == -INFINITY ? 0.0f : weight * os[u][e];  // (shares without keys hold whatever was there)
        }
        m = top;
    }
    if constexpr (GROUPS > 1) {
        *(float4_t *)&parts[group][lane_dim] = o;
        if (lane_dim == 0) states[group][0] = m, states[group][1] = l;
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int w = 1; w < GROUPS; w++) m = fmaxf(m, states[w][0]);
        const float reference = m == -INFINITY ? 0.0f : m;
        l = 0.0f, o = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < GROUPS; w++) {
            const float weight = __builtin_amdgcn_exp2f(states[w][0] - reference);
            const float4_t a = *(const float4_t *)&parts[w][lane_dim];
            l += weight * states[w][1];
            o += weight * a;
        }
    }
    if (lane_dim >= D) return;
    const uint32_t bh = row / (uint32_t)p.Sq, i = row - bh * p.Sq, b = bh / (uint32_t)p.H, h = bh - b * p.H;
    const int64_t at = b * p.os[0] + h * p.os[1] + i * p.os[2] + dim * p.os[3];
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] /= l;  // no visible key: 0 / 0 = NaN
    const bool f32 = sizeof(T) == 4 || p.out_f32;
    if (out_vec && f32) {
        *(float4_t *)((float *)p.out + at) = o;
    } else if (out_vec) {
        if constexpr (sizeof(T) == 2) {
            const T four[4] = {from_float<T>(o[0]), from_float<T>(o[1]), from_float<T>(o[2]), from_float<T>(o[3])};
            uint2r_t bits;
            __builtin_memcpy(&bits, four, 8);
            *(uint2r_t *)((T *)p.out + at) = bits;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (f32) ((float *)p.out)[at + e * p.os[3]] = o[e];
            else ((T *)p.out)[at + e * p.os[3]] = from_float<T>(o[e]);
        }
    }
}

template <typename T, int LANES>
static void merge_dims(const ContextParams &p, hipStream_t stream) {
    const long rows = (long)p.B * p.H * p.Sq;
    const int bytes = sizeof(T) == 4 || p.out_f32 ? 4 : 2;
    int out_vec = p.os[3] == 1 && (uintptr_t)p.out % (4 * bytes) == 0;
    for (int i = 0; i < 3; i++)
        if (p.os[i] % 4 != 0) out_vec = 0;
    if (p.slots <= 8 || rows > 4L * p.cus) {
        constexpr int ROWS = 256 / LANES;
        hipLaunchKernelGGL((context_merge_kernel<T, LANES, 1>), rows_grid((rows + ROWS - 1) / ROWS), dim3(256), 0, stream, p, out_vec);
    } else if (p.slots <= 32) {
        hipLaunchKernelGGL((context_merge_kernel<T, LANES, 4>), dim3((unsigned)rows), dim3(LANES * 4), 0, stream, p, out_vec);
    } else {
        hipLaunchKernelGGL((context_merge_kernel<T, LANES, 8>), dim3((unsigned)rows), dim3(LANES * 8), 0, stream, p, out_vec);
    }
}
template <typename T>
static void merge_type(const ContextParams &p, hipStream_t stream) {
    if (p.D <= 64) merge_dims<T, 16>(p, stream);
    else if (p.D <= 128) merge_dims<T, 32>(p, stream);
    else merge_dims<T, 64>(p, stream);
}
int launch_context_merge(const ContextParams &p, fhip_dtype dtype, hipStream_t stream) {
    if (dtype == FHIP_F32) merge_type<float>(p, stream);
    else if (dtype == FHIP_F16) merge_type<half_t>(p, stream);
    else merge_type<bf16_t>(p, stream);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

// ---- launch ---------------------------------------------------------------------------------------------------------------------------

// Rows of keys and values are read in pieces of 16 bytes; scores take one factor, scale times log2 e, which has to be a number.
bool context_rows_takes(const ContextParams &p, fhip_dtype dtype) {
    const int per = dtype == FHIP_F32 ? 4 : 8;
    if (p.D % 8 != 0 || p.D > 256 || !std::isfinite(p.scale * CONTEXT_LOG2E)) return false;
    auto pieces = [&](const void *at, const int64_t *strides, int n) {
        if ((uintptr_t)at % 16 != 0 || strides[n - 1] != 1) return false;
        for (int i = 0; i + 1 < n; i++)
            if (strides[i] % per != 0) return false;
        return true;
    };
    if (p.Skv > 0 && !(pieces(p.k, p.ks, 4) && pieces(p.v, p.vs, 4))) return false;
    return p.P == 0 || (pieces(p.pk, p.pks, 3) && pieces(p.pv, p.pvs, 3));
}

template <typename T, int CB>
static bool launch_rows_dims(const ContextParams &p, const ContextRows &rows, hipStream_t stream) {
    const dim3 grid((unsigned)rows.total), block(64 * CR_WAVES);
    auto run = [&](auto dims) {
        constexpr int DP = decltype(dims)::value;
        hipLaunchKernelGGL((context_rows_kernel<T, DP, CB>), grid, block, 0, stream, p, rows);
        return true;
    };
    using std::integral_constant;
    if (p.D <= 64) return run(integral_constant<int, 64>{});
    if (p.D <= 96) return run(integral_constant<int, 96>{});
    if (p.D <= 128) return run(integral_constant<int, 128>{});
    if constexpr (CB == 1) {
        if (p.D <= 192) return run(integral_constant<int, 192>{});
        return run(integral_constant<int, 256>{});
    }
    return false;
}
template <typename T>
static bool launch_rows_type(const ContextParams &p, const ContextRows &rows, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (rows.columns == 32) return launch_rows_dims<T, 2>(p, rows, stream);
    }
    return launch_rows_dims<T, 1>(p, rows, stream);
}
int launch_context_rows(const ContextParams &p, const ContextRows &rows, fhip_dtype dtype, hipStream_t stream) {
    const bool ran = dtype == FHIP_F32   ? launch_rows_type<float>(p, rows, stream)
                     : dtype == FHIP_F16 ? launch_rows_type<half_t>(p, rows, stream)
                                         : launch_rows_type<bf16_t>(p, rows, stream);
    if (!ran) {
        set_error("context_attention: no kernel for %d columns at head_dim %d", rows.columns, p.D);
        return FHIP_ERR_UNSUPPORTED;
    }
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

}  // namespace fhip
