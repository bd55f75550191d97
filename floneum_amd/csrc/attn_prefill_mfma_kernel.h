// Prefill attention for f16 / bf16 on the gfx950 matrix cores.
//
// Workgroup = 8 wavefronts = 256 query rows of one (batch, head); each wavefront owns 32 rows.
// Keys/values are walked in tiles of 64 rows that go from global memory straight into a four-stage
// LDS ring (direct-to-LDS buffer loads, no staging registers).  Per tile and wavefront:
//   S^T (64 keys x 32 queries)  = K_tile . Q^T      v_mfma_f32_32x32x16  (A = K from LDS, B = Q in registers)
//   scale * log2(e) (rr) multiplies the scores in f32: a probability is exp2(fma(s, rr, -m * rr)), one fused
//   multiply-add and one exponential per score, with m the row's reference exponent
//   online softmax down the key axis: with S^T every lane owns ONE query column and 16 keys of it per 32-key
//   block, so row sums are in-lane folds (the two half-rows are added once, at the end).  No maximum is taken
//   per tile: the reference m is the maximum the row had when it was last set, and it is moved (and l and O
//   rescaled) only when a lane's probabilities of a tile sum to more than 2^15, i.e. before one of them could
//   leave the 16-bit type's range; on random data that is the first tile and almost never again
//   O^T (D x 32 queries)       += V_tile^T . P^T    A = V^T read from row-major LDS with the
//   transposing LDS load ds_read_b64_tr_b16, B = P^T taken straight from the S^T accumulator
//   registers (the contraction index is permuted identically on both operands)
// The two wavefronts that share a SIMD (w and w + 4) run half a tile out of phase: while one is in
// its matrix phase (S^T of the current tile, P.V of the previous one, tile loads) the other is in its
// vector phase (softmax), so the MFMA pipe and the VALU are busy at the same time.
// Phases are separated by workgroup barriers; the tile loads ride on the same barriers.  The vector
// phase uses no dot-product instructions: on this chip they queue behind the MFMAs of the other
// wavefront instead of running beside them.
// Bound: power at head_dim 128 (4096 x 4096 keys, 16 heads, no mask, f16: 121 us = 1.13 PFLOP/s); below, a vector phase
// takes as long as a matrix phase or longer: its 111 vector instructions take a lone wavefront 617 cycles and beside the
// matrix instructions of the other 785, the 16 / 22 / 24 matrix instructions of head_dim 64 / 80 / 96 take 512 / 704 / 768.
// So everything but the softmax itself is done in the matrix phase, in the shadow of its instructions: tile loads, addresses,
// the mask test (an instruction on the scalar unit costs a lone wavefront as much as one on the vector unit).  f16, the
// call above at head_dim 64 / 80 / 96: 88 -> 74, 100 -> 90, 107 -> 97 us (loads, their addresses and an LDS wait in the
// vector phase before: 1350 cycles, now about 950); causal, 32/8 heads, 4000 rows at 64: 97 -> 80.
// All accumulation is f32; P is rounded to the input type for the second product.
// Key-split form (template parameter KS): the workgroup owns 128 query rows and its two wavefront groups
// take alternate key tiles of the same rows, each through the same matrix / vector phases, and merge their
// (m, l, O) through LDS at the end: twice the workgroups, half the longest one, for grids that do not fill
// the chip (see prefill_mfma_block_rows).
// Masking is by interval: every query row sees one range of keys, known analytically (causal with
// offset, sliding window, per-batch kv length, tail of the key axis) or read from the interval form
// of a dense mask tensor (attn_bounds.h, mask_intervals.hip); key tiles that are invisible to the
// whole workgroup are never loaded, and tiles fully visible to a wavefront skip the per-element test.
//
// Reference semantics: fusor-ml/fusor/src/composite/flash_attention.rs:141-199, f32 accumulation
// of 16-bit inputs as fusor-ml/core/src/composite/flash_attention.rs:186-203,323-327; head
// mapping kv_head = head / (H / Hkv) (core :135-137,163-167).
#pragma once
#include <type_traits>

#include "attn_bounds.h"
#include "common.h"
#include "context_tiles.h"
#include "device_utils.h"

namespace fhip {

constexpr int PF_WAVES = 8;
constexpr int PF_BM = 32 * PF_WAVES;  // query rows per workgroup
constexpr int PF_BN = 64;             // key rows per tile
constexpr float PF_LOG2E = 1.4426950408889634f;

#define LDS_PTR(type, byte_off) ((__attribute__((address_space(3))) type *)(lds_base + (byte_off)))

template <typename T>
struct Mma;
template <>
struct Mma<half_t> {
    typedef half8_t vec8;
    static __device__ __forceinline__ float16_t mfma(vec8 a, vec8 b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float x, float y) {
        half2_t h = {(half_t)x, (half_t)y};
        return __builtin_bit_cast(uint32_t, h);
    }
};
template <>
struct Mma<bf16_t> {
    typedef bf16x8_t vec8;
    static __device__ __forceinline__ float16_t mfma(vec8 a, vec8 b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float x, float y) {
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        const bf16x2_t h = {(__bf16)x, (__bf16)y};  // v_cvt_pk_bf16_f32: round to nearest even
        return __builtin_bit_cast(uint32_t, h);
    }
    static __device__ __forceinline__ vec8 scaled(vec8 q, float c) {
#pragma unroll
        for (int e = 0; e < 8; e++) q[e] = (__bf16)((float)q[e] * c);
        return q;
    }
};

// LDS image of a 64-row tile.  Rows are kept in NG groups: row r sits in group r % NG at position r / NG.  A group is what
// one wavefront-wide direct-to-LDS load writes (D = 128: 4 rows, D = 64: 8), or three of them (D = 96: 16 rows), whole
// kilobytes either way, so that every lane of every load moves 16 bytes.  Groups are padded apart so that
//   - rows r .. r + 3 at one column fall 16 bytes apart modulo the 256-byte bank period, and the sixteen rows that the LDS
//     serves at once in a 128-bit read (four such runs) fall into sixteen different places  (K: pitch of a group + 16)
//   - the 4 rows x 64 bytes a half-wavefront reads with the transposing load fall 64 bytes apart  (V: pitch + 64)
template <int D, bool KS>
struct PfCfg {
    static constexpr int ROWB = D * 2;                               // bytes per tile row
    static constexpr int NG = D == 128 ? 16 : D == 96 ? 4 : 8;       // groups of a tile
    static constexpr int KG = PF_BN / NG * ROWB + 16;                // K group pitch, bytes
    static constexpr int VG = PF_BN / NG * ROWB + 64;                // V group pitch, bytes
    static constexpr int K_BYTES = NG * KG;
    static constexpr int V_BYTES = NG * VG;
    static constexpr int CPR = D / 8;                                // 16-byte chunks per row
    static constexpr int LOADS = PF_BN * ROWB / 4096;                // loads of each of the four wavefronts that move a tile
    static constexpr int OFFSETS = NG == 4 ? LOADS : 1;              // (their lanes' offsets differ by a uniform value otherwise)
    // tile buffers.  Unsplit form: four stages of (K tile, V tile), tile t in stage t % 4.  Key-split form
    // (KS): a ring of five K tiles followed by a ring of four V tiles (see the slot schedule in the kernel).
    static constexpr int STAGE = K_BYTES + V_BYTES;
    static constexpr int NK = KS ? 5 : 4, NV = 4;
    static constexpr int LDS_BYTES = KS ? NK * K_BYTES + NV * V_BYTES : 4 * STAGE;
    static constexpr int BM = KS ? PF_BM / 2 : PF_BM;                // query rows per workgroup
};

__device__ __forceinline__ float half_swap_max(float x) {
    // max of x with the value held by the lane 32 away
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_swap_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// D: head_dim rounded up to 64, 96 or 128, the width of the tiles and of O.  QD: the dims contracted in K . Q^T, head_dim
// rounded up to 16.  PAD: head_dim is less than D; the dims behind it are zero in Q, K and V (their lanes fetch from beyond
// the buffer) and are not written.
// P: AttnParams, or for attention over a context in two parts (CTX, see context_tiles.h) ContextParams, of whose parts the launch takes one, or
// ContextBoth: both, unsplit form only.  Rows are then stacked, and a row sees two runs of keys.
template <typename T, int D, int QD, bool PAD, bool KS, class P>
__global__ __launch_bounds__(64 * PF_WAVES, 2) void prefill_mfma_kernel(P p, int nqb, int out_vec) {
    request_arguments<P, int, int>();
    constexpr bool CTX = std::is_base_of<ContextParams, P>::value, BOTH = std::is_same<P, ContextBoth>::value;
    static_assert(!(KS && BOTH), "the key-split form has no scalar registers for the descriptors of both parts");
    typedef PfCfg<D, KS> C;
    typedef typename Mma<T>::vec8 vec8;
    constexpr int STAGE = C::STAGE;
    constexpr int BM = C::BM;
    __shared__ __attribute__((aligned(16))) char smem[C::LDS_BYTES];
    auto lds_base = (__attribute__((address_space(3))) char *)smem;

    if (!CTX && p.iv_bad && *p.iv_bad == p.bad_tag) return;  // the mask is not made of intervals: the general kernel takes the call
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // scalar: everything derived from it is uniform
    const int lane = tid & 63;
    const int ln = lane & 31;      // query column / key row owned inside a 32-wide MFMA block
    const int h2 = lane >> 5;      // which half of the contraction slice
    const int group = wave >> 2;   // wavefronts w and w + 4 share a SIMD and run out of phase

    // workgroup -> (query block, batch, head): long query blocks first, and heads laid out so
    // the workgroups that land on one XCD (id % 8) share a KV head whenever H is a multiple of 8
    // Packed form (key-split form only, at most 32 query rows, GQA group a multiple of 4): the workgroup's four row
    // blocks are rows 0..31 of four query heads that share a KV head, so the K and V tiles it moves serve all four
    // and a few new rows on a long cache read the cache once per KV head, not once per query head.
    const int pack = KS && !CTX ? p.pf_pack : 0;
    const int heads = pack ? p.H / 4 : p.H;  // head units per batch entry
    int bh_count = p.B * heads;
    uint32_t place = blockIdx.x;
    int nks = max(p.pf_nsplit, 1);
    if constexpr (CTX) {
        place = tiles_work(p);
        bh_count = p.job.units, nqb = p.job.blocks, nks = p.job.shares;
    }
    const int ksplit = place % nks;  // which share of the keys (0 when the keys are not split over workgroups)
    const int id = place / nks;
    const int qb = nqb - 1 - id / bh_count;
    int rem = id % bh_count;
    int b = rem / heads;
    int h = rem % heads;
    if (pack) h = 4 * h + (wave & 3);
    else if ((p.H & 7) == 0) h = (h & 7) * (p.H >> 3) + (h >> 3);
    int g = h / p.G;
    if constexpr (CTX) {
        b = p.job.fold ? -1 : rem / p.Hkv;  // (-1: rows of all sequences)
        g = p.job.fold ? rem : rem - b * p.Hkv;
    }
    // Rows of a tile beyond the sequence's own keys (kv_lens below the view's length: a ragged batch in one cache
    // allocation) read as zero (the buffers end there): what such rows hold, NaN included, must not reach the result as 0 x NaN in P . V.
    // (likewise the rows behind the last query's own position when the call says where its rows stand inside a longer
    // cache view: a causal descriptor with q_pos_offset + Sq below the view's length)
    int key_end = !CTX && p.kv_lens ? min(p.Skv, max(p.kv_lens[b], 1)) : p.Skv;
    if (!CTX && p.analytic && p.causal) key_end = (int)min((int64_t)key_end, max(p.q_pos_offset + p.Sq, (int64_t)1));

    const int q0 = pack ? 0 : qb * BM;
    const int qw0 = pack ? 0 : q0 + 32 * (KS ? (wave & 3) : wave);  // KS: both groups own the same 128 rows
    const int query = qw0 + ln;
    int total_rows = p.Sq;
    RowBounds rb;
    // CTX: this lane's row and what it sees, what the wavefront's and the workgroup's rows see, and the tiles; keys are rows of the one part, or (BOTH)
    // numbered through both
    StackedRow row_at;
    ContextRow sees;
    StackedSpan wave_sees;
    ContextSpan wg_sees;
    typename std::conditional<BOTH, ContextBothTiles<PF_BN>, ContextTiles<PF_BN>>::type tiles;
    if constexpr (CTX) {
        total_rows = p.job.rows;
        row_at = stacked_row(p, b, g, min(query, total_rows - 1));
        stacked_spans<BM>(p, b, q0, qw0, lane, row_at, wave_sees, wg_sees, sees);
        if constexpr (!BOTH) {
            const bool prefix = p.job.with_prefix != 0;
            sees = sees.of(p, prefix), wave_sees = wave_sees.of(p, prefix), wg_sees = wg_sees.of(p, prefix);
        }
        tiles.set(p, wg_sees, ksplit);
    } else {
        rb = row_bounds(p, b, q0, pack ? 32 : BM, qw0, lane);
    }
    if (!CTX && nks > 1) {  // few query rows on a long cache: this workgroup takes one share of the keys
        const int c_lo = ksplit * p.pf_chunk, c_hi = c_lo + p.pf_chunk;
        rb.lo_wg = max(rb.lo_wg, c_lo), rb.hi_wg = min(rb.hi_wg, c_hi);
        rb.lo_w = max(rb.lo_w, c_lo), rb.hi_w = min(rb.hi_w, c_hi);
        rb.full_lo_w = max(rb.full_lo_w, c_lo), rb.full_hi_w = min(rb.full_hi_w, c_hi);
        rb.klo = max(rb.klo, c_lo), rb.khi = min(rb.khi, c_hi);
    }
    const int lo_wg = rb.lo_wg, hi_wg = rb.hi_wg, lo_w = rb.lo_w, hi_w = rb.hi_w;
    const int full_lo_w = rb.full_lo_w, full_hi_w = rb.full_hi_w, klo = rb.klo, khi = rb.khi;
    const int qrow = CTX ? row_at.row : min(query, p.Sq - 1);
    const int hd = PAD ? p.D : D;  // the head dim itself
    const bool wave_has_rows = qw0 < total_rows;

    // Q^T operand: Q[query][16 kb + 8 h2 .. +8], kept in registers for the whole kernel
    // (the loads are issued here; whatever scaling they take waits until the first K/V tiles are on their way too)
    const float scale2 = p.scale * PF_LOG2E;
    // rr multiplies every score in f32 right before exp2: the scores are then the f32 dot product times the scale, one
    // rounding, as the reference computes them (fusor-ml/fusor/src/composite/flash_attention.rs:145).  Folding scale2 into
    // Q instead would save that multiply but round Q's elements a second time (11 bits in f16, 8 in bf16), an error that
    // grows in proportion to the scores.  The S^T accumulators and m are in units of 1 / rr.
    // bf16 at the kernel's own head dims: Q takes the power of two in scale2 (pw), which is exact down to bf16's smallest
    // normal value and keeps dot products of very large elements inside f32's range.  f16 takes none of it: elements below
    // 2^-14 / pw would become subnormal and lose bits, and the products of f16 elements cannot leave f32's range.
    constexpr bool FOLD = std::is_same<T, bf16_t>::value && !PAD;
    const float pw = FOLD ? __uint_as_float(__float_as_uint(scale2) & 0x7F800000u) : 1.0f;
    const float rr = FOLD ? scale2 / pw : scale2;
    vec8 qreg[QD / 16];
    {
        const uint16_t *qp = (const uint16_t *)p.q + (CTX ? row_at.b : b) * p.qs[0] + (CTX ? row_at.h : h) * p.qs[1] + (int64_t)qrow * p.qs[2];
#pragma unroll
        for (int kb = 0; kb < QD / 16; kb++) {
            uint4_t raw = {0, 0, 0, 0};
            if (!PAD || 16 * kb + 8 * h2 < hd) raw = *(const uint4_t *)(qp + 16 * kb + 8 * h2);
            qreg[kb] = __builtin_bit_cast(vec8, raw);
        }
    }

    const int j_begin = (lo_wg / PF_BN) * PF_BN;
    const int ntiles = CTX ? tiles.count : hi_wg > j_begin ? (hi_wg - j_begin + PF_BN - 1) / PF_BN : 0;

    // K and V of this (batch, kv head) as raw buffers: a row beyond the end of the key axis reads as
    // zero, so the tile loop needs neither clamps nor 64-bit address arithmetic
    const uint16_t *kg = (const uint16_t *)p.k + b * p.ks[0] + g * p.ks[1];
    const uint16_t *vg = (const uint16_t *)p.v + b * p.vs[0] + g * p.vs[1];
    int krow_bytes = (int)p.ks[2] * 2, vrow_bytes = (int)p.vs[2] * 2, key_rows = p.Skv;
    // BOTH: the prefix's; key_end, key_rows and the above are the own keys'
    const uint16_t *prefix_kg, *prefix_vg;
    int prefix_krow_bytes, prefix_vrow_bytes, prefix_end;
    if constexpr (CTX) {
        prefix_kg = (const uint16_t *)p.pk + g * p.pks[0], prefix_vg = (const uint16_t *)p.pv + g * p.pvs[0];
        prefix_krow_bytes = (int)p.pks[1] * 2, prefix_vrow_bytes = (int)p.pvs[1] * 2;
        kg = (const uint16_t *)p.k + max(b, 0) * p.ks[0] + g * p.ks[1], vg = (const uint16_t *)p.v + max(b, 0) * p.vs[0] + g * p.vs[1];
        if constexpr (BOTH) {
            prefix_end = wg_sees.of(p, true).end(), key_end = wg_sees.of(p, false).end();
        } else {
            key_end = wg_sees.end();
            if (p.job.with_prefix) kg = prefix_kg, vg = prefix_vg, krow_bytes = prefix_krow_bytes, vrow_bytes = prefix_vrow_bytes, key_rows = p.P;
        }
    }

    float16_t o[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; db++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[db][r] = 0.0f;
    // m: the row's reference exponent, in units of the S^T accumulators (1 / rr of a base-2 exponent): probabilities are
    // exp2((s - m) * rr), formed as exp2(fma(s, rr, nmr)) with nmr = -m * rr.  While the row has seen no key m is -inf and
    // nmr +inf, which sends the first tile with a visible key through the branch that sets m (see softmax below).
    float m = -INFINITY, l = 0.0f, nmr = INFINITY;
    float16_t zero16;
#pragma unroll
    for (int r = 0; r < 16; r++) zero16[r] = 0.0f;

    using std::integral_constant;
    // ---- tile movement: global -> LDS directly (no registers) --------------------------------------
    // The four wavefronts of a group move one whole tile with LOADS loads each.  Load j of wavefront w writes LDS group
    // w + 4 j (D = 96: the j-th kilobyte of group w); its lanes fetch that group's 16-byte chunks in order (which is how
    // the hardware lays out a direct load).
    // Unsplit form: group 1 moves the K tiles, group 0 the V tiles.  Key-split form: the group that is in
    // its vector phase moves one K and one V tile.
    // The tensors as raw buffer descriptors (base, no stride, size in bytes, 32-bit raw format): a row beyond
    // the end of the key axis reads as zero.
    const bool moves_k = group == 1;
    const int wv = wave & 3;
    auto uniform = [](uint32_t x) __attribute__((always_inline)) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
    auto descriptor = [&](const uint16_t *base, int row_bytes, int end) __attribute__((always_inline)) {
        const uint64_t ptr = (uint64_t)base;
        if constexpr (CTX)
            return uint4_t{uniform((uint32_t)ptr), uniform((uint32_t)(ptr >> 32) & 0xffffu), uniform(end > 0 ? (end - 1) * row_bytes + hd * 2 : 0),
                           0x00020000u};
        else
            return uint4_t{(uint32_t)ptr, (uint32_t)(ptr >> 32) & 0xffffu, (uint32_t)((end - 1) * row_bytes + hd * 2), 0x00020000u};
    };
    const uint4_t krs = descriptor(kg, krow_bytes, key_end), vrs = descriptor(vg, vrow_bytes, key_end);
    int gofs_k[C::OFFSETS], gofs_v[C::OFFSETS];
#pragma unroll
    for (int j = 0; j < C::OFFSETS; j++) {
        const int chunk = lane + 64 * j, row = C::NG * (chunk / C::CPR) + wv, col = chunk % C::CPR;
        const bool padding = PAD && col * 8 >= hd;
        gofs_k[j] = padding ? 0x7ffffff0 : row * krow_bytes + col * 16;
        gofs_v[j] = padding ? 0x7ffffff0 : row * vrow_bytes + col * 16;
    }
    // where tile t lives in LDS
    auto k_stage = [&](int t) __attribute__((always_inline)) { return KS ? (int)((uint32_t)t % C::NK) * C::K_BYTES : (t & 3) * STAGE; };
    auto v_stage = [&](int t) __attribute__((always_inline)) {
        return KS ? C::NK * C::K_BYTES + (t & 3) * C::V_BYTES : (t & 3) * STAGE + C::K_BYTES;
    };
    // a tile that starts beyond the key axis is never used: clamp the (uniform) offset so it stays
    // inside 32 bits; rows past Skv inside a used tile are out of range of the buffer and read 0
    // (uniform values, pinned to scalar registers, which is what the instruction takes.  M0 takes an LDS address, not an
    // offset into the tile buffers: they are the kernel's only LDS variable and start at 0, which the compiler folds in.
    // Written as assembly on purpose: the compiler would otherwise make every later LDS read of this wavefront wait for
    // these loads, whose data is not due before a later barrier.)
    auto issue = [&](const uint4_t rs, const int (&gofs)[C::OFFSETS], int row_bytes, int soff, int lbase, int pitch, int j)
                     __attribute__((always_inline)) {
        const int lds = lbase + (C::NG == 4 ? 1024 * j : 4 * j * pitch), from = soff + (C::NG == 4 ? 0 : 4 * j * row_bytes);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :
                     : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(gofs[C::OFFSETS > 1 ? j : 0]), "s"(rs),
                       "s"(__builtin_amdgcn_readfirstlane(from))
                     : "m0");
    };
    auto first_row = [&](int tile) __attribute__((always_inline)) {  // (of its tensor)
        if constexpr (CTX) return tiles.row(tile);
        else return j_begin + tile * PF_BN;
    };
    auto row_offset = [&](int tile, int row_bytes) __attribute__((always_inline)) { return min(first_row(tile), CTX ? key_rows : p.Skv) * row_bytes; };
    // CTX: rows between the first tokens and the window, which no row of the workgroup sees, are not fetched (they may hold anything)
    auto without_hole = [&](int (&gofs)[C::OFFSETS], int first_key, int j) __attribute__((always_inline)) {
        const int chunk = lane + (C::NG == 4 ? 64 * j : 0), key = first_key + C::NG * (chunk / C::CPR) + wv + (C::NG == 4 ? 0 : 4 * j);
        if (key >= wg_sees.first && key < wg_sees.lo) gofs[C::OFFSETS > 1 ? j : 0] = 0x7ffffff0;
    };
    auto issue_tile = [&](const uint4_t rs, const int (&gofs)[C::OFFSETS], int row_bytes, int tile, int lbase, int pitch, int j) __attribute__((always_inline)) {
        int at[C::OFFSETS];
        at[C::OFFSETS > 1 ? j : 0] = gofs[C::OFFSETS > 1 ? j : 0];
        if (__builtin_expect(tiles.edge(tile), 0)) without_hole(at, first_row(tile), j);
        issue(rs, at, row_bytes, row_offset(tile, row_bytes), lbase, pitch, j);
    };
    const int lds0 = (int)(uint32_t)(uintptr_t)lds_base;
    auto issue_k = [&](int tile, int j) __attribute__((always_inline)) {
        if constexpr (CTX) issue_tile(krs, gofs_k, krow_bytes, tile, lds0 + k_stage(tile) + wv * C::KG, C::KG, j);
        else issue(krs, gofs_k, krow_bytes, row_offset(tile, krow_bytes), lds0 + k_stage(tile) + wv * C::KG, C::KG, j);
    };
    auto issue_v = [&](int tile, int j) __attribute__((always_inline)) {
        if constexpr (CTX) issue_tile(vrs, gofs_v, vrow_bytes, tile, lds0 + v_stage(tile) + wv * C::VG, C::VG, j);
        else issue(vrs, gofs_v, vrow_bytes, row_offset(tile, vrow_bytes), lds0 + v_stage(tile) + wv * C::VG, C::VG, j);
    };
    // Load n of those that a matrix phase issues.  Unsplit form: of one tile of this group's tensor (K: group 1, V: group 0).
    // Key-split form, slot s: of K(s + 4) and V(s + 1).
    constexpr int PHASE_LOADS = KS ? 2 * C::LOADS : C::LOADS;
    const uint4_t mrs = moves_k ? krs : vrs;
    const int mrow_bytes = moves_k ? krow_bytes : vrow_bytes, mpitch = moves_k ? C::KG : C::VG;
    const int mbase = lds0 + (moves_k ? 0 : C::K_BYTES) + wv * mpitch;
    int mgofs[C::OFFSETS];
#pragma unroll
    for (int j = 0; j < C::OFFSETS; j++) mgofs[j] = moves_k ? gofs_k[j] : gofs_v[j];
    uint4_t prefix_mrs;
    int prefix_mrow_bytes, prefix_mgofs[C::OFFSETS];
    if constexpr (BOTH) {
        prefix_mrow_bytes = moves_k ? prefix_krow_bytes : prefix_vrow_bytes;
        prefix_mrs = descriptor(moves_k ? prefix_kg : prefix_vg, prefix_mrow_bytes, prefix_end);
#pragma unroll
        for (int j = 0; j < C::OFFSETS; j++) {
            const int chunk = lane + 64 * j, row = C::NG * (chunk / C::CPR) + wv, col = chunk % C::CPR;
            prefix_mgofs[j] = PAD && col * 8 >= hd ? 0x7ffffff0 : row * prefix_mrow_bytes + col * 16;
        }
    }
    auto load = [&](int at, int n) __attribute__((always_inline)) {
        if (n >= PHASE_LOADS) return;
        if constexpr (KS) {
            if (n & 1) issue_v(at + 1, n >> 1);
            else issue_k(at + 4, n >> 1);
        } else if constexpr (BOTH) {
            const bool own = tiles.own(at);
            const int row0 = min(tiles.row(at), own ? p.Skv : p.P), bytes = own ? mrow_bytes : prefix_mrow_bytes, o = C::OFFSETS > 1 ? n : 0;
            int gofs[C::OFFSETS];
            gofs[o] = own ? mgofs[o] : prefix_mgofs[o];
            if (__builtin_expect(tiles.edge(at), 0)) without_hole(gofs, row0 + (own ? p.P : 0), n);
            issue(own ? mrs : prefix_mrs, gofs, bytes, row0 * bytes, mbase + (at & 3) * STAGE, mpitch, n);
        } else if constexpr (CTX) {
            issue_tile(mrs, mgofs, mrow_bytes, at, mbase + (at & 3) * STAGE, mpitch, n);
        } else {
            issue(mrs, mgofs, mrow_bytes, row_offset(at, mrow_bytes), mbase + (at & 3) * STAGE, mpitch, n);
        }
    };
    auto load_all = [&](int at) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < PHASE_LOADS; n++) load(at, n);
    };
    // all but the most recent N loads of this wavefront have landed
    auto wait_loads = [&](auto n) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(decltype(n)::value) : "memory");
    };
    // local tile index -> tile: in the key-split form group g owns the tiles t with t % 2 == g
    auto tile_of = [&](int i) __attribute__((always_inline)) { return KS ? 2 * i + group : i; };

    float16_t s[2];     // S^T of the tile in flight
    uint32_t pk[2][8];  // its probabilities, packed pairs in the MFMA operand order

    // A matrix phase: S^T of tile i (QK) and P.V of tile i - 1 (PV), and the tile loads of the slot.  S^T's K operands of the
    // first PRE contraction slices have been read in the vector phase before (PREFETCHED), the others leave the LDS several
    // matrix instructions ahead of their use, and V's likewise; each step is fenced, so that neither the reads nor the
    // loads gather in front of the matrix instructions.
    // O^T += V^T . P^T: contraction slice (t, kk) holds this half-wave's keys 32 t + 16 kk + 4 h2 + {0..3} and + 8
    constexpr int NDB = D / 32, NKB = QD / 16;
    constexpr int PFK = (D == 128) ? 2 : 4;  // K operand slices in flight (register budget)
    // Contraction slices read in the vector phase.  None where that phase is much the longer one: head_dim 64, 4096 x 4096 keys
    // 76.8 -> 75.4 us; at 80 and 96 no difference, at 128 reading none costs 1 % (499 -> 504 us for an 8192-token prompt).
    constexpr int PRE = D == 64 ? 0 : 2;
    uint4_t ka[PFK][2];
    const int i16 = lane & 15, bl = (lane & 31) >> 4;
    const int k_at = (ln % C::NG) * C::KG + (ln / C::NG) * C::ROWB + h2 * 16;
    const int v_at = (C::NG == 4 ? (i16 >> 2) * C::VG + h2 * C::ROWB : (4 * h2 + (i16 >> 2)) * C::VG) + (16 * bl + 4 * (i16 & 3)) * 2;
    constexpr int V_SLICE = 16 / C::NG * C::ROWB, V_PLUS8 = C::NG == 16 ? 8 * C::VG : 8 / C::NG * C::ROWB;
    auto read_k = [&](int kbase, int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; t++) ka[kb % PFK][t] = *LDS_PTR(uint4_t, kbase + t * (32 / C::NG) * C::ROWB + kb * 32);
    };
    auto prefetch_k = [&](int i) __attribute__((always_inline)) {
        const int kbase = k_stage(tile_of(i)) + k_at;
#pragma unroll
        for (int kb = 0; kb < PRE; kb++) read_k(kbase, kb);
    };
    bool masked = false;  // the tile whose S^T was formed last is not wholly visible to this wavefront
    auto qk_pv = [&](int i, int at, auto do_qk, auto do_pv, auto prefetched) __attribute__((always_inline)) {
        constexpr bool QK = decltype(do_qk)::value, PV = decltype(do_pv)::value, PREFETCHED = decltype(prefetched)::value;
        const int kbase = k_stage(tile_of(i)) + k_at, vbase = v_stage(tile_of(i - 1)) + v_at;
        uint4_t va[2][NDB];
        auto read_v = [&](int gq) __attribute__((always_inline)) {  // gq = 2 t + kk: rows 16 gq + 4 h2 + {0..3} and + 8
#pragma unroll
            for (int db = 0; db < NDB; db++) {
                const int addr = vbase + gq * V_SLICE + db * 64;
                short4_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(short4_t, addr));
                short4_t a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(short4_t, addr + V_PLUS8));
                const uint2_t u0 = __builtin_bit_cast(uint2_t, a0), u1 = __builtin_bit_cast(uint2_t, a1);
                va[gq & 1][db] = uint4_t{u0[0], u0[1], u1[0], u1[1]};
            }
        };
        if constexpr (QK) {
#pragma unroll
            for (int kb = PREFETCHED ? PRE : 0; kb < PFK; kb++) read_k(kbase, kb);
#pragma unroll
            for (int kb = 0; kb < NKB; kb++) {
#pragma unroll
                for (int t = 0; t < 2; t++)
                    s[t] = Mma<T>::mfma(__builtin_bit_cast(vec8, ka[kb % PFK][t]), qreg[kb], kb == 0 ? zero16 : s[t]);
                if (kb + PFK < NKB) read_k(kbase, kb + PFK);
                if (PV && kb >= NKB - 4 && kb < NKB - 2) read_v(kb + 4 - NKB);
                load(at, kb);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (BOTH) {
                const int tile = tile_of(i), end = tiles.own(tile) ? 0x7fffffff : p.P, j0 = tiles.row(tile) + (tiles.own(tile) ? p.P : 0);
                masked = !((j0 >= wave_sees.all.lo && j0 + PF_BN <= min(wave_sees.all.hi, end)) || j0 + PF_BN <= min(wave_sees.all.first, end));
            } else if constexpr (CTX) {
                const int j0 = first_row(tile_of(i));
                masked = !((j0 >= wave_sees.all.lo && j0 + PF_BN <= wave_sees.all.hi) || j0 + PF_BN <= wave_sees.all.first);
            } else {
                const int j0 = j_begin + tile_of(i) * PF_BN;
                masked = !(j0 >= full_lo_w && j0 + PF_BN <= full_hi_w);
            }
        } else {
            read_v(0);
            read_v(1);
        }
        if constexpr (PV) {
#pragma unroll
            for (int gq = 0; gq < 4; gq++) {
                const int t = gq >> 1, kk = gq & 1;
                const uint4_t braw = {pk[t][4 * kk], pk[t][4 * kk + 1], pk[t][4 * kk + 2], pk[t][4 * kk + 3]};
#pragma unroll
                for (int db = 0; db < NDB; db++)
                    o[db] = Mma<T>::mfma(__builtin_bit_cast(vec8, va[gq & 1][db]), __builtin_bit_cast(vec8, braw), o[db]);
                if (gq < 2) read_v(gq + 2);
                load(at, (QK ? NKB : 0) + gq);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int n = (QK ? NKB : 0) + (PV ? 4 : 0); n < PHASE_LOADS; n++) load(at, n);
    };
    // mask + online softmax (log2 domain, lazily rescaled) of tile i: s -> pk
    auto softmax = [&](int i) __attribute__((always_inline)) {
        if (CTX && masked) {
            int j0 = first_row(tile_of(i)), hi = sees.hi;
            if constexpr (BOTH) {
                if (tiles.own(tile_of(i))) j0 += p.P;
                else hi = min(hi, p.P);
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = j0 + 32 * t + 8 * (r >> 2) + 4 * h2 + (r & 3);
                    s[t][r] = key < hi && (key >= sees.lo || key < sees.first) ? s[t][r] : -INFINITY;
                }
        } else if (masked) {
            const int j0 = j_begin + tile_of(i) * PF_BN;
            // element r of block t is key j0 + 32 t + 8 (r / 4) + 4 h2 + r % 4
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = j0 + 32 * t + 8 * (r >> 2) + 4 * h2 + (r & 3);
                    s[t][r] = (key >= klo && key < khi) ? s[t][r] : -INFINITY;
                }
        }
        // Probabilities against the reference the row already has; no maximum is taken.  The reference is whatever maximum
        // the row had when it was last set, so a probability may exceed 1: harmless while it stays inside the 16-bit
        // type's range (P is rounded to it for the second product; l and O are f32), and that is what the check below
        // guarantees: a lane's 32 probabilities are positive, so while their sum is at most 2^15 each of them is.
        auto probabilities = [&](float nm) __attribute__((always_inline)) {
            // four products ahead of the exponentials and two exponentials ahead of their uses: a lone wavefront has nothing
            // else to issue while one waits for the other
            constexpr int AHEAD = 4, LAG = 2;
            float x[32], sum[2] = {0.0f, 0.0f};
            auto scaled = [&](int r) __attribute__((always_inline)) { x[r] = __builtin_fmaf(s[r >> 4][r & 15], rr, nm); };
#pragma unroll
            for (int r = 0; r < AHEAD; r++) scaled(r);
#pragma unroll
            for (int r = 0; r < 32 + LAG; r++) {
                if (r < 32) x[r] = __builtin_amdgcn_exp2f(x[r]);
                if (r + AHEAD < 32) scaled(r + AHEAD);
                const int d = r - LAG;
                if (d >= 0) sum[d & 1] = d < 2 ? x[d] : sum[d & 1] + x[d];  // (a dot-product instruction would queue behind the MFMAs)
                if (d >= 0 && (d & 1)) pk[d >> 4][(d & 15) >> 1] = Mma<T>::pack2(x[d - 1], x[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
            return sum[0] + sum[1];
        };
        float ts = probabilities(nmr);
        // Not at most 2^15 (which also catches the +inf and NaN a row without a reference produces): some row of the
        // wavefront needs its reference moved.  Take the tile's maximum, move every row's reference to at least that,
        // rescale what the row has accumulated, and form the tile's probabilities again.
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(ts <= 32768.0f)) != 0, 0)) {
            float mx = s[0][0];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[t][r]);
            mx = half_swap_max(mx);
            const float m_new = fmaxf(m, mx);
            const float corr = (m == -INFINITY) ? 0.0f : __builtin_amdgcn_exp2f((m - m_new) * rr);
            m = m_new;
            l *= corr;
#pragma unroll
            for (int db = 0; db < D / 32; db++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[db][r] *= corr;
            // still no visible key: the tile's probabilities are exp2(-inf) = 0 and the row stays without a reference
            nmr = (m == -INFINITY) ? INFINITY : -m * rr;
            ts = probabilities((m == -INFINITY) ? 0.0f : nmr);
        }
        l += ts;
    };

    // ---- slot schedule ---------------------------------------------------------------------------------
    // Slots are separated by workgroup barriers.  Group 0 is in its matrix phase in even slots and in
    // its vector phase in odd slots; group 1 the other way round, one slot later.  Matrix phase of
    // tile i: S^T of tile i (reads K(i)), then P.V of tile i-1 (reads V(i-1)); K(i) is read in slots 2i - 1 (ahead, by
    // group 0) to 2i+1, V(i) in slots 2i+2 and 2i+3.  Vector phase: read the first K operands of the next matrix phase,
    // softmax, wait for a tile issued two matrix phases ago.
    // Tile t lives in stage t % 4.  In odd slot 2j+1 group 1 issues K(j+3) (its stage was last read for
    // K(j-1) in slot 2j-1) and makes sure in slot 2j+2 that K(j+2) has landed; in even slot 2j group 0 issues V(j+2)
    // (stage last read for V(j-2) in slot 2j-1) and makes sure in slot 2j+1 that V(j) has landed.  Every tile is thus
    // complete, and published by a barrier, before the slot of its first reader, and has had at least three
    // slots to arrive.
    // The tiles visible to a wavefront form one contiguous range [ia, ib).  Each group walks the slot
    // sequence in five static segments (nothing / first tile / steady state / last tile / nothing) so
    // that the steady-state loop body is branch-free and no state changes registers between phases.
    //
    // Key-split form (KS): both groups own the same 128 rows and group g takes the tiles t with t % 2 == g,
    // so a slot is the matrix phase of tile s for one group and the vector phase of tile s-1 for the other;
    // the groups' (m, l, O) are merged at the end.  K(t) is read in slot t (its first operands in
    // slot t-1), V(t) in slot t+2.  The group in its matrix phase in slot s issues K(s+4) into the stage K(s-1)
    // has just left (ring of 5) and V(s+1) into the stage of V(s-3), last read in slot s-1 (ring of 4), and
    // makes sure its loads of slot s-2, K(s+2) and V(s-1), have landed: each is published by a barrier
    // before the slot of its first reader and has had two slots to arrive.  The segments below then run on the
    // group's own tile count: local tile i of group g is tile 2 i + g.
    int ia = 0, ib = 0;
    if constexpr (CTX) {
        if (wave_has_rows && wave_sees.some.keys() > 0) {
            ia = min(max(tiles.holding(p, wave_sees.some.begin()), 0), ntiles);
            ib = min(max(tiles.holding(p, wave_sees.some.end() - 1) + 1, ia), ntiles);
        }
    } else if (wave_has_rows && hi_w > lo_w) {
        ia = (lo_w - j_begin) / PF_BN;
        ib = min(ntiles, (hi_w - j_begin + PF_BN - 1) / PF_BN);
        if (ib < ia) ib = ia;
    }
    int n_iter = ntiles + 1;  // iterations (two slots each) of either group
    if constexpr (KS) {
        ia = (ia + 1 - group) >> 1;  // this group's tiles below ia / below ib
        ib = (ib + 1 - group) >> 1;
        n_iter = (ntiles + 3) >> 1;
    }
    // MODE bit 0: S^T of tile i; bit 1: P.V of tile i-1; bit 2: softmax of tile i (group 0) / i-1 (group 1);
    // bit 3: the K operands of tile i were prefetched by the preceding vector phase;
    // bit 4: prefetch the K operands for the next matrix phase in the vector phase
    auto matrix_phase = [&](int i, int at, auto mode) __attribute__((always_inline)) {
        constexpr int MODE = decltype(mode)::value;
        __builtin_amdgcn_s_setprio(1);
        if constexpr ((MODE & 3) != 0)
            qk_pv(i, at, integral_constant<bool, (MODE & 1) != 0>{}, integral_constant<bool, (MODE & 2) != 0>{},
                  integral_constant<bool, (MODE & 8) != 0>{});
        else load_all(at);
        __builtin_amdgcn_s_setprio(0);
        if constexpr (KS) wait_loads(integral_constant<int, PHASE_LOADS>{});  // those of the matrix phase before have landed
    };
    // next_k: the tile whose S^T this wavefront computes in its next matrix phase
    auto vector_phase = [&](int i, int next_k, auto newer, auto mode) __attribute__((always_inline)) {
        constexpr int MODE = decltype(mode)::value;
        if constexpr ((MODE & 16) != 0) prefetch_k(next_k);
        if constexpr ((MODE & 4) != 0) softmax(i);
        if constexpr (!KS) wait_loads(newer);
    };
    // Between slots nothing but the barrier itself: no wavefront writes to LDS in the loop, and the K operands read ahead may
    // still be on their way (their stage is written two slots later at the earliest).
    auto slot_end = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto segment0 = [&](int i0, int i1, auto mode) __attribute__((always_inline)) {  // group 0: slot 2i matrix + V(i+2), slot 2i+1 vector
        for (int i = i0; i < i1; i++) {
            matrix_phase(i, KS ? 2 * i : i + 2, mode);
            slot_end();
            vector_phase(i, i + 1, integral_constant<int, 2 * C::LOADS>{}, mode);
            slot_end();
        }
    };
    auto segment1 = [&](int i0, int i1, auto mode) __attribute__((always_inline)) {  // group 1: slot 2i vector (tile i-1), slot 2i+1 matrix + K(i+3)
        for (int i = i0; i < i1; i++) {
            vector_phase(i - 1, i, integral_constant<int, C::LOADS>{}, mode);
            slot_end();
            matrix_phase(i, KS ? 2 * i + 1 : i + 3, mode);
            slot_end();
        }
    };
    if (ntiles > 0) {
        if constexpr (KS) {  // what slots -4 .. -1 would have issued
#pragma unroll
            for (int j = 0; j < C::LOADS; j++) {
                if (group == 0) issue_k(0, j), issue_k(2, j), issue_v(0, j);
                else issue_k(1, j), issue_k(3, j);
            }
        } else {
            // (tiles that are there: three of 64 keys at head_dim 128 cost a prompt of 18 rows 0.4 us of 8.5)
            load_all(0);
            if (ntiles > 1) load_all(1);
            if (moves_k && ntiles > 2) load_all(2);
        }
        if constexpr (FOLD) {
#pragma unroll
            for (int kb = 0; kb < QD / 16; kb++) qreg[kb] = Mma<T>::scaled(qreg[kb], pw);
        }
        wait_loads(integral_constant<int, 0>{});
        lds_barrier();
        if (group == 0) {
            // iteration i: S^T(i), softmax(i), P.V(i-1)
            segment0(0, ia, integral_constant<int, 0>{});
            if (ia < ib) {
                segment0(ia, ia + 1, integral_constant<int, 1 | 4 | 16>{});
                segment0(ia + 1, ib, integral_constant<int, 1 | 2 | 4 | 8 | 16>{});
                segment0(ib, ib + 1, integral_constant<int, 2>{});
                segment0(ib + 1, n_iter, integral_constant<int, 0>{});
            } else {
                segment0(ia, n_iter, integral_constant<int, 0>{});
            }
        } else {
            // iteration i: softmax(i-1), then S^T(i) and P.V(i-1)
            segment1(0, ia, integral_constant<int, 0>{});
            if (ia < ib) {
                segment1(ia, ia + 1, integral_constant<int, 1 | 8 | 16>{});
                segment1(ia + 1, ib, integral_constant<int, 1 | 2 | 4 | 8 | 16>{});
                segment1(ib, ib + 1, integral_constant<int, 2 | 4>{});
                segment1(ib + 1, n_iter, integral_constant<int, 0>{});
            } else {
                segment1(ia, n_iter, integral_constant<int, 0>{});
            }
        }
    }

    // the epilogue reuses the tile buffers: no tile load may still be on its way into them
    wait_loads(integral_constant<int, 0>{});
    lds_barrier();
    constexpr int SLICE = 32 * (D * 2 + 16);  // bytes per wavefront of the output transposition below
    if constexpr (KS) {
        // Group 1 hands its state to group 0, which holds the other half of the keys of the same rows:
        // log-sum-exp merge, as the split-KV combine does.  One f32 per lane per slot, above the slices the
        // output transposition uses.
        constexpr int PARK = 4 * SLICE;
        constexpr int NSLOT = D / 2 + 2;
        static_assert(PARK + NSLOT * 1024 <= C::LDS_BYTES, "merge area exceeds the tile buffers");
        auto park = (__attribute__((address_space(3))) float *)(lds_base + PARK) + (wave & 3) * 64 + lane;
        if (group == 1) {
#pragma unroll
            for (int db = 0; db < D / 32; db++)
#pragma unroll
                for (int r = 0; r < 16; r++) park[(db * 16 + r) * 256] = o[db][r];
            park[(D / 2) * 256] = m;
            park[(D / 2 + 1) * 256] = l;
        }
        lds_barrier();
        if (group == 1) return;
        const float m1 = park[(D / 2) * 256], l1 = park[(D / 2 + 1) * 256];
        const float mn = fmaxf(m, m1);
        const float c0 = (m == -INFINITY) ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * rr);
        const float c1 = (m1 == -INFINITY) ? 0.0f : __builtin_amdgcn_exp2f((m1 - mn) * rr);
#pragma unroll
        for (int db = 0; db < D / 32; db++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[db][r] = o[db][r] * c0 + park[(db * 16 + r) * 256] * c1;
        l = l * c0 + l1 * c1;
        m = mn;
    }
    // ---- epilogue: out[query][dim] = O^T[dim][query] / l ----------------------------------------------
    const float l_tot = half_swap_sum(l);
    // With the keys split over workgroups the "output" is this share's row in the partials: O unnormalised
    // as f32 in 16-byte pieces, then (m, l); the merge kernel normalises.
    const bool parked = [&]() __attribute__((always_inline)) {
        if constexpr (CTX) return p.slots > 1;
        else return nks > 1;
    }();
    int64_t row_start = 0;  // CTX: where this lane's row is written
    if constexpr (CTX) row_start = stacked_output(p, row_at, ksplit);
    const float inv = parked ? 1.0f : 1.0f / l_tot;
    const bool dead = !parked && (l_tot == 0.0f);  // no visible key: the reference gives NaN (0/0)
    const bool out_f32 = parked || p.out_f32;
    const int64_t os0 = parked ? (int64_t)p.H * p.Sq * nks * p.pf_pitch : p.os[0];
    const int64_t os1 = parked ? (int64_t)p.Sq * nks * p.pf_pitch : p.os[1];
    const int64_t os2 = parked ? (int64_t)nks * p.pf_pitch : p.os[2];
    char *const og = parked ? (char *)(p.partials + (CTX ? 0 : (int64_t)ksplit * p.pf_pitch)) : (char *)p.out;
    if (parked && query < total_rows && h2 == 0) {
        float *ws;
        if constexpr (CTX) ws = (float *)og + row_start;
        else ws = (float *)og + b * os0 + h * os1 + (int64_t)query * os2;
        ws[hd] = m * rr;  // base-2 exponent units
        ws[hd + 1] = l_tot;
    }
    if (out_vec || parked) {
        // transpose through a wavefront-private slice of the LDS so that every global store is a
        // 16-byte piece of a contiguous row; 32 rows per round for 2-byte outputs, 16 for f32
        const int esz = out_f32 ? 4 : 2;
        const int pitch = D * esz + 16;                      // rows stay 16-byte aligned, 4 banks apart
        static_assert(PF_WAVES * SLICE <= C::LDS_BYTES, "epilogue staging exceeds the tile buffers");
        auto wbase = lds_base + wave * SLICE;
        const int rounds = out_f32 ? 2 : 1;
        const int rows_per_round = 32 / rounds;
        const int cpr = D * esz / 16;
        for (int rd = 0; rd < rounds; rd++) {
            const int row_lo_ = rd * rows_per_round;
            if (ln >= row_lo_ && ln < row_lo_ + rows_per_round) {
#pragma unroll
                for (int db = 0; db < D / 32; db++)
#pragma unroll
                    for (int rq = 0; rq < 4; rq++) {
                        float v4[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) v4[e] = dead ? __builtin_nanf("") : o[db][4 * rq + e] * inv;
                        const int dim = 32 * db + 8 * rq + 4 * h2;
                        if (out_f32) {
                            *(__attribute__((address_space(3))) float4_t *)(wbase + (ln - row_lo_) * pitch + dim * 4) =
                                float4_t{v4[0], v4[1], v4[2], v4[3]};
                        } else {
                            const uint2_t pk2 = {Mma<T>::pack2(v4[0], v4[1]), Mma<T>::pack2(v4[2], v4[3])};
                            *(__attribute__((address_space(3))) uint2_t *)(wbase + ln * pitch + dim * 2) = pk2;
                        }
                    }
            }
            wave_lds_sync();
            for (int c = lane; c < rows_per_round * cpr; c += 64) {
                const int row = c / cpr, col = c % cpr;
                const int qr = qw0 + row_lo_ + row;
                int64_t start = 0;
                if constexpr (CTX) start = lane_value(row_start, row_lo_ + row);
                if (qr < total_rows && (!PAD || col * 16 < hd * esz)) {
                    const uint4_t val = *(__attribute__((address_space(3))) uint4_t *)(wbase + row * pitch + col * 16);
                    int64_t eidx;
                    if constexpr (CTX) eidx = start;
                    else eidx = b * os0 + h * os1 + (int64_t)qr * os2;
                    *(uint4_t *)(og + eidx * esz + col * 16) = val;
                }
            }
            wave_lds_sync();
        }
    } else if (query < total_rows) {
        int64_t obase;
        if constexpr (CTX) obase = row_start;
        else obase = b * p.os[0] + h * p.os[1] + (int64_t)query * p.os[2];
#pragma unroll
        for (int db = 0; db < D / 32; db++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int dim = 32 * db + 8 * (r >> 2) + 4 * h2 + (r & 3);
                if (PAD && dim >= hd) continue;
                const float val = dead ? __builtin_nanf("") : o[db][r] * inv;
                if (p.out_f32) ((float *)p.out)[obase + dim * p.os[3]] = val;
                else ((T *)p.out)[obase + dim * p.os[3]] = from_float<T>(val);
            }
    }
}

}  // namespace fhip
