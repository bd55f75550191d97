// Device code of the tiled kernels of attention over a context in two parts: which rows and which tiles of keys a workgroup takes.
#pragma once
#include <type_traits>

#include "context_device.h"

namespace fhip {

// The workgroup's place in its job, which p.job is from here on.
template <class P>
__device__ __forceinline__ uint32_t tiles_work(P &p) {
    if constexpr (!std::is_same<P, ContextBoth>::value) {
        if ((int)blockIdx.x >= p.second) {
            p.job = p.other;
            return blockIdx.x - p.second;
        }
    }
    return blockIdx.x;
}

// Stacked rows of a KV head: the heads of its group within a query row, query rows within a sequence, and where the rows of all sequences meet
// the prefix together (fold) sequences behind each other.
struct StackedRow {
    int b, h, row;
};
__device__ __forceinline__ StackedRow stacked_row(const ContextParams &p, int b, int g, int r) {
    const int query = p.G == 1 ? r : (int)((uint32_t)r / (uint32_t)p.G), head = g * p.G + r - query * p.G;
    if (b >= 0) return {b, head, query};
    const int seq = (int)((uint32_t)query / (uint32_t)p.Sq);
    return {seq, head, query - seq * p.Sq};
}

// Of stacked rows: what some of them sees, and what all of them see, the latter as the least `first`, the largest `lo` and the least `hi`.
struct StackedSpan {
    ContextSpan some;
    ContextRow all;
    __device__ __forceinline__ StackedSpan of(const ContextParams &p, bool prefix) const {
        return {some.of(p, prefix), all.of(p, prefix)};
    }
};
// Of the wavefront's 32 rows from qw0 on and of the workgroup's BM rows from q0 on; sees: of the lane's row, qw0 + lane % 32.  What the sequences bring is
// asked for once and together: each time it is waited for costs a launch of few tiles a memory latency.
template <int BM>
__device__ __forceinline__ void stacked_spans(const ContextParams &p, int b, int q0, int qw0, int lane, const StackedRow &at, StackedSpan &wave, ContextSpan &wg,
                                              ContextRow &sees) {
    const int last = p.job.rows - 1;
    if (b >= 0) {  // a sequence's rows: both ends move forward with the row
        const ContextSequence s = context_sequence(p, b);
        auto query = [&](int r) __attribute__((always_inline)) { return p.G == 1 ? min(r, last) : min(r, last) / p.G; };
        auto between = [&](int r0, int r1) __attribute__((always_inline)) {
            const ContextRow x = s.row(p, query(r0)).uniform(), y = s.row(p, query(r1)).uniform();
            const int lo = max(x.lo, y.first);
            return StackedSpan{{y.first, lo, max(y.hi, lo)}, {x.first, y.lo, x.hi}};
        };
        sees = s.row(p, at.row);
        wave = between(qw0, qw0 + 31);
        wg = between(q0, q0 + BM - 1).some;
        return;
    }
    constexpr int N = (BM + 63) / 64;
    ContextSequence s[N], mine = context_sequence(p, at.b);
    int row[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const StackedRow x = stacked_row(p, -1, 0, min(q0 + min(lane + 64 * i, BM - 1), last));
        row[i] = x.row, s[i] = context_sequence(p, x.b);
    }
    auto least = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(wave_reduce_i(x, [](int a, int c) { return min(a, c); })); };
    auto most = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(wave_reduce_i(x, [](int a, int c) { return max(a, c); })); };
    sees = mine.row(p, at.row);
    if (p.window == 0) {  // [0, hi) each
        int hi = 0;
#pragma unroll
        for (int i = 0; i < N; i++) hi = max(hi, s[i].row(p, row[i]).hi);
        wg = {0, 0, most(hi)};
        wave = {{0, 0, most(sees.hi)}, {0, 0, least(sees.hi)}};
        return;
    }
    int first = 0, lo = 0x7fffffff, hi = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const ContextRow x = s[i].row(p, row[i]);
        first = max(first, x.first), hi = max(hi, x.hi);
        if (x.first > 0 || x.lo < x.hi) lo = min(lo, x.lo);
    }
    auto span = [&](int f, int l, int h) __attribute__((always_inline)) {
        ContextSpan r;
        r.first = most(f), r.lo = max(least(l), r.first), r.hi = max(most(h), r.lo);
        if (r.lo == 0x7fffffff) r.lo = r.hi = 0;
        return r;
    };
    wg = span(first, lo, hi);
    wave.some = span(sees.first, sees.first > 0 || sees.lo < sees.hi ? sees.lo : 0x7fffffff, sees.hi);
    wave.all = ContextRow{least(sees.first), most(sees.lo), least(sees.hi)};
}

// The tiles of KEYS keys that hold what some row sees, in order.  Tiles start at multiples of KEYS rows of their tensor, and none is listed twice.
// Of one part, in its rows: up to `first`, then from `lo` on.
template <int KEYS>
struct ContextTiles {
    int end0;          // tiles [0, end0) and [end0, count)
    int from0, from1;  // tile t starts at row KEYS t + from
    int count;
    static constexpr int SHIFT = KEYS == 64 ? 6 : 5;
    static_assert(1 << SHIFT == KEYS, "");

    __device__ __forceinline__ int row(int t) const { return KEYS * t + (t < end0 ? from0 : from1); }
    // rows of these may lie between first and lo
    __device__ __forceinline__ bool edge(int t) const { return t == end0 - 1 || t == end0; }
    // the tile that holds a key that is seen (below 0, or count and more: it is another share's)
    __device__ __forceinline__ int holding(const ContextParams &, int key) const {
        const int t = (key - from0) >> SHIFT;
        return t < end0 ? t : (key - from1) >> SHIFT;
    }
    __device__ __forceinline__ void set(const ContextParams &p, const ContextSpan &s, int share) {
        const int n0 = (s.first + KEYS - 1) >> SHIFT, s1 = max(s.lo >> SHIFT, n0);
        const int n1 = s.hi > s.lo ? max(((s.hi + KEYS - 1) >> SHIFT) - s1, 0) : 0;
        const int t0 = share * p.job.chunk, left = n0 + n1 - t0;
        end0 = n0 - t0, from0 = KEYS * t0, from1 = KEYS * (s1 - n0 + t0);
        count = max(share + 1 < p.job.shares ? min(left, p.job.chunk) : left, 0);
    }
};
// Of both parts, keys numbered through them: the prefix's up to `first`, then either the prefix's from `lo` on or own ones up to `first`, then own ones
// from `lo` on.
template <int KEYS>
struct ContextBothTiles {
    int end0, end1;           // tiles [0, end0), [end0, end1) and [end1, count)
    int from0, from1, from2;  // tile t starts at row KEYS t + from of its tensor
    bool own1;                // the second run lies in the own keys
    int count;
    static constexpr int SHIFT = ContextTiles<KEYS>::SHIFT;

    __device__ __forceinline__ int row(int t) const { return KEYS * t + (t < end0 ? from0 : t < end1 ? from1 : from2); }
    __device__ __forceinline__ bool own(int t) const { return t >= end1 || (own1 && t >= end0); }
    __device__ __forceinline__ bool edge(int t) const { return t == end0 - 1 || t == end0 || t == end1 - 1 || t == end1; }
    __device__ __forceinline__ int holding(const ContextParams &p, int key) const {
        if (key < p.P) {
            const int t = (key - from0) >> SHIFT;
            return t < end0 ? t : (key - from1) >> SHIFT;
        }
        const int t = (key - p.P - from1) >> SHIFT;
        return own1 && t < end1 ? t : (key - p.P - from2) >> SHIFT;
    }
    __device__ __forceinline__ void set(const ContextParams &p, const ContextSpan &s, int share) {
        const ContextSpan a = s.of(p, true), b = s.of(p, false);
        const int n0 = (a.first + KEYS - 1) >> SHIFT;
        int n1 = 0, s1 = 0, n2 = 0, s2 = 0;
        own1 = b.first > 0;
        if (own1) n1 = (b.first + KEYS - 1) >> SHIFT;
        else if (a.hi > a.lo) s1 = max(a.lo >> SHIFT, n0), n1 = max(((a.hi + KEYS - 1) >> SHIFT) - s1, 0);
        if (b.hi > b.lo) s2 = max(b.lo >> SHIFT, own1 ? n1 : 0), n2 = max(((b.hi + KEYS - 1) >> SHIFT) - s2, 0);
        const int t0 = share * p.job.chunk, left = n0 + n1 + n2 - t0;
        end0 = n0 - t0, end1 = n0 + n1 - t0;
        from0 = KEYS * t0, from1 = KEYS * (s1 - n0 + t0), from2 = KEYS * (s2 - n0 - n1 + t0);
        count = max(share + 1 < p.job.shares ? min(left, p.job.chunk) : left, 0);
    }
};

// Where this lane's row of the result, or of the shares, starts, in elements.
__device__ __forceinline__ int64_t stacked_output(const ContextParams &p, const StackedRow &at, int share) {
    if (p.slots > 1) return ((((int64_t)at.b * p.H + at.h) * p.Sq + at.row) * p.slots + p.job.slot0 + share) * p.pf_pitch;
    return at.b * p.os[0] + at.h * p.os[1] + at.row * p.os[2];
}
__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
    return (int64_t)(((uint64_t)(uint32_t)__shfl((int)(x >> 32), lane, 64) << 32) | (uint32_t)__shfl((int)x, lane, 64));
}

}  // namespace fhip
