// Device code that the kernels of attention over a context in two parts share: which keys a query row sees.
#pragma once
#include "context.h"
#include "device_utils.h"

namespace fhip {

constexpr float CONTEXT_LOG2E = 1.4426950408889634f;

// Keys are numbered through both parts: j < P is row j of the prefix, the others row j - P of the sequence's own.  A row sees
// [0, first) and [lo, hi), with first <= lo <= hi.
struct ContextRow {
    int first, lo, hi;
    __device__ __forceinline__ ContextRow of(const ContextParams &p, bool prefix) const;  // within one part, in rows of that part
    __device__ __forceinline__ ContextRow uniform() const {
        return {__builtin_amdgcn_readfirstlane(first), __builtin_amdgcn_readfirstlane(lo), __builtin_amdgcn_readfirstlane(hi)};
    }
};
// what a sequence brings
struct ContextSequence {
    int keys;    // of both parts
    int64_t at;  // position of its first row
    __device__ __forceinline__ ContextRow row(const ContextParams &p, int i) const {
        ContextRow r;
        r.hi = p.causal ? (int)min((int64_t)keys, max(at + i + 1, (int64_t)0)) : keys;
        r.lo = p.window > 0 ? (int)min((int64_t)r.hi, max(at + i - p.window + 1, (int64_t)0)) : 0;
        r.first = min(p.sinks, r.lo);
        return r;
    }
};
__device__ __forceinline__ ContextSequence context_sequence(const ContextParams &p, int b) {
    const int own = p.kv_lens ? p.kv_lens[b] : p.Skv, start = p.q_positions ? p.q_positions[b] : 0;
    return {p.P + min(max(own, 0), p.Skv), p.q_pos_offset + start};
}
__device__ __forceinline__ ContextRow context_row(const ContextParams &p, int b, int row) { return context_sequence(p, b).row(p, row); }
__device__ __forceinline__ int part_row(const ContextParams &p, bool prefix, int key) { return prefix ? min(key, p.P) : max(key - p.P, 0); }
__device__ __forceinline__ ContextRow ContextRow::of(const ContextParams &p, bool prefix) const {
    return {part_row(p, prefix, first), part_row(p, prefix, lo), part_row(p, prefix, hi)};
}

// What some row of several sees: [0, first) and [lo, hi) again.  Rows that see nothing do not count.
struct ContextSpan {
    int first, lo, hi;
    // visible keys in order: key v, or v + gap from `first` on
    __device__ __forceinline__ int keys() const { return first + max(hi - lo, 0); }
    __device__ __forceinline__ int gap() const { return lo - first; }
    // the first visible key and the one behind the last (of a span that has some)
    __device__ __forceinline__ int begin() const { return first > 0 ? 0 : lo; }
    __device__ __forceinline__ int end() const { return lo < hi ? hi : first; }
    __device__ __forceinline__ ContextSpan of(const ContextParams &p, bool prefix) const {
        return {part_row(p, prefix, first), part_row(p, prefix, lo), part_row(p, prefix, hi)};
    }
};
// of the rows that the lanes of a wavefront hold
__device__ __forceinline__ ContextSpan context_span(const ContextRow &r) {
    const bool none = r.first == 0 && r.lo >= r.hi;
    ContextSpan s;
    s.first = __builtin_amdgcn_readfirstlane(wave_reduce_i(r.first, [](int x, int y) { return max(x, y); }));
    s.lo = __builtin_amdgcn_readfirstlane(wave_reduce_i(none ? 0x7fffffff : r.lo, [](int x, int y) { return min(x, y); }));
    s.hi = __builtin_amdgcn_readfirstlane(wave_reduce_i(none ? 0 : r.hi, [](int x, int y) { return max(x, y); }));
    s.lo = max(s.lo, s.first);
    if (s.hi < s.lo) s.hi = s.lo = s.first;
    return s;
}

}  // namespace fhip
