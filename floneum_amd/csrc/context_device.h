// Device code that the kernels of attention over a context in two parts share: which keys a query row sees.
#pragma once
#include "context.h"
#include "device_utils.h"

namespace fhip {

// Keys are numbered through both parts: j < P is row j of the prefix, the others row j - P of the sequence's own.  A row sees
// [0, first) and [lo, hi), with first <= lo <= hi.
struct ContextRow {
    int first, lo, hi;
};
__device__ __forceinline__ ContextRow context_row(const ContextParams &p, int b, int row) {
    const int own = p.kv_lens ? min(max(p.kv_lens[b], 0), p.Skv) : p.Skv;
    const int64_t at = p.q_pos_offset + (p.q_positions ? p.q_positions[b] : 0) + row;
    ContextRow r;
    r.hi = p.P + own;
    if (p.causal) r.hi = (int)min((int64_t)r.hi, max(at + 1, (int64_t)0));
    r.lo = p.window > 0 ? (int)min((int64_t)r.hi, max(at - p.window + 1, (int64_t)0)) : 0;
    r.first = min(p.sinks, r.lo);
    return r;
}

}  // namespace fhip
