// Internal declarations of attention over a context in two parts (a prefix that the batch shares, the sequences' own keys): what its kernels
// receive, how its calls are planned, and its launchers.
#pragma once
#include "common.h"

namespace fhip {

// k, v, Skv, kv_lens of AttnParams are the sequences' own; q_pos_offset and window as there, positions counted from the prefix's first key.
struct ContextParams : AttnParams {
    const void *pk, *pv;     // the prefix, [Hkv, P, D]
    int64_t pks[3], pvs[3];  // strides: head, row, dim
    int32_t P;
    int32_t sinks;           // first keys that the window does not hide
    const int32_t *q_positions;
    // shares of the keys: every (sequence, head, query row) has `slots` places in `partials`, each pf_pitch floats: D values, the
    // reference exponent (base 2) and the sum of the weights
    int32_t slots;
};

int launch_context_any(const ContextParams &p, fhip_dtype dtype, hipStream_t stream);

}  // namespace fhip
