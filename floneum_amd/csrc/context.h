// Internal declarations of attention over a context in two parts (a prefix that the batch shares, the sequences' own keys): what its kernels
// receive, how its calls are planned, and its launchers.
#pragma once
#include "common.h"

namespace fhip {

// A tiled kernel's rows and tiles: rows of a KV head are stacked, see context_tiles.h; the tiles of their visible keys are dealt to `shares` of `chunk`
// tiles.
struct ContextTilesJob {
    int32_t fold;                   // rows of all sequences together (on the prefix alone)
    int32_t with_prefix, with_own;
    int32_t units, rows, blocks;    // KV heads (times the batch, if not folded), stacked rows of each, workgroups that these fill
    int32_t shares, chunk;
    int32_t slot0;                  // of the first share
};
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
    // tiled kernels: workgroups from `second` on take the other job
    ContextTilesJob job, other;
    int32_t second;
};
struct ContextBoth : ContextParams {};  // of a launch that takes both parts

// The kernel for few rows.  A job streams one part's keys for columns, (query row, head of the group) pairs of a KV head: of one sequence
// (its own keys), or of all of them (the prefix).
struct ContextRowsJob {
    int32_t prefix;  // else the sequences' own keys
    int32_t units;   // KV heads, times the batch for own keys
    int32_t blocks;  // column blocks of a unit
    int32_t nsplit, chunk;  // shares of the visible keys, `chunk` keys each (more where that is too little for all)
    int32_t slot0;
};
struct ContextRows {
    ContextRowsJob job[2];
    int32_t second;  // first workgroup of job[1]
    int32_t total;   // workgroups
    int32_t columns; // of a workgroup: 16 or 32
};

// A launch of a tiled kernel.
struct ContextTilesLaunch {
    int32_t rows_per_group;  // stacked rows of a workgroup
    int32_t key_groups;      // wavefronts of a workgroup that share its rows, see the kernels
    int32_t jobs;            // 0: no launch
    ContextTilesJob job[2];
    int32_t second, total;   // workgroups of job[0], of both
};
inline void set_tiles_launch(ContextParams &p, const ContextTilesLaunch &how) { p.job = how.job[0], p.other = how.job[1], p.second = how.second; }

// A launch has less than 2^32 threads in a dimension: the workgroups of one with a workgroup for every few rows in two.
inline dim3 rows_grid(int64_t workgroups) {
    const int64_t x = workgroups < 1 << 22 ? workgroups : 1 << 22;
    return dim3((unsigned)x, (unsigned)((workgroups + x - 1) / x));
}

// What a call runs, in this order, and the merge where a row has several places.
struct ContextPlan {
    bool any;  // the kernel that takes every call, alone
    ContextTilesLaunch tiles;
    ContextRows rows;  // total 0: none
    int slots;
    size_t bytes;  // of workspace
    double us;     // estimated
};
// A call, or its first query rows and then the others; both use the same workspace.
struct ContextCall {
    int parts;
    int first_row[2], rows[2];
    ContextPlan plan[2];
    size_t bytes;
};
ContextCall context_call(const ContextParams &p, fhip_dtype dtype);

int launch_context_any(const ContextParams &p, fhip_dtype dtype, hipStream_t stream);
bool context_rows_takes(const ContextParams &p, fhip_dtype dtype);
int launch_context_rows(const ContextParams &p, const ContextRows &rows, fhip_dtype dtype, hipStream_t stream);
bool context_tiles_takes(const ContextParams &p, fhip_dtype dtype);
int launch_context_tiles(const ContextParams &p, const ContextTilesLaunch &how, fhip_dtype dtype, hipStream_t stream);
bool context_terms_takes(const ContextParams &p, fhip_dtype dtype);
int launch_context_wide(const ContextParams &p, const ContextTilesLaunch &how, fhip_dtype dtype, hipStream_t stream);  // one part
int launch_context_terms(const ContextParams &p, const ContextTilesLaunch &how, hipStream_t stream);
int launch_context_merge(const ContextParams &p, fhip_dtype dtype, hipStream_t stream);

}  // namespace fhip
