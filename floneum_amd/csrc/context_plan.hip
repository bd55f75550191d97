// Attention over a context in two parts: which kernels a call runs, and in how many shares of its keys.
#include <algorithm>
#include <cstring>

#include "context.h"

namespace fhip {

static int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Visible keys of a part at most: all of them, or what the rows' windows and the first tokens take (a window that ends at the rows' own positions;
// without a causal mask it has no end).
static int64_t most_visible(const ContextParams &p, int64_t keys, int64_t rows, int64_t first) {
    if (!p.causal || p.window == 0 || p.window >= keys) return keys;
    return std::min(keys, p.window + rows - 1 + first);
}

static ContextRowsJob rows_job(const ContextParams &p, bool prefix, int columns, int step, int64_t target) {
    ContextRowsJob job;
    job.prefix = prefix;
    job.units = prefix ? p.Hkv : p.B * p.Hkv;
    job.blocks = (int32_t)div_up((int64_t)(prefix ? p.B : 1) * p.G * p.Sq, columns);
    // (rows of a batch may stand anywhere over the prefix)
    const int64_t keys = prefix ? (p.q_positions ? (int64_t)p.P : most_visible(p, p.P, p.Sq, p.sinks))
                                : most_visible(p, p.Skv, p.Sq, std::max<int64_t>((int64_t)p.sinks - p.P, 0));
    const int64_t workgroups = (int64_t)job.units * job.blocks;
    int64_t shares = std::min(div_up(target, std::max<int64_t>(workgroups, 1)), div_up(keys, step));
    shares = std::max(shares, div_up(keys, 1024));
    shares = std::max<int64_t>(shares, 1);
    job.chunk = (int32_t)(div_up(div_up(keys, shares), step) * step);
    job.chunk = std::max(job.chunk, step);
    job.nsplit = (int32_t)std::max<int64_t>(div_up(keys, job.chunk), 1);
    job.slot0 = 0;
    return job;
}
static int64_t workgroups_of(const ContextRowsJob &job) {
    const int64_t shares = (int64_t)job.units * job.nsplit;
    return job.blocks == 1 ? shares : div_up(shares, 8) * 8 * job.blocks;
}

ContextPlan context_plan(const ContextParams &p, fhip_dtype dtype) {
    ContextPlan plan;
    memset(&plan, 0, sizeof(plan));
    plan.any = true;
    if (!context_rows_takes(p, dtype)) return plan;
    const int64_t most = (int64_t)p.G * p.Sq * (p.P > 0 ? p.B : 1);
    ContextRows &rows = plan.rows;
    rows.columns = most > 16 && p.D <= 128 ? 32 : 16;
    const int step = dtype == FHIP_F32 ? 64 : 128;
    const int64_t target = (int64_t)p.cus * (p.D > 128 ? 1 : 2);
    int jobs = 0;
    int64_t total = 0, slots = 0;
    for (const bool prefix : {true, false}) {
        if ((prefix ? p.P : p.Skv) == 0) continue;
        ContextRowsJob job = rows_job(p, prefix, rows.columns, step, target);
        job.slot0 = (int32_t)slots;
        slots += job.nsplit;
        if (jobs == 1) rows.second = (int32_t)total;
        rows.job[jobs++] = job;
        total += workgroups_of(job);
    }
    if (jobs == 1) rows.second = (int32_t)total;
    if (total > 0x7fffffff || slots > 0x7fffffff) return plan;
    rows.total = (int32_t)total;
    plan.any = false;
    plan.slots = (int)slots;
    if (slots > 1) plan.bytes = (size_t)p.B * p.H * p.Sq * (size_t)slots * (size_t)(p.D + 4) * sizeof(float);
    return plan;
}

}  // namespace fhip
