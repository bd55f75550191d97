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

static int64_t part_keys(const ContextParams &p, bool prefix) {
    // (rows of a batch may stand anywhere over the prefix)
    if (prefix) return p.q_positions ? (int64_t)p.P : most_visible(p, p.P, p.Sq, p.sinks);
    return most_visible(p, p.Skv, p.Sq, std::max<int64_t>((int64_t)p.sinks - p.P, 0));
}
static ContextRowsJob rows_job(const ContextParams &p, bool prefix, int columns, int step, int64_t target) {
    ContextRowsJob job;
    job.prefix = prefix;
    job.units = prefix ? p.Hkv : p.B * p.Hkv;
    job.blocks = (int32_t)div_up((int64_t)(prefix ? p.B : 1) * p.G * p.Sq, columns);
    const int64_t keys = part_keys(p, prefix);
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

// Time of a launch of the 16-bit kernels in us, from the constants of prefill_mfma_time (attn_prefill_mfma.hip) and prefill_wide_time
// (attn_prefill_mfma_wide.hip): rounds of workgroups that walk their tiles of 64 keys, above head_dim 128 32.
static double tiles_time(const ContextParams &p, const ContextTilesLaunch &how, int64_t keys) {
    const int64_t wgs = (int64_t)how.units * div_up(how.rows, how.rows_per_group) * how.shares, rounds = div_up(wgs, p.cus);
    if (p.D > 128) return 5.0 + rounds * (6.5 + 0.70 * div_up(div_up(keys, how.shares), 32));
    const double dims = p.D <= 64 ? 1.0 : p.D <= 96 ? 1.43 : 1.86, tiles = (double)div_up(div_up(keys, how.shares), 64);
    return 4.6 + rounds * (how.rows_per_group == 128 ? 5.3 + 0.356 * dims * tiles : 3.9 + 0.579 * dims * tiles);
}
static ContextTilesLaunch tiles_launch(const ContextParams &p, fhip_dtype dtype, bool fold, bool with_prefix, bool with_own, bool parked) {
    const bool f32 = dtype == FHIP_F32, both = with_prefix && with_own;
    const int tile = f32 || p.D > 128 ? 32 : 64;
    // (rows per workgroup, key groups); to head_dim 128 the 16-bit form of 128 rows takes one part
    static const int FORMS[3][3][2] = {{{256, 1}, {128, 2}, {0, 0}}, {{128, 1}, {0, 0}, {0, 0}}, {{128, 1}, {128, 2}, {64, 2}}};
    ContextTilesLaunch best, how;
    memset(&how, 0, sizeof(how));
    how.fold = fold, how.with_prefix = with_prefix, how.with_own = with_own;
    how.units = fold ? p.Hkv : p.B * p.Hkv;
    how.rows = (fold ? p.B : 1) * p.G * p.Sq;
    best = how;
    double least = 0.0;
    for (const auto &form : FORMS[f32 ? 2 : p.D > 128 ? 1 : 0]) {
        if (form[0] == 0 || (!f32 && p.D <= 128 && form[0] == 128 && both) || (f32 && p.D > 128 && form[1] > 1)) continue;
        how.rows_per_group = form[0], how.key_groups = form[1];
        const int64_t positions = std::min<int64_t>(p.Sq, form[0] / p.G + 2);
        int64_t keys = 0;
        if (with_prefix) keys += fold ? part_keys(p, true) : most_visible(p, p.P, positions, p.sinks);
        if (with_own) keys += most_visible(p, p.Skv, positions, std::max<int64_t>((int64_t)p.sinks - p.P, 0));
        if (both && p.causal && p.window > 0) keys = std::min(keys, p.window + positions + p.sinks);
        const int64_t tiles = std::max<int64_t>(div_up(keys, tile), 1), wgs = (int64_t)how.units * div_up(how.rows, form[0]);
        for (int64_t shares = 1; shares <= tiles; shares++) {
            if (shares > 1 && wgs * shares > 3 * p.cus) break;
            how.chunk = (int32_t)div_up(tiles, shares);
            how.shares = (int32_t)div_up(tiles, how.chunk);
            if (how.shares != shares) continue;
            double us;
            if (f32) {
                const TermsCall call = {1, how.units, 1, how.rows, (int)keys, p.D, p.cus, false, 0, true, false};
                us = prefill_f32_terms_time(call, {form[0] / 32, form[1]}, how.shares);
                if (how.shares > 1) us -= prefill_f32_merge_time(call, how.shares);
            } else {
                us = tiles_time(p, how, keys);
            }
            if (how.shares > 1 || parked) us += 0.488e-6 * (double)p.B * p.H * p.Sq * how.shares * (p.D + 4) * sizeof(float);
            if (how.shares > 1 && !parked) us += 3.0;
            if (least == 0.0 || us < 0.98 * least) least = us, best = how;
        }
    }
    return best;
}

ContextPlan context_plan(const ContextParams &p, fhip_dtype dtype) {
    ContextPlan plan;
    memset(&plan, 0, sizeof(plan));
    plan.any = true;
    if (!context_rows_takes(p, dtype)) return plan;
    const bool tiles = context_tiles_takes(p, dtype) || context_terms_takes(p, dtype);
    const int64_t each = (int64_t)p.G * p.Sq;  // columns of a sequence and KV head
    // rows of all sequences meet the prefix together where they see one run of it
    const bool can_fold = p.P > 0 && p.B > 1 && (p.window == 0 || !p.q_positions);
    const bool own_by_rows = !tiles || each <= (dtype == FHIP_F32 ? 64 : 32);
    const bool one_part = dtype != FHIP_F32 && p.D > 128;  // the tiled kernel takes one part per launch
    bool prefix_by_rows = p.P > 0 && (!tiles || (own_by_rows && (each * p.B <= (dtype == FHIP_F32 ? 64 : 32) || !can_fold)));
    int64_t slots = 0;
    auto add_tiles = [&](bool fold, bool with_prefix, bool with_own, bool parked) {
        ContextTilesLaunch &how = plan.tiles[plan.tile_launches++];
        how = tiles_launch(p, dtype, fold, with_prefix, with_own, parked);
        how.slot0 = (int32_t)slots;
        slots += how.shares;
    };
    if (p.P > 0 && !prefix_by_rows) {
        if (own_by_rows) add_tiles(p.B > 1, true, false, p.Skv > 0);
        else if ((can_fold && each < 128) || (one_part && p.Skv > 0))
            add_tiles(can_fold, true, false, true), add_tiles(false, false, true, true);
        else add_tiles(false, true, p.Skv > 0, false);
    } else if (!own_by_rows) {
        add_tiles(false, false, true, false);
    }
    if (own_by_rows) {
        ContextRows &rows = plan.rows;
        const int64_t most = each * (prefix_by_rows ? p.B : 1);
        rows.columns = most > 16 && p.D <= 128 ? 32 : 16;
        const int step = dtype == FHIP_F32 ? 64 : 128;
        const int64_t target = (int64_t)p.cus * (p.D > 128 ? 1 : 2);
        int jobs = 0;
        int64_t total = 0;
        for (const bool prefix : {true, false}) {
            if (prefix ? !prefix_by_rows : p.Skv == 0) continue;
            ContextRowsJob job = rows_job(p, prefix, rows.columns, step, target);
            job.slot0 = (int32_t)slots;
            slots += job.nsplit;
            if (jobs == 1) rows.second = (int32_t)total;
            rows.job[jobs++] = job;
            total += workgroups_of(job);
        }
        if (jobs == 1) rows.second = (int32_t)total;
        if (total > 0x7fffffff) return plan;
        rows.total = (int32_t)total;
    }
    for (int i = 0; i < plan.tile_launches; i++) {
        const ContextTilesLaunch &how = plan.tiles[i];
        if ((int64_t)how.units * div_up(how.rows, how.rows_per_group) * how.shares > 0x7fffffff) return plan;
        if (dtype == FHIP_F32 && (how.units > 65535 || div_up(how.rows, how.rows_per_group) > 65535)) return plan;  // (dimensions of its grid)
    }
    if (slots > 0x7fffffff) return plan;
    plan.any = false;
    plan.slots = (int)slots;
    if (slots > 1) plan.bytes = (size_t)p.B * p.H * p.Sq * (size_t)slots * (size_t)(p.D + 4) * sizeof(float);
    return plan;
}

}  // namespace fhip
