// Attention over a context in two parts: which kernels a call runs, and in how many shares of its keys.
#include <algorithm>
#include <cstring>
#include <initializer_list>

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
// Writing shares' results and reading them again.
static double partials_us(const ContextParams &p, int64_t slots) { return 0.488e-6 * (double)p.B * p.H * p.Sq * (double)slots * (p.D + 4) * sizeof(float); }

// Workgroups of a job of the launch for few rows, in rounds of what the chip holds, beyond which its keys are dealt to no more shares: what a call asks for as workspace and
// writes and reads again is then bounded by the chip, not by rows times keys, and sequences that hold little of a long view, or see little of a long prefix, do not merge
// hundreds of empty shares.  Against shares of at most 8 steps however many: 64 sequences of 200 to 1000 keys in a view of 32768, f16, 32/8 heads at 128, 37 us
// instead of 83 (8 rounds: 48), 16 in f32 under windows of 1000 on a prefix of 100000 41 (68; 55), 16384 keys of 32 sequences 323 (336; 336); 24 other calls 0.78 to 1.04.
constexpr int64_t SHARE_ROUNDS = 4;

// The launch for few rows: its jobs and their shares, and its time in us with the merge's.
struct RowsPlan {
    ContextRows rows;
    int64_t slots;
    double us;
};
static RowsPlan rows_launch_of(const ContextParams &p, fhip_dtype dtype, bool with_prefix, int64_t slots_before, int columns) {
    const int64_t each = (int64_t)p.G * p.Sq, most = each * (with_prefix ? p.B : 1);
    const bool f32 = dtype == FHIP_F32;
    const int step = f32 || p.D > 128 ? 64 : 128, size = f32 ? 4 : 2;
    // Fitted to 101 calls at six lengths of the shares each, and 40 at eight above head_dim 128; the shares it picks are 1.5 per cent slower than each call's best in the mean, 12 at most.
    // A step of a workgroup, what all of them take in from the caches and from memory, bytes per us,
    // and workgroups per CU.  0.3 of the longest share is left over at the end.
    const double step_us = f32 ? 0.24 + 0.0119 * p.D : p.D > 128 ? 0.36 + 0.0028 * p.D : 0.35 + 0.0063 * p.D;
    const double cached = f32 ? 10e6 : 10.8e6, memory = 6.2e6;  // (above head_dim 128 up to 14e6: tiles then pass for slower than they are)
    const double start_us = 2.7 + (columns == 32 ? 0.03 * p.D : 0.0);
    const int64_t at_once = (int64_t)p.cus * (p.D > 128 && f32 ? 1 : p.D > 64 ? 2 : 3);
    RowsPlan best;
    memset(&best, 0, sizeof(best));  // (us 0: too many workgroups for a launch)
    for (int steps = 1; steps <= (f32 || p.D <= 128 ? 8 : 16); steps++) {
        RowsPlan plan;
        memset(&plan, 0, sizeof(plan));
        plan.rows.columns = columns;
        plan.slots = slots_before;
        const int64_t chunk = (int64_t)steps * step;
        int64_t total = 0, workgroups = 0, all_steps = 0, longest = 0;
        double taken = 0.0, read = 0.0;
        int jobs = 0;
        for (const bool prefix : {true, false}) {
            if (prefix ? !with_prefix : p.Skv == 0) continue;
            ContextRowsJob &job = plan.rows.job[jobs];
            const int64_t keys = part_keys(p, prefix);
            job.prefix = prefix;
            job.units = prefix ? p.Hkv : p.B * p.Hkv;
            job.blocks = (int32_t)div_up(prefix ? most : each, columns);
            job.chunk = (int32_t)chunk;
            // (the kernel deals longer shares where these do not hold all keys)
            job.nsplit = (int32_t)std::max<int64_t>(std::min(div_up(keys, chunk), SHARE_ROUNDS * at_once / ((int64_t)job.units * job.blocks)), 1);
            job.slot0 = (int32_t)plan.slots;
            plan.slots += job.nsplit;
            const int64_t shares = (int64_t)job.units * job.nsplit;
            if (jobs++ == 1) plan.rows.second = (int32_t)total;
            total += job.blocks == 1 ? shares : div_up(shares, 8) * 8 * job.blocks;
            const int64_t walked = std::max<int64_t>(std::max(std::min<int64_t>(div_up(keys, step), steps), div_up(div_up(keys, job.nsplit), step)), 1);
            workgroups += shares * job.blocks;
            all_steps += shares * job.blocks * walked;
            longest = std::max(longest, walked);
            taken += (double)job.units * job.blocks * keys * p.D * 2 * size;
            read += (double)job.units * keys * p.D * 2 * size;
        }
        if (total >= 1 << 24) continue;  // (2^32 threads)
        if (jobs == 1) plan.rows.second = (int32_t)total;
        plan.rows.total = (int32_t)total;
        const double last = step_us * (double)longest;
        plan.us = start_us + (double)div_up(workgroups, at_once) * (f32 && p.D > 128 ? 4.5 : 2.8) + 0.3 * last +
                  std::max({last, step_us * (double)all_steps / (double)at_once, taken / cached, read / memory});
        if (plan.slots > 1) plan.us += 1.5 + partials_us(p, plan.slots - slots_before);
        if (best.us == 0.0 || plan.us < best.us) best = plan;
    }
    return best;
}

// 32 columns halve what is taken in for a unit with so many, but the other part's few columns pay for them too: 32 sequences on 8192 keys at head_dim 128
// take 26.2 us with 32 and 37.5 with 16, on 512 keys 18.0 and 14.9.  f32 tensors take 16 (faster in 60 of 60 calls, by up to a third).
static RowsPlan rows_launch(const ContextParams &p, fhip_dtype dtype, bool with_prefix, int64_t slots_before) {
    const RowsPlan one = rows_launch_of(p, dtype, with_prefix, slots_before, 16);
    if ((int64_t)p.G * p.Sq * (with_prefix ? p.B : 1) <= 16 || p.D > 128 || dtype == FHIP_F32) return one;
    const RowsPlan two = rows_launch_of(p, dtype, with_prefix, slots_before, 32);
    return two.us == 0.0 || (one.us != 0.0 && one.us < two.us) ? one : two;
}

// Time in us of a launch of the 16-bit kernels, from the constants of prefill_mfma_time (attn_prefill_mfma.hip) and prefill_wide_time
// (attn_prefill_mfma_wide.hip): rounds of workgroups that walk their tiles of 64 keys, above head_dim 128 32.
static double tiles_time(const ContextParams &p, int rows_per_group, int64_t workgroups, int64_t tiles) {
    const double rounds = (double)div_up(workgroups, p.cus), dims = p.D <= 64 ? 1.0 : p.D <= 96 ? 1.43 : 1.86;
    if (p.D > 128) return 5.0 + rounds * (6.5 + 0.70 * (double)tiles);
    return 4.6 + rounds * (rows_per_group == 128 ? 5.3 + 0.356 * dims * (double)tiles : 3.9 + 0.579 * dims * (double)tiles);
}
static ContextTilesJob tiles_job(const ContextParams &p, bool fold, bool with_prefix, bool with_own) {
    ContextTilesJob job;
    memset(&job, 0, sizeof(job));
    job.fold = fold, job.with_prefix = with_prefix, job.with_own = with_own;
    job.units = fold ? p.Hkv : p.B * p.Hkv;
    job.rows = (fold ? p.B : 1) * p.G * p.Sq;
    return job;
}
// The launch of one job, or of two that share the length of their shares; parked: other results of its rows are merged with its own anyway.
static ContextTilesLaunch tiles_launch(const ContextParams &p, fhip_dtype dtype, std::initializer_list<ContextTilesJob> of, bool parked, double *time) {
    const bool f32 = dtype == FHIP_F32;
    const int tile = f32 || p.D > 128 ? 32 : 64;
    // (rows per workgroup, key groups); to head_dim 128 the 16-bit form of 128 rows takes one part
    static const int FORMS[3][3][2] = {{{256, 1}, {128, 2}, {0, 0}}, {{128, 1}, {0, 0}, {0, 0}}, {{128, 1}, {128, 2}, {64, 2}}};
    ContextTilesLaunch best, how;
    memset(&how, 0, sizeof(how));
    best = how;
    how.jobs = (int32_t)of.size();
    double least = 0.0;
    for (const auto &form : FORMS[f32 ? 2 : p.D > 128 ? 1 : 0]) {
        const bool both = of.begin()->with_prefix && of.begin()->with_own;
        if (form[0] == 0 || (!f32 && p.D <= 128 && form[0] == 128 && both) || (f32 && p.D > 128 && form[1] > 1)) continue;
        how.rows_per_group = form[0], how.key_groups = form[1];
        const int64_t positions = std::min<int64_t>(p.Sq, form[0] / p.G + 2);
        int64_t tiles[2] = {0, 0}, keys_of[2] = {0, 0}, groups[2] = {0, 0};
        for (int j = 0; j < how.jobs; j++) {
            ContextTilesJob &job = how.job[j] = of.begin()[j];
            int64_t keys = 0;
            if (job.with_prefix) keys += job.fold ? part_keys(p, true) : most_visible(p, p.P, positions, p.sinks);
            if (job.with_own) keys += most_visible(p, p.Skv, positions, std::max<int64_t>((int64_t)p.sinks - p.P, 0));
            if (both && p.causal && p.window > 0) keys = std::min(keys, p.window + positions + p.sinks);
            keys_of[j] = std::max<int64_t>(keys, 1), tiles[j] = div_up(keys_of[j], tile);
            job.blocks = (int32_t)div_up(job.rows, form[0]);
            groups[j] = (int64_t)job.units * job.blocks;
        }
        const int longest = tiles[1] > tiles[0];
        for (int64_t shares = 1; shares <= tiles[longest]; shares++) {
            const int64_t chunk = div_up(tiles[longest], shares);
            if (div_up(tiles[longest], chunk) != shares) continue;
            int64_t total = 0, slots = 0;
            for (int j = 0; j < how.jobs; j++) {
                ContextTilesJob &job = how.job[j];
                job.chunk = (int32_t)chunk, job.shares = (int32_t)div_up(tiles[j], chunk);
                job.slot0 = (int32_t)slots;
                slots += job.shares;
                if (j == 1) how.second = (int32_t)std::min<int64_t>(total, 0x7fffffff);
                total += groups[j] * job.shares;
            }
            if (shares > 1 && total > 3 * p.cus) break;
            if (total >= 1 << 23) break;  // (2^32 threads)
            if (how.jobs == 1) how.second = (int32_t)total;
            how.total = (int32_t)total;
            double us;
            if (!f32) {
                us = tiles_time(p, form[0], total, chunk);
            } else if (how.jobs == 1) {
                const TermsCall call = {1, how.job[0].units, 1, how.job[0].rows, (int)keys_of[0], p.D, p.cus, false, 0, true, false};
                us = prefill_f32_terms_time(call, {form[0] / 32, form[1]}, (int)shares);
                if (shares > 1) us -= prefill_f32_merge_time(call, (int)shares);
            } else {
                if (total * form[0] > 0x7fffffff) break;
                const TermsCall call = {1, 1, 1, (int)total * form[0], (int)chunk * tile, p.D, p.cus, false, 0, true, false};
                us = prefill_f32_terms_time(call, {form[0] / 32, form[1]}, 1);
            }
            if (slots > 1 || parked) us += partials_us(p, slots);
            if (slots > 1 && !parked) us += 3.0;
            if (least == 0.0 || us < 0.98 * least) least = us, best = how;
        }
    }
    *time = least;
    return best;  // (of no jobs: too many workgroups for a launch)
}

// The sequences' own keys in the kernel for few rows, or on tiles.
static ContextPlan plan_with(const ContextParams &p, fhip_dtype dtype, bool tiles, bool own_by_rows) {
    ContextPlan plan;
    memset(&plan, 0, sizeof(plan));
    plan.any = true;
    const int64_t each = (int64_t)p.G * p.Sq;  // columns of a sequence and KV head
    // rows of all sequences meet the prefix together where they see one run of it
    const bool can_fold = p.P > 0 && p.B > 1 && (p.window == 0 || !p.q_positions);
    const bool one_part = dtype != FHIP_F32 && p.D > 128;  // the tiled kernel takes one part per launch
    int64_t slots = 0;
    auto set_tiles = [&](std::initializer_list<ContextTilesJob> of, bool parked) {
        plan.tiles = tiles_launch(p, dtype, of, parked, &plan.us);
        slots = (int64_t)plan.tiles.job[0].shares + plan.tiles.job[1].shares;
        return plan.tiles.jobs > 0;
    };
    if (own_by_rows) {
        RowsPlan rows = rows_launch(p, dtype, p.P > 0, 0);
        if (rows.us == 0.0) return plan;
        bool on_tiles = false;
        if (p.P > 0 && tiles && can_fold && set_tiles({tiles_job(p, true, true, false)}, p.Skv > 0)) {
            // rows of all sequences on the prefix: with the own keys' launch, or on tiles in one of their own
            const RowsPlan own = rows_launch(p, dtype, false, slots);
            if (p.Skv > 0) plan.us += own.us;
            on_tiles = plan.us < rows.us;
            if (on_tiles) rows = own;
        }
        if (!on_tiles) memset(&plan.tiles, 0, sizeof(plan.tiles)), plan.us = rows.us;
        if (!on_tiles || p.Skv > 0) plan.rows = rows.rows, slots = rows.slots;
    } else if (p.P > 0 && ((can_fold && each < 128) || (one_part && p.Skv > 0))) {
        const ContextTilesJob prefix = tiles_job(p, can_fold, true, false);
        if (!(p.Skv > 0 ? set_tiles({prefix, tiles_job(p, false, false, true)}, false) : set_tiles({prefix}, false))) return plan;
    } else if (!set_tiles({tiles_job(p, false, p.P > 0, p.Skv > 0)}, false)) {
        return plan;
    }
    if (slots > 0x7fffffff) return plan;
    plan.any = false;
    plan.slots = (int)slots;
    if (slots > 1) plan.bytes = (size_t)p.B * p.H * p.Sq * (size_t)slots * (size_t)(p.D + 4) * sizeof(float);
    return plan;
}
static ContextPlan context_plan(const ContextParams &p, fhip_dtype dtype) {
    if (!context_rows_takes(p, dtype)) {
        ContextPlan any;
        memset(&any, 0, sizeof(any));
        any.any = true;
        return any;
    }
    const bool tiles = context_tiles_takes(p, dtype) || context_terms_takes(p, dtype);
    const int64_t each = (int64_t)p.G * p.Sq;
    const ContextPlan few = !tiles || each <= 256 ? plan_with(p, dtype, tiles, true) : ContextPlan();
    if (!tiles || (each <= 16 && !few.tiles.jobs)) return few;
    const ContextPlan many = plan_with(p, dtype, true, false);
    if (each > 256) return many;
    // (252 calls of 20 to 256 columns: 1 per cent slower than the faster of the two in the mean, 30 at most; a limit of 32 columns, f32 64, is 6 per cent
    // slower: 12 f16 rows of one sequence on 600 keys at head_dim 128 take 9.9 us here and 13.6 on tiles, 5 of 32 sequences at 256 on 4000 124 and 70)
    return !few.any && (many.any || 0.9 * few.us < many.us) ? few : many;
}

ContextCall context_call(const ContextParams &p, fhip_dtype dtype) {
    ContextCall call;
    memset(&call, 0, sizeof(call));
    call.parts = 1, call.rows[0] = p.Sq;
    call.plan[0] = context_plan(p, dtype);
    // Where the last workgroup of each unit would hold few of its rows, these go to the kernel for few rows if that is estimated to take less: 8 x 257
    // rows of 32 heads on a prefix of 8192 keys take 301 us instead of 369, 32 x 65 rows at head_dim 256 on 2048 138 instead of 179.
    const int limit = dtype == FHIP_F32 ? 64 : 32;
    const int64_t group = call.plan[0].tiles.rows_per_group, first = group ? (int64_t)p.G * p.Sq / group * group / p.G : 0, rest = p.Sq - first;
    if (first > 0 && rest > 0 && rest * p.G <= limit && call.plan[0].rows.total == 0) {
        ContextParams q = p;
        q.Sq = (int)first;
        const ContextPlan most = context_plan(q, dtype);
        q.Sq = (int)rest, q.q_pos_offset += first;
        const ContextPlan last = context_plan(q, dtype);
        if (!most.any && !last.any && most.us + last.us < call.plan[0].us) {
            call.parts = 2;
            call.rows[0] = call.first_row[1] = (int)first, call.rows[1] = (int)rest;
            call.plan[0] = most, call.plan[1] = last;
        }
    }
    call.bytes = std::max(call.plan[0].bytes, call.plan[1].bytes);
    return call;
}

}  // namespace fhip
