// Prefill attention in f32 precision on the 16-bit matrix cores: which form a call takes, and the launch.  The kernel is in
// attn_prefill_f32_terms_kernel.h.
#include <algorithm>

#include "attn_prefill_f32_terms_kernel.h"

namespace fhip {

// ---- which form a call takes ------------------------------------------------------------------------------------------------

static long units_of(const TermsCall &c) { return (long)c.G * ((c.Sq + 31) / 32); }

// workgroups of the form with U units each, in ns shares of the keys
static long terms_workgroups(const TermsCall &c, int U, int ns) {
    return (units_of(c) + U - 1) / U * c.B * c.Hkv * (ns > 1 ? ns : 1);
}

// The form by the numbers of its workgroups (measured on f32 calls, time per call in us; w2, w4: workgroups with 2 or 4 units):
//   (4, 1)  two workgroups per CU, least splitting per tile: grids that fill the chip twice.  Head dims above 128, one workgroup per CU
//           (106 KiB of LDS, 512 registers): a wavefront per SIMD issues its matrix and vector work in turn, 12200 cycles a tile
//           at 256, 6144 of them matrix instructions (5.3 to 5.6 us by the clock; profiles/prefill_f32_terms.txt; 16/4 heads causal, us before, on the f32 matrix instruction: 148 rows on 3510 keys
//           192 -> 80, 1024 x 1024 181 -> 119, 3191 x 3191 826 -> 555, 1500 x 6000 1577 -> 1020)
//   (4, 2)  eight wavefronts, one workgroup per CU: D = 128 1500 rows 115 against 142 for (4, 1), 4000 rows of 8 heads
//           262 against 348, 129 rows on 8003 keys (keys split over workgroups) 111 against 133
//   (2, 2)  D > 64: one wavefront per SIMD with 512 registers, half the units per workgroup, for short prompts (700 rows
//           48 against 55 for (4, 2), 200 rows 21 against 24) and others that fit the CUs once.  With the keys split there is no
//           short workgroup beside a long one unless the prompt is causal (768 rows of 8/2 heads, 288 workgroups: 33 against 36
//           with causality, 51 against 39 without; 16/4 heads, 384 workgroups: 58 against 47).  D <= 64: two workgroups per CU;
//           square causal prompts, whose later rows see more keys, are spread more evenly by half the units (1024 rows 38
//           against 47 for (4, 2), 2048 rows 111 and 2560 rows 159 against 118 and 165 for (4, 1); 3072 rows 224 against 216,
//           4096 rows 388 against 336), and up to two tiles have nothing for more than two groups (55 rows of 16/4 heads 9.4 in
//           (2, 4), 8.0)
//   (2, 4)  D <= 64, eight wavefronts: 512 rows 18 against 21.5 for (2, 2), 1000 rows of 16 heads without a mask 31
//           against 38
static TermsForm form_by_workgroups(const TermsCall &c, int ns) {
    const int cus = c.cus;
    const long w2 = terms_workgroups(c, 2, ns), w4 = terms_workgroups(c, 4, ns);
    const bool few_rows = 2L * c.Sq <= c.Skv;
    if (c.D <= 64) {
        if (c.Skv <= 2 * PT_BN) return {2, 2};
        if (2 * w2 <= (c.uneven ? 3L : 2L) * cus) return {2, 4};
        if (c.uneven && 2 * w4 <= 5L * cus) return {2, 2};
        if (!c.uneven && w4 <= cus) return {4, 2};
    } else {
        const bool fits = w2 <= cus || (ns > 1 ? c.uneven && 4 * w2 <= 5L * cus : !few_rows && 2 * w2 <= 3L * cus);
        if (fits) return {2, 2};
        if (w4 < 2L * cus) return {4, 2};
    }
    return {4, 1};
}

// Time of a call whose rows all see about the same keys, in us: rounds of workgroups that walk their tiles, and parking and
// merging the shares.  Constants fitted to 210 random calls (chunks, turns, images and encoders of 8 to 32 heads at 64 to 128
// dims, each in every form and up to 48 shares): 6 % off in the mean square.
double prefill_f32_merge_time(const TermsCall &c, int ns) {
    return 3.24 + 0.456e-6 * prefill_f32_workspace_bytes(c.B, c.Hkv * c.G, c.Sq, c.D, ns);
}
static double wide_terms_time(const TermsCall &c, int ns);
namespace {
// Of a workgroup: a tile of one of its key groups, its ends, and what a tile takes where a CU has one of two workgroups.
struct FormTimes {
    double tile, ends, alone;
    bool two_per_cu;
};
FormTimes times_of_form(int D, TermsForm f) {
    const double dims = (D <= 64 ? 64 : D <= 96 ? 96 : 128) / 64.0;
    if (f.U == 2 && f.KG == 2 && D <= 64) return {2.65, 1.4, 0.71, true};
    if (f.U == 2 && f.KG == 2) return {0.38 + 1.494 * dims, 3.9, 1.0, false};
    if (f.KG == 2) return {0.306 + 1.945 * dims, 3.45, 1.0, false};
    if (f.KG == 4) return {2.65, 3.87, 1.0, false};
    return {0.374 + 1.78 * dims, 0.8, 0.74, true};
}
}  // namespace
double prefill_f32_terms_time(const TermsCall &c, TermsForm f, int ns) {
    if (c.D > 128) return wide_terms_time(c, ns);
    const FormTimes t = times_of_form(c.D, f);
    const int chunk = ((c.Skv + ns - 1) / ns + PT_BN - 1) / PT_BN * PT_BN, n = (c.Skv + chunk - 1) / chunk;
    int tiles = chunk / PT_BN;
    // (a workgroup's rows see the window's keys and as many more as there are rows: counted for 32 rows in every form, ungrouped heads took
    // four units too often, 16 heads at 96, three sequences of 156 rows under 32 21.7 us for 13.9, over 110 chunks 1.09 of the time; wider windows
    // than 0.7 of the keys are taken for none: 32/8 heads at 128, 1100 rows under 2885 of 3984 keys would stay unsplit and take 1.21 times as long)
    const int rows = 32 * ((f.U + c.G - 1) / c.G);
    if (c.window > 0 && c.window < c.Skv && 10 * (c.window + PT_BN) < 7LL * c.Skv) tiles = std::min(tiles, ((int)c.window + rows + PT_BN - 1) / PT_BN + 1);
    const double walk = t.tile * ((tiles + f.KG - 1) / f.KG);
    const long wgs = terms_workgroups(c, f.U, n), slots = (t.two_per_cu ? 2L : 1L) * c.cus, rest = wgs % slots;
    double us = 4.9 + wgs / slots * (t.ends + walk);
    if (rest) us += t.ends + walk * (rest <= c.cus ? t.alone : 1.0);
    if (n > 1) us += prefill_f32_merge_time(c, n);
    return us;
}

// Unsplit chunks under a causal mask that need more than one round: the rows of the later rounds see the fewest keys, and start first where rows
// of few keys end.  1.15 times what the second (third) round's first workgroup takes twice (three times), or the mean load: 5 % off over nine
// chunks of 272 to 376 workgroups, which as even calls were taken for 1.1 to 1.5 times their time and split for nothing (us, four sequences
// of 1071 rows of 8/4 heads at 128 on 2216 keys 203 unsplit and 261 in two shares, three of 1832 of 8/2 at 96 on 3665 289 and 336).
double prefill_f32_unsplit_time(const TermsCall &c, TermsForm f) {
    const double even = prefill_f32_terms_time(c, f, 1);
    if (c.D > 128 || !c.causal || c.window > 0) return even;
    const FormTimes t = times_of_form(c.D, f);
    const double walk = t.tile * (((c.Skv + PT_BN - 1) / PT_BN + f.KG - 1) / f.KG), part = (double)c.Sq / c.Skv;
    const double wgs = (double)terms_workgroups(c, f.U, 1), slots = (t.two_per_cu ? 2.0 : 1.0) * c.cus;
    if (wgs <= slots) return even;
    double us = std::max(t.ends + walk, 1.08 * wgs / slots * (t.ends + walk * (1.0 - 0.5 * part)));
    us = std::max(us, 2.0 * (t.ends + walk * (1.0 - part * slots / wgs)));
    if (wgs > 2 * slots) us = std::max(us, 3.0 * (t.ends + walk * (1.0 - part * 2.0 * slots / wgs)));
    return std::min(even, 4.9 + 1.15 * us);
}

// The same above head_dim 128, where the form is (4, 1) with one workgroup per CU, of uneven calls too: even shares in rounds; of uneven
// ones, dealt out the longest first, the longest, the mean load, or twice (three times) the first workgroup of the second (third) round.
// Over 420 random calls at 160 to 256 dims in up to 48 shares it is 6 % off in the mean square, 9 % under a window.
// Under a window a row block sees the window's keys and meets few of the shares; the
// workgroups of the others still split Q, park a state and have it merged (us, planned without the window and with it: 16/8 heads at 256,
// 786 rows under a window of 127 59 -> 47; 12/12 at 160, 1317 under 103 58 -> 46; 6/3 at 192, three sequences of 718 under 117 50 -> 38).
static double wide_terms_time(const TermsCall &c, int ns) {
    const double tile = 1.33 * (c.D <= 192 ? 3 : 4), ends = 6.9;
    const int chunk = ((c.Skv + ns - 1) / ns + PT_BN - 1) / PT_BN * PT_BN, n = (c.Skv + chunk - 1) / chunk;
    const long wgs = terms_workgroups(c, 4, 1);
    const int rows = std::min(c.Sq, 32 * ((4 + c.G - 1) / c.G));  // of a workgroup
    const bool narrow = c.window > 0 && c.window < c.Skv - rows;
    const double sight = narrow ? (double)c.window + rows : c.Skv;  // keys from the first to the last that a workgroup's rows see
    double most = chunk / PT_BN;
    if (narrow && sight <= chunk) most = (int)(sight - 1 + PT_BN - 1) / PT_BN + 1;
    const double longest = ends + tile * most;
    double us;
    if (!c.uneven) {
        us = (double)((wgs * n + c.cus - 1) / c.cus) * longest;
    } else {
        const double first = c.Skv > c.Sq ? c.Skv - c.Sq : 0.0;  // keys before the first row
        // workgroups that see this many keys of their share
        auto with_keys = [&](double keys) {
            double sum = 0.0;
            for (int i = 0; i < n; i++) {
                const double from = std::max(first, (double)i * chunk + keys);
                const double to = narrow ? std::min<double>(c.Skv, std::min<double>(c.Skv, (i + 1.0) * chunk) + sight - keys) : c.Skv;
                const double part = (to - from) / (c.Skv - first);
                sum += part < 0.0 ? 0.0 : part > 1.0 ? 1.0 : part;
            }
            return sum * wgs;
        };
        auto time_of = [&](double nth) {  // of the nth workgroup
            if (with_keys(0.0) < nth) return narrow && wgs * n >= nth ? ends : 0.0;
            double keys = 0.0;
            for (double step = 0.5 * chunk; step >= 16.0; step *= 0.5)
                if (keys + step <= sight && with_keys(keys + step) >= nth) keys += step;
            return ends + tile / PT_BN * keys;
        };
        double seen = (first + c.Skv) * 0.5;  // by a row in the mean
        if (narrow) seen = first >= sight ? sight : (0.5 * (sight * sight - first * first) + sight * (c.Skv - sight)) / (c.Skv - first);
        const double load = wgs * (n * ends + seen / PT_BN * tile) / c.cus;
        us = std::max({longest, 1.08 * load, 2.0 * time_of(c.cus + 1.0), 3.0 * time_of(2.0 * c.cus + 1.0)});
    }
    us += 4.9;
    if (n > 1) us += prefill_f32_merge_time(c, n);
    return us;
}

TermsForm prefill_f32_terms_quickest(const TermsCall &c, int ns) {
    if (c.D > 128 || !c.f32) return {4, 1};
    TermsForm best = {4, 1};
    double least = prefill_f32_terms_time(c, best, ns);
    for (const TermsForm f : {TermsForm{4, 2}, TermsForm{2, 2}, TermsForm{2, 4}}) {
        if (f.KG == 4 && c.D > 64) continue;
        const double us = prefill_f32_terms_time(c, f, ns);
        if (us < least) least = us, best = f;
    }
    return best;
}

// Where all rows see about the same keys the rule above leaves much to gain, and the form is the quickest by the time above if that
// is 10 % better (us a call: 16 heads without a mask, 1356 rows at 128 169 -> 99; 6 encoder sequences of 436 tokens 41.5 -> 30.6, 11
// of 169 23.2 -> 18.4; at 7 % ten sequences of 154, 240 workgroups of five tiles, 16.4 -> 17.1).  Up to 128 rows the rule is as good.
TermsForm prefill_f32_terms_form(const TermsCall &c, int ns) {
    if (c.D > 128 || !c.f32) return {4, 1};
    const TermsForm ordinary = form_by_workgroups(c, ns);
    if (c.uneven || c.Sq <= 128 || c.Skv <= 2 * PT_BN) return ordinary;
    const TermsForm other = prefill_f32_terms_quickest(c, ns);
    return prefill_f32_terms_time(c, other, ns) < 0.9 * prefill_f32_terms_time(c, ordinary, ns) ? other : ordinary;
}

// (of f32 tensors)
TermsCall prefill_f32_terms_call(const AttnParams &p) {
    const bool uneven = prefill_f32_uneven(p.Sq, p.Skv, p.D, p.analytic && p.causal, p.mask_kind == FHIP_MASK_QK, p.q_pos_offset, p.window);
    return {p.B, p.Hkv, p.G, p.Sq, p.Skv, p.D, p.cus > 0 ? p.cus : 256, uneven, p.analytic ? p.window : 0, true,
            (p.analytic && p.causal) || p.mask_kind == FHIP_MASK_QK};
}

template <typename T, int U, int KG, int MODE>
static int launch_form(const AttnParams &p_in, hipStream_t stream) {
    AttnParams p = p_in;
    const int cus = p.cus > 0 ? p.cus : 256;
    const long blocks = terms_workgroups(prefill_f32_terms_call(p), U, p.pf_nsplit);
    if (blocks > 0x7fffffffL) {
        set_error("prefill f32: too many workgroups (%ld)", blocks);
        return FHIP_ERR_UNSUPPORTED;
    }
    TermsLaunch tl;
    const unsigned nks = p.pf_nsplit > 1 ? p.pf_nsplit : 1, groups = (unsigned)(p.B * p.Hkv), nwg = (unsigned)(blocks / nks / groups);
    tl.level_pitch = 0;
    // (grids of one round too: without it calls of 500 rows take 2 to 5 % longer, those of 300 1 to 2 % less; under a window the same
    // workgroups of a share still see alike: the grid's order takes 1.07 to 1.16 times as long in two to eight shares of 120 random prompts)
    if (p.D > 128 && nks > 1 && prefill_f32_terms_call(p).uneven) tl.level_pitch = std::max(1, (int)((int64_t)p.pf_chunk * p.G / (32 * U)));
    tl.g_magic = p.G > 1 ? (uint32_t)((0x100000000ull + p.G - 1) / p.G) : 0;
    const bool two_per_cu = (KG == 1 && p.D <= 128) || (U * KG == 4 && p.D <= 64);
    tl.snake = (two_per_cu && blocks > cus && blocks <= 2L * cus) ? (int)((cus + nks * groups - 1) / (nks * groups)) : 0;
    // rows of the result written in 16-byte (f32) or 8-byte pieces
    const int oeb = sizeof(T) == 4 || p.out_f32 ? 4 : 2;
    tl.out_vec = p.os[3] == 1 && (uintptr_t)p.out % (4 * oeb) == 0 ? 4 * oeb : 0;
    for (int i = 0; i < 3; i++)
        if (p.os[i] % 4 != 0) tl.out_vec = 0;
    // rows of the mask in 16-byte (f32, element-aligned) or 8-byte pieces, within a buffer's 32-bit offsets
    const int64_t mask_span = ((p.mask_kind == FHIP_MASK_QK ? (int64_t)(p.Sq - 1) * p.ms0 : 0) + p.Skv) * (int64_t)sizeof(T);
    tl.mask_rows = p.mask_kind != FHIP_MASK_NONE && p.ms1 == 1 && p.ms0 >= 0 && mask_span < 0x7fffffffLL &&
                   (sizeof(T) == 4 || ((uintptr_t)p.mask % 8 == 0 && p.ms0 % 4 == 0));
    dim3 grid(nks, groups, nwg), block(64 * U * KG);
    switch ((p.D + 31) / 32 * 32) {  // the kernel's D is head_dim rounded up to a multiple of 32
        case 32: FHIP_LAUNCH_MAIN((prefill_f32_terms_kernel<T, 32, U, KG, MODE, AttnParams>), grid, block, stream, p, p, tl); break;
        case 64: FHIP_LAUNCH_MAIN((prefill_f32_terms_kernel<T, 64, U, KG, MODE, AttnParams>), grid, block, stream, p, p, tl); break;
        case 96:
            if constexpr (MODE != PF32_EITHER && KG < 4) FHIP_LAUNCH_MAIN((prefill_f32_terms_kernel<T, 96, U, KG, MODE, AttnParams>), grid, block, stream, p, p, tl);
            break;
        case 128:
            if constexpr (MODE != PF32_EITHER && KG < 4) FHIP_LAUNCH_MAIN((prefill_f32_terms_kernel<T, 128, U, KG, MODE, AttnParams>), grid, block, stream, p, p, tl);
            break;
        case 160:
        case 192:
            if constexpr (sizeof(T) == 4 && U == 4 && KG == 1 && MODE == PF32_INTERVALS) FHIP_LAUNCH_MAIN((prefill_f32_terms_kernel<T, 192, U, KG, MODE, AttnParams>), grid, block, stream, p, p, tl);
            break;
        case 224:
        case 256:
            if constexpr (sizeof(T) == 4 && U == 4 && KG == 1 && MODE == PF32_INTERVALS) FHIP_LAUNCH_MAIN((prefill_f32_terms_kernel<T, 256, U, KG, MODE, AttnParams>), grid, block, stream, p, p, tl);
            break;
        default: set_error("prefill f32 kernel: head_dim %d is not a multiple of 4 up to 256", p.D); return FHIP_ERR_UNSUPPORTED;
    }
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

template <typename T, int MODE>
static int launch_terms(const AttnParams &p, hipStream_t stream) {
    // 16-bit storage takes (4, 1) always
    if constexpr (sizeof(T) == 4) {
        const TermsForm f = prefill_f32_terms_form(prefill_f32_terms_call(p), p.pf_nsplit > 1 ? p.pf_nsplit : 1);
        if (f.U == 2 && f.KG == 4) return launch_form<T, 2, 4, MODE>(p, stream);
        if (f.U == 2) return launch_form<T, 2, 2, MODE>(p, stream);
        if (f.KG == 2) return launch_form<T, 4, 2, MODE>(p, stream);
    }
    return launch_form<T, 4, 1, MODE>(p, stream);
}

// (16-bit storage above head_dim 128 is not asked for: attn_prefill_mfma_wide.hip has it.)
// K and V rows are fetched through 32-bit buffer offsets: rows must not overlap, and one (batch, kv head) slice must span
// less than 2 GiB, the tiles behind its end included.
bool prefill_f32_terms_takes(const AttnParams &p) {
    const int64_t rows = (int64_t)p.Skv + 8 * PT_BN, units = (int64_t)p.G * ((p.Sq + 31) / 32);
    // (grid dimensions, and the exactness of unit / G by multiplication)
    if ((int64_t)p.B * p.Hkv > 65535 || units > 65535 || units * p.G > 0x7fffffffLL) return false;
    if (p.qs[2] < 0 || (int64_t)p.Sq * p.qs[2] * 4 >= 0x7fffffffLL) return false;
    return p.D <= 256 && p.ks[2] >= p.D && p.vs[2] >= p.D && rows * p.ks[2] * 4 < 0x7fffffffLL && rows * p.vs[2] * 4 < 0x7fffffffLL;
}

// A BatchKeyMask whose row every wavefront can look at for itself, four keys per load and all loads at once: no scan launch.
// Longer rows, rows of a QKMask (each read by all heads) and 16-bit rows, whose last piece a buffer's bounds would cut, are
// scanned once per call.
bool prefill_f32_terms_scans(const AttnParams &p, fhip_dtype dtype) {
    return dtype == FHIP_F32 && p.mask_kind == FHIP_MASK_BATCH_KEY && p.D <= 64 && p.Skv <= SCAN_KEYS && p.ms1 == 1 &&
           prefill_f32_terms_takes(p);
}

int launch_prefill_f32_terms(const AttnParams &p, fhip_dtype dtype, int mode, hipStream_t stream) {
    auto by_type = [&](auto type) {
        typedef decltype(type) T;
        if (mode == PF32_EITHER) return launch_terms<T, PF32_EITHER>(p, stream);
        if (mode == PF32_BIAS) return launch_terms<T, PF32_BIAS>(p, stream);
        return launch_terms<T, PF32_INTERVALS>(p, stream);
    };
    if (dtype == FHIP_F16) return by_type(half_t{});
    if (dtype == FHIP_BF16) return by_type(bf16_t{});
    return by_type(float{});
}

}  // namespace fhip
