// Prefill attention for f16 / bf16 on the gfx950 matrix cores: which form a call takes, in how many shares of its keys, and the launch.  The
// kernel is in attn_prefill_mfma_kernel.h.
#include <algorithm>
#include <type_traits>

#include "attn_prefill_mfma_kernel.h"

namespace fhip {

// Query blocks of 256 rows leave CUs idle when there are few of them (short prompts, a few new rows on a long
// cache), and a causal prompt's last blocks are several times longer than its first.  The key-split form (128
// rows, twice the workgroups, the longest one half as long) costs about 11 % per tile (f16, 32/8 heads at 128, 8192-token
// prompt: 535 us against 481) and a longer prologue and epilogue; measured, it wins while the 256-row grid fills at most half the CUs (8 to 32
// heads, 1024 to 2049 rows: 1.25 - 1.5 x), for up to 128 query rows (where the second wavefront group would have no
// rows at all; 1.07 x at 128, 1.15 at 64), and, where later rows see more keys than earlier ones, for one workgroup per CU
// when a head has 8 or more query blocks; it loses with fewer than three key tiles.
// For one workgroup per CU the 256-row form takes as long as its longest block, the key-split form about a quarter more than the
// mean one (two of its workgroups follow each other on a CU).  f16, us a call, 256-row and key-split form on one card: without a
// mask, 16 heads, head_dim 80, 4096 x 4096 keys 90 and 99, 3000 57 and 66; 64, 2500 40 and 49; 128, 2500 58 and 76, 4096 122 and 136;
// causal, 128, 32/8 heads, 2048 rows on 2048 keys 50 and 47, 4096 106.1 and 105.5, 5120 133.8 and 136.2, 8192 218 and 227; 24/8
// heads 46 and 39, on 4096 keys 91 and 88, 5120 113.2 and 112.9, 6144 136 and 138; 16/8 heads, 3000 rows on 3000 keys 61 and 48, 6000 125
// and 121, 7500 158.2 and 157.4, 9000 190 and 193.  So rows that all see the same keys keep the 256-row form, and where they see
// the keys up to their own position the line is 2.5 keys per row.  Under a window narrower than that it stays at 2, beyond which
// the 256-row form wins by more (2048 rows on 4096 keys under a window of 2048: 68 and 78).  Rows with half a window or more behind the
// first of them see about the same keys as well, however few the call as a whole sees (12/12 heads at 128, 3132 rows under 2512 68 and 85,
// at 80, two sequences of 1939 under 208 22 and 26), but where the key-split form has one workgroup per CU, or little more and the first rows see less
// than a window (12/12 at 128, 2668 behind 226 under 452 29 and 20; 8/4 at 64, 4130 behind 1313 under 2626 50 and 41).  Sequences of different lengths in
// a batch are even grids in this sense (2 to 8 of them, 500 to 2048 keys long: 0.80 to 0.85 of the key-split form's time).
// later_rows_see: the keys up to the last row's own where rows see the keys up to their own position, 0 where all see the same.
int prefill_mfma_block_rows(int B, int H, int Sq, int Skv, int key_shares, int64_t later_rows_see, int64_t window, int compute_units) {
    const int nqb = (Sq + PF_BM - 1) / PF_BM;
    const long wgs = (long)nqb * B * H * (key_shares > 1 ? key_shares : 1);
    if (Skv <= 2 * PF_BN) return PF_BM;
    if (Sq <= PF_BM / 2 || 2 * wgs <= compute_units) return PF_BM / 2;
    if (wgs > compute_units || nqb < 8 || later_rows_see <= 0) return PF_BM;
    const int64_t keys = later_rows_see < Skv ? later_rows_see : Skv;
    const bool narrow = window > 0 && window < keys;
    const long of_half = (long)((Sq + PF_BM / 2 - 1) / (PF_BM / 2)) * B * H;
    const int64_t before = later_rows_see - Sq + 1;  // keys that the first row sees without the window
    // (before < window + 128: the keys begin where the first row's window does; they do not where the call brings lengths)
    if (narrow && window <= Sq && before < window + 128 &&
        (before >= window ? of_half > compute_units : 2 * before >= window && 4 * of_half > 5L * compute_units))
        return PF_BM;
    return 2L * Sq > Skv || (!narrow && 5L * Sq >= 2 * keys) ? PF_BM / 2 : PF_BM;
}

// Head dims 64, 96 and 128 are this kernel's own.  The other multiples of 8 above 64 run on it padded, quicker than on the
// wide-head kernel, whose wavefronts read every LDS operand for half as many matrix instructions (both in turn on one card, us a
// call; f16, 16 heads, 4096 x 4096 keys without a mask: head_dim 72 147 -> 120, 80 150 -> 124, 88 163 -> 130, 104 196 -> 136, 112
// 202 -> 144, 120 201 -> 147; causal, 80: 157 -> 75 (two of that kernel's 128-row blocks per CU wait for the longest); 512-token
// causal prompt, 32/8 heads, 80: 17.0 -> 15.9).  Below 64 the padding costs what the kernel gains unless the grid fills the
// chip (head_dim 40: 4096 keys 134 -> 104; head_dim 32: 116 -> 102), and to 32, where it is half of the work or more, also in
// short row blocks (300 rows of four sequences 60 -> 64).
bool prefill_mfma_rows256_takes(int D, float scale, int B, int H, int Sq, int compute_units) {
    if (!(D % 8 == 0 && D >= 8 && D <= 128 && scale > 0.0f && scale * PF_LOG2E < 2.0f)) return false;
    if (D >= 64) return true;
    const long blocks = (long)B * H * ((Sq + PF_BM - 1) / PF_BM);
    return blocks >= compute_units && (D > 32 || Sq >= 1024);
}

template <typename T>
static int launch_t(const AttnParams &p0, hipStream_t stream) {
    AttnParams p = p0;
    const int cus = p.cus > 0 ? p.cus : 256;
    const int64_t later_rows_see = p.analytic && p.causal ? p.q_pos_offset + p.Sq : p.mask_kind == FHIP_MASK_QK ? p.Skv : 0;
    const int bm = prefill_mfma_block_rows(p.B, p.H, p.Sq, p.Skv, p.pf_nsplit, later_rows_see, p.analytic ? p.window : 0, cus);
    const bool ks = bm == PF_BM / 2;
    p.pf_pack = ks ? prefill_mfma_pack(p.B, p.H, p.G, p.Sq, p.Skv, cus) : 0;
    const int nqb = p.pf_pack ? 1 : (p.Sq + bm - 1) / bm;
    const long blocks = (long)nqb * p.B * (p.pf_pack ? p.H / 4 : p.H) * (p.pf_nsplit > 1 ? p.pf_nsplit : 1);
    if (blocks > 0x7fffffffL) {
        set_error("prefill: too many workgroups (%ld)", blocks);
        return FHIP_ERR_UNSUPPORTED;
    }
    dim3 grid((unsigned)blocks), block(64 * PF_WAVES);
    // rows of the output can be written in 16-byte pieces when they are contiguous and aligned
    const int oeb = p.out_f32 ? 4 : 2;
    int out_vec = (p.os[3] == 1 || p.D == 1) && ((uintptr_t)p.out % 16 == 0);
    for (int i = 0; i < 3; i++)
        if ((p.os[i] * oeb) % 16 != 0) out_vec = 0;
#define PF_LAUNCH(DIM, QDIM, PAD)                                                                               \
    if (ks) FHIP_LAUNCH_MAIN((prefill_mfma_kernel<T, DIM, QDIM, PAD, true, AttnParams>), grid, block, stream, p, p, nqb, out_vec); \
    else FHIP_LAUNCH_MAIN((prefill_mfma_kernel<T, DIM, QDIM, PAD, false, AttnParams>), grid, block, stream, p, p, nqb, out_vec)
    if (p.D % 8 != 0 || p.D < 8 || p.D > 128) {
        set_error("prefill MFMA kernel: head_dim %d is not a multiple of 8 up to 128", p.D);
        return FHIP_ERR_UNSUPPORTED;
    }
    if (p.D == 64) { PF_LAUNCH(64, 64, false); }
    else if (p.D == 96) { PF_LAUNCH(96, 96, false); }
    else if (p.D == 128) { PF_LAUNCH(128, 128, false); }
    else if (p.D < 64) { PF_LAUNCH(64, 64, true); }
    else if (p.D <= 80) { PF_LAUNCH(96, 80, true); }
    else if (p.D < 96) { PF_LAUNCH(96, 96, true); }
    else if (p.D <= 112) { PF_LAUNCH(128, 112, true); }
    else { PF_LAUNCH(128, 128, true); }
#undef PF_LAUNCH
    FHIP_HIP_CHECK(hipGetLastError());
    if (p.pf_nsplit > 1) return launch_prefill_merge(p, sizeof(T) == 2 && std::is_same<T, half_t>::value ? FHIP_F16 : FHIP_BF16, stream);
    return FHIP_OK;
}

// Few query rows on a long cache: 256-row query blocks alone leave most CUs idle, so the keys are split over
// workgroups too, down to 1024 keys per share, until there are about two workgroups per CU.
// Query heads per workgroup of the packed form (0: not packed).  Packing divides the workgroups by four, and a share of
// the keys is at least 1024 keys long, so it is taken when the packed grid still reaches half the CUs (12..32 rows:
// batch 8 on 8192 keys 98 -> 66..81 us, batch 4 on 4096 keys 45 -> 28 us, batch 1 on 32768 keys 68 -> 40 us; with a
// quarter of the CUs, batch 1 on 8192 keys, the unpacked grid is as quick: 25.7 against 26.5 us).
int prefill_mfma_pack(int B, int H, int G, int Sq, int Skv, int compute_units) {
    if (!(Sq <= 32 && G >= 4 && G % 4 == 0) || Skv <= 2 * PF_BN) return 0;
    const long shares = Skv / 1024 > 1 ? Skv / 1024 : 1;
    return 2 * (long)B * (H / 4) * shares >= compute_units ? 4 : 0;
}

// Time of a call in us, by the form it takes in that many shares: rounds of workgroups that walk their tiles, and parking and
// merging the shares.  Constants fitted to 140 random calls (chunks, turns and images of 8 to 32 heads at 64 to 128 dims, each in both
// forms and up to 48 shares): 10 % off in the mean square.
static double prefill_mfma_time(int B, int H, int G, int Sq, int Skv, int D, int64_t later_rows_see, int64_t window, int compute_units, int ns) {
    const int c = ((Skv + ns - 1) / ns + PF_BN - 1) / PF_BN * PF_BN, n = (Skv + c - 1) / c;
    const int bm = prefill_mfma_block_rows(B, H, Sq, Skv, n, later_rows_see, window, compute_units);
    const bool ks = bm == PF_BM / 2, packed = ks && prefill_mfma_pack(B, H, G, Sq, Skv, compute_units);
    const long wgs = (long)B * (packed ? H / 4 : H) * ((Sq + bm - 1) / bm) * n, rounds = (wgs + compute_units - 1) / compute_units;
    const double dims = D <= 64 ? 1.0 : D <= 96 ? 1.43 : 1.86;
    double us = 4.6 + rounds * (ks ? 5.3 + 0.356 * dims * (c / PF_BN) : 3.9 + 0.579 * dims * (c / PF_BN));
    if (n > 1) us += 3.0 + 0.488e-6 * prefill_mfma_workspace_bytes(B, H, Sq, D, n);
    return us;
}

// uneven: a square call whose rows see the keys up to their own position (a mask tensor is taken for one): by the rules alone.
// later_rows_see, window: as for prefill_mfma_block_rows.
void prefill_mfma_plan(int B, int H, int G, int Sq, int Skv, int D, bool causal_square, bool uneven, int64_t later_rows_see, int64_t window,
                       bool unknown_lengths, int compute_units, int *nsplit, int *chunk) {
    *nsplit = 1;
    *chunk = Skv;
    if (causal_square) return;
    const long wgs = (long)B * (prefill_mfma_pack(B, H, G, Sq, Skv, compute_units) ? H / 4 : H) * ((Sq + PF_BM - 1) / PF_BM);
    if (wgs == 0) return;
    // By rule a grid of query blocks that keeps half the chip busy by itself is not split (the times below may find otherwise).
    const long want = (2L * compute_units + wgs - 1) / wgs;
    long most = Skv / 1024;
    // A few rows on a short cache: shares down to 512 keys, and for up to 64 rows to 256, while CUs would stay without a
    // workgroup (f16, 32/8 heads, head_dim 128, B1: 12...32 rows on 2048 keys 24.6 -> 17.8 us, on 4096 keys 24.7 -> 20.7;
    // 128 rows on 2048 keys 28.8 -> 25.7).  On 1024 keys two shares of 512 lose with more than 64 rows (21.2 -> 23.4 us).
    const bool few_rows = 2L * Sq <= Skv && (Sq <= 64 || Skv >= 2048);
    if (few_rows && (want < most ? want : most) * wgs < compute_units) most = Skv / 512;
    if (few_rows && Sq <= 64 && (want < most ? want : most) * wgs < compute_units) most = Skv / 256;
    long ns = 2 * wgs > compute_units ? 1 : want < most ? want : most;
    if (ns < 1) ns = 1;
    // These rules count workgroups and not their rounds, nor the bytes of the partials: the shares of least time by the function
    // above, the fewest within 1 % of it, are taken where that is 5 % less than the rules' (shares_gain), or 10 % for grids that the rules do not split
    // (us a call: four sequences of 207 rows of 32/8 heads at 96 under a window of 4096 84 -> 56 in none; 189 rows of 8/4 heads at 80 on 1993 keys 23.5 -> 19, 231 of 32/8 at 64 on 14900
    // 59 -> 48, 49 of 32/32 at 128 on 3032 36 -> 22; over 500 random calls without lengths or a mask tensor 0.93 of the rules' time, the
    // worst 1.11; at 5 % everywhere large ones lost up to 14 %: 32/32 heads at 80, 2859 rows on 7370 keys 209 and 238).
    constexpr int SHARES[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48};
    double times[sizeof(SHARES) / sizeof(SHARES[0])], least = 0.0;
    int tried = 0;
    for (const int n : SHARES) {
        if (uneven) break;
        // (three rounds gain nothing more; partials of at most 64 MiB)
        if (n > 1 && (Skv / n < 128 || (n - 1) * wgs > 3L * compute_units || prefill_mfma_workspace_bytes(B, H, Sq, D, n) > ((size_t)64 << 20)))
            break;
        times[tried] = prefill_mfma_time(B, H, G, Sq, Skv, D, later_rows_see, window, compute_units, n);
        if (tried == 0 || times[tried] < least) least = times[tried];
        tried++;
    }
    for (int i = 0; i < tried; i++) {
        if (times[i] > 1.01 * least) continue;
        const double gain = std::min(shares_gain(unknown_lengths), 2 * wgs > compute_units ? 0.9 : 1.0);
        if (times[i] < gain * prefill_mfma_time(B, H, G, Sq, Skv, D, later_rows_see, window, compute_units, (int)ns)) ns = SHARES[i];
        break;
    }
    if (ns < 2) return;
    long c = (Skv + ns - 1) / ns;
    c = (c + PF_BN - 1) / PF_BN * PF_BN;
    *chunk = (int)c;
    *nsplit = (int)((Skv + c - 1) / c);
}

size_t prefill_mfma_workspace_bytes(int B, int H, int Sq, int D, int nsplit) {
    if (nsplit <= 1) return 0;
    return (size_t)B * H * Sq * nsplit * (size_t)(D + 4) * sizeof(float);
}

int launch_prefill_mfma(const AttnParams &p, fhip_dtype dtype, hipStream_t stream) {
    if (dtype == FHIP_F16) return launch_t<half_t>(p, stream);
    if (dtype == FHIP_BF16) return launch_t<bf16_t>(p, stream);
    set_error("prefill MFMA kernel takes f16/bf16 only");
    return FHIP_ERR_UNSUPPORTED;
}

}  // namespace fhip
