// Attention over a context in two parts in f32 precision on the 16-bit matrix cores (attn_prefill_f32_terms_kernel.h): prompts and chunks of f32 tensors under
// a window with first tokens, behind a prefix, and the rows of a whole batch on the prefix that it shares.
// Bound: as that kernel's few rows on many keys: 129 rows of 16 heads at 80 on 2180 visible keys 27 us and 4.7 of merging their shares (under the
// window alone 25 and 4.6).
#include <type_traits>

#include "attn_prefill_f32_terms_kernel.h"
#include "context.h"

namespace fhip {

bool context_terms_takes(const ContextParams &p, fhip_dtype dtype) {
    if (dtype != FHIP_F32 || p.D > 256 || !(p.scale > 0.0f) || !context_rows_takes(p, dtype)) return false;
    // queries are read in pieces of 16 bytes
    if ((uintptr_t)p.q % 16 != 0 || p.qs[3] != 1) return false;
    for (int i = 0; i < 3; i++)
        if (p.qs[i] % 4 != 0) return false;
    // keys and values through 32-bit buffer offsets: rows that do not overlap, less than 2 GiB of a tensor's head with the tiles behind its end
    auto fits = [&](int64_t row, int64_t rows) { return row >= p.D && (rows + 8 * PT_BN) * row * 4 < 0x7fffffffLL; };
    if (p.Skv > 0 && !(fits(p.ks[2], p.Skv) && fits(p.vs[2], p.Skv))) return false;
    return p.P == 0 || (fits(p.pks[1], p.P) && fits(p.pvs[1], p.P));
}

template <int U, int KG, class P>
static void launch_form(const P &p, const ContextTilesLaunch &how, hipStream_t stream) {
    TermsLaunch tl = {};
    tl.out_vec = p.os[3] == 1 && (uintptr_t)p.out % 16 == 0 ? 16 : 0;
    for (int i = 0; i < 3; i++)
        if (p.os[i] % 4 != 0) tl.out_vec = 0;
    const dim3 grid((unsigned)how.total), block(64 * U * KG);
    auto run = [&](auto dims) {
        hipLaunchKernelGGL((prefill_f32_terms_kernel<float, decltype(dims)::value, U, KG, PF32_INTERVALS, P>), grid, block, 0, stream, p, tl);
    };
    using std::integral_constant;
    if (p.D <= 64) run(integral_constant<int, 64>{});
    else if (p.D <= 96) run(integral_constant<int, 96>{});
    else if (p.D <= 128) run(integral_constant<int, 128>{});
    if constexpr (U == 4 && KG == 1) {
        if (p.D > 192) run(integral_constant<int, 256>{});
        else if (p.D > 128) run(integral_constant<int, 192>{});
    }
}
template <class P>
static void launch_parts(const P &p, const ContextTilesLaunch &how, hipStream_t stream) {
    if (how.rows_per_group == 64) launch_form<2, 2>(p, how, stream);
    else if (how.key_groups == 2) launch_form<4, 2>(p, how, stream);
    else launch_form<4, 1>(p, how, stream);
}

int launch_context_terms(const ContextParams &p0, const ContextTilesLaunch &how, hipStream_t stream) {
    ContextBoth p;
    (ContextParams &)p = p0;
    set_tiles_launch(p, how);
    if (p.job.with_prefix && p.job.with_own) launch_parts(p, how, stream);
    else launch_parts((const ContextParams &)p, how, stream);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

}  // namespace fhip
