// Attention over a context in two parts on the tiled kernels of the 16-bit matrix cores: prompts and chunks under a window with first tokens, behind a
// prefix, and the rows of a whole batch on the prefix that it shares.  Here the 256-row kernel (attn_prefill_mfma_kernel.h), head dims to 128.
// Bound: as that kernel without the lists of tiles, power: 8192 f16 rows of 32/8 heads at 128 under a window of 4096 with 64 first tokens 388 us
// (1.07 PFLOP/s; the window alone 383), four bf16 chunks of 512 rows 127 (123), eight times 256 rows on 8192 shared keys 280 (1.0 PFLOP/s).
#include <type_traits>

#include "attn_prefill_mfma_kernel.h"
#include "context.h"

namespace fhip {

bool context_tiles_takes(const ContextParams &p, fhip_dtype dtype) {
    if (dtype == FHIP_F32 || !context_rows_takes(p, dtype)) return false;
    // In bf16 at the kernels' own widths Q takes the power of two of the factor of the scores: up to 1, so that no element leaves the type's range above, and not so small
    // that elements in use leave the normal range below.  Elsewhere the factor multiplies f32 sums of products, which of f16 elements are less than 2^40.  (8192 f16
    // rows of 32/8 heads at 128 under a window of 4096 at a scale of 1.5: 346 us here, 1260 in the kernel for few rows.)
    const float factor = p.scale * PF_LOG2E;
    const bool in_q = dtype == FHIP_BF16 && (p.D > 128 || p.D == 64 || p.D == 96 || p.D == 128);
    if (!(p.scale > 0.0f && factor < (in_q ? 2.0f : 0x1p64f))) return false;
    if (in_q && factor < (p.D > 128 ? 0x1p-8f : 0x1p-64f)) return false;
    // queries are read in pieces of 16 bytes
    if ((uintptr_t)p.q % 16 != 0 || p.qs[3] != 1) return false;
    for (int i = 0; i < 3; i++)
        if (p.qs[i] % 8 != 0) return false;
    // keys and values through 32-bit buffer offsets: rows that do not overlap, less than 2 GiB of a tensor's head
    auto fits = [&](int64_t row, int64_t rows) { return row >= p.D && rows * row * 2 < 0x7fffffff - 65536; };
    if (p.Skv > 0 && !(fits(p.ks[2], p.Skv) && fits(p.vs[2], p.Skv))) return false;
    return p.P == 0 || (fits(p.pks[1], p.P) && fits(p.pvs[1], p.P));
}

template <typename T>
static void launch_type(const ContextParams &p, const ContextTilesLaunch &how, hipStream_t stream) {
    const bool half = how.rows_per_group == PF_BM / 2;
    const dim3 grid((unsigned)how.total), block(64 * PF_WAVES);
    const int bytes = p.out_f32 ? 4 : 2;
    int out_vec = p.os[3] == 1 && (uintptr_t)p.out % 16 == 0;
    for (int i = 0; i < 3; i++)
        if (p.os[i] * bytes % 16 != 0) out_vec = 0;
    auto run = [&](auto dim, auto contracted, auto padded) {
        constexpr int DIM = decltype(dim)::value, QDIM = decltype(contracted)::value;
        constexpr bool PAD = decltype(padded)::value;
        if (p.job.with_prefix && p.job.with_own) {
            ContextBoth both;
            (ContextParams &)both = p;
            hipLaunchKernelGGL((prefill_mfma_kernel<T, DIM, QDIM, PAD, false, ContextBoth>), grid, block, 0, stream, both, 0, out_vec);
        } else if (half) hipLaunchKernelGGL((prefill_mfma_kernel<T, DIM, QDIM, PAD, true, ContextParams>), grid, block, 0, stream, p, 0, out_vec);
        else hipLaunchKernelGGL((prefill_mfma_kernel<T, DIM, QDIM, PAD, false, ContextParams>), grid, block, 0, stream, p, 0, out_vec);
    };
    using std::integral_constant;
    using std::true_type;
    using std::false_type;
    if (p.D == 64) run(integral_constant<int, 64>{}, integral_constant<int, 64>{}, false_type{});
    else if (p.D == 96) run(integral_constant<int, 96>{}, integral_constant<int, 96>{}, false_type{});
    else if (p.D == 128) run(integral_constant<int, 128>{}, integral_constant<int, 128>{}, false_type{});
    else if (p.D < 64) run(integral_constant<int, 64>{}, integral_constant<int, 64>{}, true_type{});
    else if (p.D <= 80) run(integral_constant<int, 96>{}, integral_constant<int, 80>{}, true_type{});
    else if (p.D < 96) run(integral_constant<int, 96>{}, integral_constant<int, 96>{}, true_type{});
    else run(integral_constant<int, 128>{}, integral_constant<int, 128>{}, true_type{});
}

int launch_context_tiles(const ContextParams &p0, const ContextTilesLaunch &how, fhip_dtype dtype, hipStream_t stream) {
    if (dtype == FHIP_F32) return launch_context_terms(p0, how, stream);
    if (p0.D > 128) return launch_context_wide(p0, how, dtype, stream);
    ContextParams p = p0;
    set_tiles_launch(p, how);
    if (dtype == FHIP_F16) launch_type<half_t>(p, how, stream);
    else launch_type<bf16_t>(p, how, stream);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

}  // namespace fhip
