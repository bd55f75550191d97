// Attention over one part of a context on the kernel of four 32-row wavefronts (attn_prefill_mfma_rows32_kernel.h): 16-bit tensors at head dims above 128,
// padded with zeros up to 256.
// Bound: ends of workgroups that walk few tiles, of a wavefront per SIMD: four rows of 16 sequences on 4001 shared and up to 600 own keys, 16/4 heads at 256,
// 24 us in 232 workgroups of nine or ten tiles, a round, and 4.8 of merging (two launches for the two parts: 23 and, few rows, 15.5).
#include <type_traits>

#include "attn_prefill_mfma_rows32_kernel.h"
#include "context.h"

namespace fhip {

template <typename T>
static void launch_type(const ContextParams &p, const ContextTilesLaunch &how, hipStream_t stream) {
    const dim3 grid((unsigned)how.total), block(256);
    const int bytes = p.out_f32 ? 4 : 2;
    int out_vec = p.os[3] == 1 && (uintptr_t)p.out % 16 == 0;
    for (int i = 0; i < 3; i++)
        if (p.os[i] * bytes % 16 != 0) out_vec = 0;
    if (p.slots > 1) hipLaunchKernelGGL((prefill_mfma_wide_rows32_kernel<T, true, ContextParams>), grid, block, 0, stream, p, 0, out_vec);
    else hipLaunchKernelGGL((prefill_mfma_wide_rows32_kernel<T, false, ContextParams>), grid, block, 0, stream, p, 0, out_vec);
}

int launch_context_wide(const ContextParams &p0, const ContextTilesLaunch &how, fhip_dtype dtype, hipStream_t stream) {
    ContextParams p = p0;
    set_tiles_launch(p, how);
    if (dtype == FHIP_F16) launch_type<half_t>(p, how, stream);
    else launch_type<bf16_t>(p, how, stream);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

}  // namespace fhip
