// Prefill attention for f16 / bf16 at head dims above 192: which calls the kernel of attn_prefill_mfma_rows32_kernel.h takes, and the launch.
#include <type_traits>

#include "attn_prefill_mfma_rows32_kernel.h"

namespace fhip {

namespace {

template <typename T>
int launch_rows32_t(const AttnParams &p, hipStream_t stream) {
    const int nqb = (p.Sq + R32_BM - 1) / R32_BM;
    const long blocks = (long)nqb * p.B * p.H * (p.pf_nsplit > 1 ? p.pf_nsplit : 1);
    if (blocks > 0x7fffffffL) {
        set_error("prefill: too many workgroups (%ld)", blocks);
        return FHIP_ERR_UNSUPPORTED;
    }
    // rows of the output can be written in 16-byte pieces when they are contiguous and aligned
    const int oeb = p.out_f32 ? 4 : 2;
    int out_vec = p.os[3] == 1 && ((uintptr_t)p.out % 16 == 0);
    for (int i = 0; i < 3; i++)
        if ((p.os[i] * oeb) % 16 != 0) out_vec = 0;
    if (p.pf_nsplit > 1) FHIP_LAUNCH_MAIN((prefill_mfma_wide_rows32_kernel<T, true, AttnParams>), dim3((unsigned)blocks), dim3(256), stream, p, p, nqb, out_vec);
    else FHIP_LAUNCH_MAIN((prefill_mfma_wide_rows32_kernel<T, false, AttnParams>), dim3((unsigned)blocks), dim3(256), stream, p, p, nqb, out_vec);
    FHIP_HIP_CHECK(hipGetLastError());
    if (p.pf_nsplit > 1) return launch_prefill_merge(p, std::is_same<T, half_t>::value ? FHIP_F16 : FHIP_BF16, stream);
    return FHIP_OK;
}

}  // namespace

// The calls this form takes: head dims above 192 (padded with zeros up to 256: f16, 4096 x 4096 causal, 16 heads, head_dim
// 200 / 224 / 232 195 / 208 / 218 -> 155 / 160 / 161 us against the 16-row form; up to 192 a wavefront of that form holds
// 32 rows itself), no packed heads, keys split over workgroups only from 65 query rows on (f16, head_dim 256, 16 / 4
// heads, 128 rows on B8 x 8192 keys 263 -> 186 us, on B1 x 32768 keys 120 -> 102), and a scale whose power-of-two part Q
// can carry without leaving the 16-bit type's normal range.
bool prefill_mfma_rows32_takes(const AttnParams &p) {
    const float scale2 = p.scale * R32_LOG2E;
    // (keys split over workgroups: from 65 query rows on; up to 64 the 16-row kernel's 64-row and packed forms serve)
    return p.D > 192 && p.D <= R32_D && p.D % 8 == 0 && (p.pf_nsplit <= 1 || p.Sq > 64) && !p.pf_pack && scale2 >= 0.00390625f &&
           scale2 < 2.0f;
}

int launch_prefill_mfma_rows32(const AttnParams &p, fhip_dtype dtype, hipStream_t stream) {
    if (dtype == FHIP_F16) return launch_rows32_t<half_t>(p, stream);
    if (dtype == FHIP_BF16) return launch_rows32_t<bf16_t>(p, stream);
    set_error("prefill MFMA kernel takes f16/bf16 only");
    return FHIP_ERR_UNSUPPORTED;
}

}  // namespace fhip
