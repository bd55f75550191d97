// Attention over a context in two parts, the kernel for everything that the tiled ones do not take: any element type, any strides, head
// dims to 512.  One wavefront owns one query row; its lanes split 64 keys for the scores and the head's dims for the weighted sum, weights
// pass from lane to lane.  Only keys that the row sees are touched.
//   s_j = scale * q . k_j;  out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s), the maximum and the sums running, in f32
// Bound: every key is read once per query row, a key per lane (rows of a tensor apart): 16 sequences of one token on 4112 visible f16 keys of
// 32/8 heads at 128 take 4.0 ms, 8192 rows under a window of 4096 185 (the other kernels: 0.05 and 0.39).
#include "context_device.h"

namespace fhip {

constexpr int CA_WAVES = 4;
constexpr int CA_DIMS = 8;  // a lane's dims: head_dim <= 512

template <typename T>
__global__ __launch_bounds__(64 * CA_WAVES) void context_any_kernel(ContextParams p) {
    __shared__ float q_lds[CA_WAVES][64 * CA_DIMS];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, D = p.D;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * CA_WAVES + wave;
    if (row >= (int64_t)p.B * p.H * p.Sq) return;  // (a whole wavefront, and no barrier follows)
    const int i = (int)(row % p.Sq), h = (int)(row / p.Sq % p.H), b = (int)(row / ((int64_t)p.Sq * p.H)), g = h / p.G;

    const T *q = (const T *)p.q + b * p.qs[0] + h * p.qs[1] + i * p.qs[2];
    for (int d = lane; d < D; d += 64) q_lds[wave][d] = to_float(q[d * p.qs[3]]);
    wave_lds_sync();

    const ContextRow seen = context_row(p, b, i);
    float m = -INFINITY, l = 0.0f, acc[CA_DIMS];
#pragma unroll
    for (int t = 0; t < CA_DIMS; t++) acc[t] = 0.0f;

    // keys [from, to) of one tensor pair
    auto walk = [&](const T *k, int64_t k_row, int64_t k_dim, const T *v, int64_t v_row, int64_t v_dim, int from, int to) {
        for (int j0 = from; j0 < to; j0 += 64) {
            const int count = min(64, to - j0);
            float s = -INFINITY;
            if (lane < count) {
                const T *kr = k + (j0 + lane) * k_row;
                float dot = 0.0f;
                for (int d = 0; d < D; d++) dot = fmaf(q_lds[wave][d], to_float(kr[d * k_dim]), dot);
                s = dot * p.scale;
            }
            const float m_new = fmaxf(m, wave_max(s));
            // (a NaN among the scores passes the maximum by and reaches the sums)
            const float reference = m_new == -INFINITY ? 0.0f : m_new;
            const float weight = expf(s - reference), moved = expf(m - reference);
            l = l * moved + wave_sum(weight);
            m = m_new;
#pragma unroll
            for (int t = 0; t < CA_DIMS; t++) {
                const int d = lane + 64 * t;
                if (d < D) {
                    float a = acc[t] * moved;
                    const T *vr = v + j0 * v_row + d * v_dim;
                    for (int j = 0; j < count; j++) a = fmaf(read_lane(weight, j), to_float(vr[j * v_row]), a);
                    acc[t] = a;
                }
            }
        }
    };
    const T *pk = (const T *)p.pk + g * p.pks[0], *pv = (const T *)p.pv + g * p.pvs[0];
    const T *k = (const T *)p.k + b * p.ks[0] + g * p.ks[1], *v = (const T *)p.v + b * p.vs[0] + g * p.vs[1];
    const int from[2] = {0, seen.lo}, to[2] = {seen.first, seen.hi};
#pragma unroll 1
    for (int part = 0; part < 2; part++) {
        walk(pk, p.pks[1], p.pks[2], pv, p.pvs[1], p.pvs[2], from[part], min(to[part], p.P));
        walk(k, p.ks[2], p.ks[3], v, p.vs[2], p.vs[3], max(from[part], p.P) - p.P, to[part] - p.P);
    }

    const int64_t at = b * p.os[0] + h * p.os[1] + i * p.os[2];
#pragma unroll
    for (int t = 0; t < CA_DIMS; t++) {
        const int d = lane + 64 * t;
        if (d < D) {
            const float o = acc[t] / l;  // no visible key: 0 / 0 = NaN
            if (p.out_f32 || sizeof(T) == 4) ((float *)p.out)[at + d * p.os[3]] = o;
            else ((T *)p.out)[at + d * p.os[3]] = from_float<T>(o);
        }
    }
}

int launch_context_any(const ContextParams &p, fhip_dtype dtype, hipStream_t stream) {
    const int64_t rows = (int64_t)p.B * p.H * p.Sq;
    const dim3 grid = rows_grid((rows + CA_WAVES - 1) / CA_WAVES), block(64 * CA_WAVES);
    if (dtype == FHIP_F32) hipLaunchKernelGGL(context_any_kernel<float>, grid, block, 0, stream, p);
    else if (dtype == FHIP_F16) hipLaunchKernelGGL(context_any_kernel<half_t>, grid, block, 0, stream, p);
    else hipLaunchKernelGGL(context_any_kernel<bf16_t>, grid, block, 0, stream, p);
    FHIP_HIP_CHECK(hipGetLastError());
    return FHIP_OK;
}

}  // namespace fhip
