// C ABI of attention over a context in two parts: checks of arguments, planning, dispatch.
#include <cmath>
#include <cstring>

#include "context.h"
#include "handles.h"

namespace fhip {

static int bytes_of(fhip_dtype d) { return d == FHIP_F32 ? 4 : 2; }
static bool known(int d) { return d == FHIP_F32 || d == FHIP_F16 || d == FHIP_BF16; }
static bool empty(const uint32_t shape[4]) { return shape[0] == 0 || shape[1] == 0 || shape[2] == 0 || shape[3] == 0; }
static int invalid(const char *text) {
    set_error("context_attention: %s", text);
    return FHIP_ERR_INVALID_ARG;
}

static int check_shapes(const fhip_context_attn_args *a) {
    const uint32_t *qs = a->q.shape, *ks = a->k.shape, *vs = a->v.shape, *os = a->out.shape, *ps = a->prefix_k.shape, *pvs = a->prefix_v.shape;
    for (int i = 0; i < 4; i++)
        if (qs[i] > 0x7fffffffu || ks[i] > 0x7fffffffu || ps[i] > 0x7fffffffu) return invalid("dimension larger than 2^31-1");
    const uint32_t B = qs[0], H = qs[1], D = qs[3], Hkv = ks[1];
    if (Hkv == 0 ? H != 0 : H % Hkv != 0) {
        set_error("Number of Q heads (%u) must be divisible by number of K/V heads (%u)", H, Hkv);
        return FHIP_ERR_INVALID_ARG;
    }
    if (ks[0] != B || ks[3] != D) {
        set_error("K shape [%u, %u, %u, %u] does not match Q shape [%u, %u, %u, %u] in batch/head_dim", ks[0], ks[1], ks[2], ks[3], B, H, qs[2], D);
        return FHIP_ERR_INVALID_ARG;
    }
    for (int i = 0; i < 4; i++) {
        if (vs[i] != ks[i]) {
            set_error("V shape [%u, %u, %u, %u] does not match K shape [%u, %u, %u, %u]", vs[0], vs[1], vs[2], vs[3], ks[0], ks[1], ks[2], ks[3]);
            return FHIP_ERR_INVALID_ARG;
        }
        if (os[i] != qs[i]) {
            set_error("output shape [%u, %u, %u, %u] does not match Q shape [%u, %u, %u, %u]", os[0], os[1], os[2], os[3], B, H, qs[2], D);
            return FHIP_ERR_INVALID_ARG;
        }
        if (pvs[i] != ps[i]) {
            set_error("prefix V shape [%u, %u, %u, %u] does not match prefix K shape [%u, %u, %u, %u]", pvs[0], pvs[1], pvs[2], pvs[3], ps[0], ps[1],
                      ps[2], ps[3]);
            return FHIP_ERR_INVALID_ARG;
        }
    }
    if (ps[2] != 0 && (ps[0] != 1 || ps[1] != Hkv || ps[3] != D)) {
        set_error("prefix shape [%u, %u, %u, %u] does not match expected [1, %u, _, %u]", ps[0], ps[1], ps[2], ps[3], Hkv, D);
        return FHIP_ERR_INVALID_ARG;
    }
    return FHIP_OK;
}

static int validate_context(const fhip_context_attn_args *a) {
    if (!a) return invalid("args is NULL");
    if (!known(a->dtype) || !known(a->out_dtype)) {
        set_error("unknown dtype %d / out_dtype %d", (int)a->dtype, (int)a->out_dtype);
        return FHIP_ERR_INVALID_ARG;
    }
    if (a->out_dtype != a->dtype && a->out_dtype != FHIP_F32) return invalid("out_dtype must equal dtype, or be f32 for 16-bit inputs");
    const int rc = check_shapes(a);
    if (rc) return rc;
    const uint32_t *qs = a->q.shape, *os = a->out.shape;
    if (!empty(qs)) {
        if (!a->q.ptr || !a->out.ptr) return invalid("q and out need device pointers");
        if (a->k.shape[2] != 0 && (!a->k.ptr || !a->v.ptr)) return invalid("k and v need device pointers");
        if (a->prefix_k.shape[2] != 0 && (!a->prefix_k.ptr || !a->prefix_v.ptr)) return invalid("prefix_k and prefix_v need device pointers");
        for (int i = 0; i < 4; i++)
            if (os[i] > 1 && a->out.stride[i] == 0) {
                set_error("output stride %d is 0 (overlapping writes)", i);
                return FHIP_ERR_INVALID_ARG;
            }
    }
    if (!std::isfinite(a->scale)) return invalid("scale must be finite");
    if (a->window < 0 || a->q_pos_offset < 0 || a->sinks < 0) return invalid("window, q_pos_offset and sinks must be >= 0");
    if (a->q_pos_offset > INT64_MAX / 4 || a->window > INT64_MAX / 4) return invalid("q_pos_offset or window of 2^61 and more");  // positions are added up in 64 bits
    if (a->q_positions && !a->causal && a->window == 0) return invalid("q_positions needs a causal mask or a window");
    if (qs[3] > 512) {
        set_error("head_dim %u > 512 has no kernel", qs[3]);
        return FHIP_ERR_UNSUPPORTED;
    }
    if ((uint64_t)qs[1] * qs[2] > 0x7fffffffull - 4096 || (uint64_t)qs[0] * qs[1] * qs[2] > 0x7fffffffull - 4096) {
        set_error("context_attention: more than 2^31-4097 query rows in one call");
        return FHIP_ERR_UNSUPPORTED;
    }
    if ((uint64_t)a->prefix_k.shape[2] + a->k.shape[2] > 0x7fffffffull - 4096) {  // (the kernels look a few tiles ahead in 32 bits)
        set_error("context_attention: more than 2^31-4097 keys");
        return FHIP_ERR_UNSUPPORTED;
    }
    return FHIP_OK;
}

static void fill_context(const fhip_context_attn_args *a, int cus, ContextParams *p) {
    memset((void *)p, 0, sizeof(*p));
    const uint64_t e = (uint64_t)bytes_of(a->dtype);
    auto start = [&](const fhip_tensor4 &t, uint64_t bytes) { return t.ptr ? (char *)t.ptr + t.offset * bytes : nullptr; };
    p->q = start(a->q, e), p->k = start(a->k, e), p->v = start(a->v, e), p->pk = start(a->prefix_k, e), p->pv = start(a->prefix_v, e);
    p->out = start(a->out, (uint64_t)bytes_of(a->out_dtype));
    for (int i = 0; i < 4; i++) {
        p->qs[i] = a->q.stride[i], p->ks[i] = a->k.stride[i], p->vs[i] = a->v.stride[i], p->os[i] = a->out.stride[i];
        if (i > 0) p->pks[i - 1] = a->prefix_k.stride[i], p->pvs[i - 1] = a->prefix_v.stride[i];
    }
    p->kv_lens = a->kv_lens, p->q_positions = a->q_positions;
    p->B = (int)a->q.shape[0], p->H = (int)a->q.shape[1], p->Sq = (int)a->q.shape[2], p->D = (int)a->q.shape[3];
    p->Hkv = (int)a->k.shape[1], p->Skv = (int)a->k.shape[2], p->P = (int)a->prefix_k.shape[2];
    p->G = p->H / p->Hkv;
    p->analytic = 1, p->causal = a->causal ? 1 : 0;
    p->q_pos_offset = a->q_pos_offset, p->window = a->window;
    p->sinks = a->window > 0 ? (int)(a->sinks < 0x7fffffff ? a->sinks : 0x7fffffff) : 0;
    p->scale = a->scale;
    p->out_f32 = a->out_dtype == FHIP_F32 && a->dtype != FHIP_F32;
    p->cus = cus > 0 ? cus : 256;
}

static int run_plan(ContextParams &p, const ContextPlan &plan, fhip_dtype dtype, hipStream_t stream) {
    if (plan.any) return launch_context_any(p, dtype, stream);
    p.slots = plan.slots;
    int rc = FHIP_OK;
    if (plan.tiles.jobs) rc = launch_context_tiles(p, plan.tiles, dtype, stream);
    if (!rc && plan.rows.total) rc = launch_context_rows(p, plan.rows, dtype, stream);
    return rc || plan.slots == 1 ? rc : launch_context_merge(p, dtype, stream);
}

// What a call that passes the checks runs on a device of `cus` compute units, for tests: of its up to two parts, behind each other, their query rows (0: no such
// part), whether the kernel for every call takes them, rows per workgroup, key groups and jobs of the tiled launch, each job's {fold, with_prefix, with_own, shares},
// the few-row launch's columns (0: no such launch), its jobs' {prefix, shares} (no job: 0 shares), and the places of a row in the workspace.
constexpr int FORM_WORDS = 19;
void context_forms(const fhip_context_attn_args *args, int cus, int32_t *forms) {
    ContextParams p;
    fill_context(args, cus, &p);
    const ContextCall call = context_call(p, args->dtype);
    memset(forms, 0, 2 * FORM_WORDS * sizeof(int32_t));
    for (int i = 0; i < call.parts; i++) {
        const ContextPlan &plan = call.plan[i];
        int32_t *f = forms + i * FORM_WORDS;
        *f++ = call.rows[i], *f++ = plan.any;
        if (plan.any) continue;
        *f++ = plan.tiles.rows_per_group, *f++ = plan.tiles.key_groups, *f++ = plan.tiles.jobs;
        for (int j = 0; j < 2; j++, f += 4)
            if (j < plan.tiles.jobs) f[0] = plan.tiles.job[j].fold, f[1] = plan.tiles.job[j].with_prefix, f[2] = plan.tiles.job[j].with_own, f[3] = plan.tiles.job[j].shares;
        *f++ = plan.rows.total ? plan.rows.columns : 0;
        for (const ContextRowsJob &job : plan.rows.job) *f++ = job.prefix, *f++ = plan.rows.total ? job.nsplit : 0;
        *f = plan.slots;
    }
}

}  // namespace fhip

using namespace fhip;

extern "C" {

int fhip_context_attention_validate(const fhip_context_attn_args *args) { return validate_context(args); }

int fhip_context_attention_workspace_bytes(const fhip_context_attn_args *args, int32_t compute_units, size_t *bytes) {
    if (!bytes) return invalid("bytes is NULL");
    *bytes = 0;
    const int rc = validate_context(args);
    if (rc || empty(args->q.shape)) return rc;
    if (args->k.shape[2] == 0 && args->prefix_k.shape[2] == 0) return FHIP_OK;
    ContextParams p;
    fill_context(args, compute_units, &p);
    *bytes = context_call(p, args->dtype).bytes;
    return FHIP_OK;
}

int fhip_context_attention(fhip_stream *s, const fhip_context_attn_args *args) {
    if (!s) return invalid("stream is NULL");
    int rc = validate_context(args);
    if (rc || empty(args->q.shape)) return rc;
    FHIP_HIP_CHECK(hipSetDevice(s->dev->ordinal));
    if (args->k.shape[2] == 0 && args->prefix_k.shape[2] == 0) {  // no keys at all: zeros, as fhip_flash_attention
        char *out = (char *)args->out.ptr + args->out.offset * (uint64_t)bytes_of(args->out_dtype);
        return launch_fill_zero_rows(out, args->out.stride, args->out.shape, bytes_of(args->out_dtype), s->s);
    }
    ContextParams p;
    fill_context(args, s->dev->prop.multiProcessorCount, &p);
    const ContextCall call = context_call(p, args->dtype);
    if (call.bytes && (!args->workspace || ((uintptr_t)args->workspace & 15) != 0 || args->workspace_bytes < call.bytes)) {
        set_error("context_attention: needs %zu bytes of 16-byte aligned workspace, got %zu", call.bytes, args->workspace ? args->workspace_bytes : 0);
        return FHIP_ERR_WORKSPACE;
    }
    p.partials = (float *)args->workspace, p.pf_pitch = p.D + 4;
    for (int i = 0; i < call.parts && !rc; i++) {
        ContextParams part = p;
        part.q = (const char *)p.q + call.first_row[i] * p.qs[2] * bytes_of(args->dtype);
        part.out = (char *)p.out + call.first_row[i] * p.os[2] * bytes_of(args->out_dtype);
        part.Sq = call.rows[i], part.q_pos_offset = p.q_pos_offset + call.first_row[i];
        rc = run_plan(part, call.plan[i], args->dtype, s->s);
    }
    return rc;
}

}  // extern "C"
