// C-ABI layer of the 8-bit key / value cache: argument checks, launch parameters, the growable cache.  Host code only.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

#include "handles.h"
#include "q8.h"

namespace fhip {

static int bytes_of(fhip_dtype d) { return d == FHIP_F32 ? 4 : 2; }
static bool known(int d) { return d == FHIP_F32 || d == FHIP_F16 || d == FHIP_BF16; }
static bool block_ok(uint32_t T) { return T == 1 || T == 8 || T == 16 || T == 32 || T == 64; }
static uint32_t pitch_of(uint32_t D) { return (D + 15) & ~15u; }
static bool empty(const uint32_t s[4]) { return s[0] == 0 || s[1] == 0 || s[2] == 0 || s[3] == 0; }

static int invalid(const char *what) {
    set_error("%s", what);
    return FHIP_ERR_INVALID_ARG;
}

static int check_format(int format, uint32_t block_tokens) {
    if (format != FHIP_Q8_INT8 && format != FHIP_Q8_E4M3) {
        set_error("q8: unknown format %d", format);
        return FHIP_ERR_INVALID_ARG;
    }
    if (!block_ok(block_tokens)) {
        set_error("q8: block_tokens %u is none of 1, 8, 16, 32, 64", block_tokens);
        return FHIP_ERR_INVALID_ARG;
    }
    return FHIP_OK;
}
static int check_dim(uint32_t D) {
    if (D == 0 || D % 8 != 0 || D > Q8_MAX_DIM) {
        set_error("q8: head_dim %u is no multiple of 8 up to %d", D, Q8_MAX_DIM);
        return FHIP_ERR_UNSUPPORTED;
    }
    return FHIP_OK;
}
// a view of codes and scales; `written`: rows must not overlap
static int check_view(const fhip_q8_tensor *x, const char *name, bool written) {
    int rc = check_format(x->format, x->block_tokens);
    if (rc) return rc;
    if (x->first >= x->block_tokens) {
        set_error("q8: %s: first %u is not below block_tokens %u", name, x->first, x->block_tokens);
        return FHIP_ERR_INVALID_ARG;
    }
    for (int i = 0; i < 4; i++)
        if (x->shape[i] > 0x7fffffffu) return invalid("dimension larger than 2^31-1");
    if ((uint64_t)x->shape[2] + x->block_tokens > 0x7fffffffull) return invalid("q8: more than 2^31-1 rows");
    if (empty(x->shape)) return FHIP_OK;
    if ((rc = check_dim(x->shape[3]))) return rc;
    if (!x->codes || !x->scales) {
        set_error("q8: %s needs codes and scales", name);
        return FHIP_ERR_INVALID_ARG;
    }
    if (((uintptr_t)x->codes + x->offset) % 16 != 0 || x->stride[0] % 16 != 0 || x->stride[1] % 16 != 0 || x->stride[2] % 16 != 0 ||
        (uintptr_t)x->scales % 4 != 0) {
        set_error("q8: %s: codes and strides have to be multiples of 16 bytes, scales of 4", name);
        return FHIP_ERR_INVALID_ARG;
    }
    if (x->shape[2] > 1 && (x->stride[2] < (int64_t)pitch_of(x->shape[3]) || x->stride[2] >= (1 << 26))) {
        set_error("q8: %s: row stride %lld is below a row or 2^26 and more", name, (long long)x->stride[2]);
        return FHIP_ERR_INVALID_ARG;
    }
    if (written)
        for (int i = 0; i < 2; i++)
            if (x->shape[i] > 1 && (x->stride[i] == 0 || x->scale_stride[i] == 0)) {
                set_error("q8: %s: stride %d is 0 (overlapping writes)", name, i);
                return FHIP_ERR_INVALID_ARG;
            }
    return FHIP_OK;
}
static int check_pair(const fhip_q8_tensor *k, const fhip_q8_tensor *v, bool written) {
    int rc = check_view(k, "k", written);
    if (rc || (rc = check_view(v, "v", written))) return rc;
    for (int i = 0; i < 4; i++)
        if (k->shape[i] != v->shape[i]) {
            set_error("V shape [%u, %u, %u, %u] does not match K shape [%u, %u, %u, %u]", v->shape[0], v->shape[1], v->shape[2], v->shape[3],
                      k->shape[0], k->shape[1], k->shape[2], k->shape[3]);
            return FHIP_ERR_INVALID_ARG;
        }
    if (k->format != v->format || k->block_tokens != v->block_tokens) return invalid("q8: k and v differ in format or block_tokens");
    return FHIP_OK;
}
static Q8View view_of(const fhip_q8_tensor &x) {
    Q8View v;
    v.codes = (uint8_t *)x.codes + x.offset;
    v.scales = (float *)x.scales + x.scale_offset;
    for (int i = 0; i < 3; i++) v.cs[i] = x.stride[i];
    if (x.shape[2] <= 1) v.cs[2] = pitch_of(x.shape[3]);
    for (int i = 0; i < 2; i++) v.ss[i] = x.scale_stride[i];
    v.rows = x.shape[2];
    v.log2_block = __builtin_ctz(x.block_tokens);
    v.first = (int32_t)x.first;
    return v;
}

// rows readable four elements at a time
static bool fours(const fhip_tensor4 &t, int eb) {
    if (t.stride[3] != 1 || ((uintptr_t)t.ptr + t.offset * (uint64_t)eb) % (4 * eb) != 0) return false;
    for (int i = 0; i < 3; i++)
        if (t.shape[i] > 1 && t.stride[i] % 4 != 0) return false;
    return true;
}

// ---- append -----------------------------------------------------------------------------------------------------------------------------

struct AppendShape {
    uint32_t B, Hkv, n, D;
};

static int check_norm(const fhip_rms_norm *n) {
    return n && (!n->weight || !known(n->dtype)) ? invalid("rms norm: NULL weight or bad dtype") : FHIP_OK;
}

// everything but the place that the rows go to
static int check_new_rows(const fhip_q8_append_args *a, AppendShape *s) {
    if (!known(a->in_dtype)) return invalid("q8_append: bad dtype");
    const uint32_t *ks = a->k_new.shape;
    *s = {ks[0], ks[1], ks[2], ks[3]};
    for (int i = 0; i < 4; i++) {
        if (a->v_new.shape[i] != ks[i]) {
            set_error("q8_append: key shape [%u, %u, %u, %u] != value shape [%u, %u, %u, %u]", ks[0], ks[1], ks[2], ks[3],
                      a->v_new.shape[0], a->v_new.shape[1], a->v_new.shape[2], a->v_new.shape[3]);
            return FHIP_ERR_INVALID_ARG;
        }
        if (ks[i] > 0x7fffffffu) return invalid("dimension larger than 2^31-1");
    }
    if (empty(ks)) return invalid("q8_append: empty tensor");
    int rc = check_dim(s->D);
    if (rc) return rc;
    if (!a->k_new.ptr || !a->v_new.ptr) return invalid("q8_append: new keys/values need device pointers");
    if (a->rope) {
        const fhip_rope_tables *r = a->rope;
        if (!r->cos || !r->sin) return invalid("rope: NULL tables");
        if (r->table_rows == 0) return invalid("rope: tables without rows");  // (rows that are left out are read at position 0)
        if (r->table_rows > 0x7fffffffffffull || r->start_pos > r->table_rows || (!a->lens && s->n > r->table_rows - r->start_pos)) {
            set_error("rope: positions %llu..%llu exceed the %llu rows of the tables", (unsigned long long)r->start_pos,
                      (unsigned long long)(r->start_pos + s->n), (unsigned long long)r->table_rows);
            return FHIP_ERR_INVALID_ARG;
        }
    }
    if ((rc = check_norm(a->k_norm)) || (rc = check_norm(a->q_norm))) return rc;
    uint64_t heads = s->Hkv;
    if (a->q.ptr) {
        if (!known(a->q_dtype) || !known(a->q_out_dtype)) return invalid("q8_append: bad dtype of q or q_out");
        if (!a->q_out.ptr) return invalid("q8_append: q without q_out");
        for (int i = 0; i < 4; i++)
            if (a->q_out.shape[i] != a->q.shape[i]) return invalid("q8_append: q_out shape differs from q's");
        if (a->q.shape[0] != s->B || a->q.shape[2] != s->n || a->q.shape[3] != s->D || a->q.shape[1] == 0) {
            set_error("q8_append: q shape [%u, %u, %u, %u] does not match [%u, _, %u, %u]", a->q.shape[0], a->q.shape[1], a->q.shape[2],
                      a->q.shape[3], s->B, s->n, s->D);
            return FHIP_ERR_INVALID_ARG;
        }
        for (int i = 0; i < 4; i++)
            if (a->q_out.shape[i] > 1 && a->q_out.stride[i] == 0) return invalid("q8_append: output stride is 0 (overlapping writes)");
        heads = std::max<uint64_t>(heads, a->q.shape[1]);
    }
    // slots are numbered in 32 bits, a last workgroup's beyond the end included
    if (heads > 0x40000000u || s->B * heads > 0x40000000u / ((uint64_t)s->n + 2 * Q8_MAX_BLOCK)) {
        set_error("q8_append: more than 2^30 rows in one call");
        return FHIP_ERR_UNSUPPORTED;
    }
    return FHIP_OK;
}

// The new rows from `skip` on to row `row` of k / v; all of q.
static int append_rows(hipStream_t stream, const fhip_q8_append_args *a, const AppendShape &s, const fhip_q8_tensor &k,
                       const fhip_q8_tensor &v, uint64_t row, uint32_t skip) {
    Q8AppendParams p;
    memset(&p, 0, sizeof(p));
    p.D = (int)s.D;
    p.format = k.format;
    p.row = (int64_t)row;
    p.lens = a->lens;
    p.counts = a->counts;
    int64_t pos0 = 0;
    int mode = 2;
    if (a->rope) {
        p.cos = a->rope->cos, p.sin = a->rope->sin;
        p.table_rows = (int64_t)a->rope->table_rows;
        pos0 = (int64_t)a->rope->start_pos;
        mode = a->rope->interleaved ? 1 : 0;
    }
    const uint32_t T = k.block_tokens, n = s.n - skip;
    const bool alone = T == 1 || s.n == 1;  // new rows in blocks of their own
    auto job = [&](const fhip_tensor4 &src, fhip_dtype dtype, uint32_t heads, int md, const fhip_rms_norm *norm) -> Q8Rows & {
        Q8Rows &j = p.job[p.jobs++];
        j.src = (const char *)src.ptr + src.offset * (uint64_t)bytes_of(dtype);
        for (int i = 0; i < 4; i++) j.s[i] = src.stride[i];
        j.src_dtype = dtype;
        j.vec = fours(src, bytes_of(dtype));
        j.heads = (int32_t)heads;
        j.mode = md;
        if (norm) j.norm_w = norm->weight, j.norm_b = norm->bias, j.norm_dtype = norm->dtype, j.eps = norm->eps;
        return j;
    };
    if (a->q.ptr) {
        Q8Rows &j = job(a->q, a->q_dtype, a->q.shape[1], mode, a->q_norm);
        j.is_q = 1;
        j.n = (int32_t)s.n;
        j.pos0 = pos0;
        j.span = s.n;
        j.dst_dtype = a->q_out_dtype;
        j.dst = (char *)a->q_out.ptr + a->q_out.offset * (uint64_t)bytes_of(a->q_out_dtype);
        for (int i = 0; i < 4; i++) j.d[i] = a->q_out.stride[i];
        j.vec = j.vec && fours(a->q_out, bytes_of(a->q_out_dtype));
        j.out.rows = a->lens ? (int64_t)k.shape[2] : INT64_MAX / 2;  // without lens the host has seen that the rows have their places
        j.total = s.B * a->q.shape[1] * j.span;
    }
    for (int side = 0; side < 2; side++) {
        fhip_tensor4 src = side == 0 ? a->k_new : a->v_new;
        src.offset += (uint64_t)((int64_t)skip * src.stride[2]);
        Q8Rows &j = job(src, a->in_dtype, s.Hkv, side == 0 ? mode : 2, side == 0 ? a->k_norm : nullptr);
        j.n = (int32_t)n;
        j.pos0 = pos0 + skip;
        j.out = view_of(side == 0 ? k : v);
        j.span = alone ? n : (n + 2 * (T - 1)) / T * T;
        j.total = s.B * s.Hkv * j.span;
    }
    return launch_q8_append(p, (int)T, alone, a->q_norm || a->k_norm, stream);
}

// ---- attention --------------------------------------------------------------------------------------------------------------------------

static int validate_attention(const fhip_q8_attn_args *a) {
    if (!a) return invalid("args is NULL");
    if (!known(a->dtype) || !known(a->out_dtype)) {
        set_error("unknown dtype %d / out_dtype %d", (int)a->dtype, (int)a->out_dtype);
        return FHIP_ERR_INVALID_ARG;
    }
    if (a->out_dtype != a->dtype && a->out_dtype != FHIP_F32) return invalid("out_dtype must equal dtype, or be f32 for 16-bit inputs");
    const uint32_t *qs = a->q.shape, *ks = a->k.shape, *os = a->out.shape;
    for (int i = 0; i < 4; i++)
        if (qs[i] > 0x7fffffffu) return invalid("dimension larger than 2^31-1");
    const uint32_t B = qs[0], H = qs[1], Sq = qs[2], D = qs[3], Hkv = ks[1], Skv = ks[2];
    int rc = check_pair(&a->k, &a->v, false);
    if (rc) return rc;
    if (Hkv == 0 ? H != 0 : H % Hkv != 0) {
        set_error("Number of Q heads (%u) must be divisible by number of K/V heads (%u)", H, Hkv);
        return FHIP_ERR_INVALID_ARG;
    }
    if (ks[0] != B || ks[3] != D) {
        set_error("K shape [%u, %u, %u, %u] does not match Q shape [%u, %u, %u, %u] in batch/head_dim", ks[0], ks[1], ks[2], ks[3], B, H, Sq, D);
        return FHIP_ERR_INVALID_ARG;
    }
    for (int i = 0; i < 4; i++)
        if (os[i] != qs[i]) {
            set_error("output shape [%u, %u, %u, %u] does not match Q shape [%u, %u, %u, %u]", os[0], os[1], os[2], os[3], B, H, Sq, D);
            return FHIP_ERR_INVALID_ARG;
        }
    if (!empty(qs)) {
        if (!a->q.ptr || !a->out.ptr) return invalid("q and out need device pointers");
        if ((rc = check_dim(D))) return rc;
        for (int i = 0; i < 4; i++)
            if (os[i] > 1 && a->out.stride[i] == 0) {
                set_error("output stride %d is 0 (overlapping writes)", i);
                return FHIP_ERR_INVALID_ARG;
            }
    }
    if (!std::isfinite(a->scale)) return invalid("scale must be finite");
    switch (a->mask_kind) {
        case FHIP_MASK_NONE:
            if (a->mask.ptr) return invalid("mask pointer given with FHIP_MASK_NONE");
            break;
        case FHIP_MASK_QK:
        case FHIP_MASK_BATCH_KEY: {
            const uint32_t rows = a->mask_kind == FHIP_MASK_QK ? Sq : B;
            if (a->mask.shape[0] != rows || a->mask.shape[1] != Skv) {
                set_error("%s shape [%u, %u] does not match expected [%u, %u]", a->mask_kind == FHIP_MASK_QK ? "QKMask" : "BatchKeyMask",
                          a->mask.shape[0], a->mask.shape[1], rows, Skv);
                return FHIP_ERR_INVALID_ARG;
            }
            if (!a->mask.ptr) return invalid("mask_kind set but mask pointer is NULL");
            break;
        }
        default:
            set_error("unknown mask_kind %d", (int)a->mask_kind);
            return FHIP_ERR_INVALID_ARG;
    }
    if (a->analytic.enabled) {
        if (a->mask_kind != FHIP_MASK_NONE) return invalid("analytic mask and mask tensor are mutually exclusive");
        if (a->analytic.window < 0 || a->analytic.q_pos_offset < 0) return invalid("analytic mask: window and q_pos_offset must be >= 0");
        // positions are added up in 64 bits
        if (a->analytic.q_pos_offset > INT64_MAX / 4 || a->analytic.window > INT64_MAX / 4) return invalid("analytic mask: offset or window of 2^61 and more");
    } else if (a->q_positions) {
        return invalid("q_positions needs an analytic mask");
    }
    if ((uint64_t)H * Sq > 0x7fffffffull || (uint64_t)B * H * Sq > 0x7fffffffull) {
        set_error("q8_attention: more than 2^31-1 query rows in one call");
        return FHIP_ERR_UNSUPPORTED;
    }
    if (Skv > 0x7fffffffu - 4096) {  // (the kernels look a few tiles ahead in 32 bits)
        set_error("q8_attention: more than 2^31-4097 keys");
        return FHIP_ERR_UNSUPPORTED;
    }
    return FHIP_OK;
}

static void fill_attention(const fhip_q8_attn_args *a, int cus, Q8AttnParams *p) {
    memset(p, 0, sizeof(*p));
    p->q = (const char *)a->q.ptr + a->q.offset * (uint64_t)bytes_of(a->dtype);
    p->out = (char *)a->out.ptr + a->out.offset * (uint64_t)bytes_of(a->out_dtype);
    for (int i = 0; i < 4; i++) p->qs[i] = a->q.stride[i], p->os[i] = a->out.stride[i];
    p->q_vec = fours(a->q, bytes_of(a->dtype));
    p->out_vec = fours(a->out, bytes_of(a->out_dtype));
    p->q_dtype = a->dtype;
    p->out_dtype = a->out_dtype;
    p->k = view_of(a->k), p->v = view_of(a->v);
    p->B = (int)a->q.shape[0], p->H = (int)a->q.shape[1], p->Sq = (int)a->q.shape[2], p->D = (int)a->q.shape[3];
    p->Hkv = (int)a->k.shape[1], p->Skv = (int)a->k.shape[2];
    p->G = p->H / p->Hkv;
    p->format = a->k.format;
    if (a->analytic.enabled) {
        p->causal = a->analytic.causal ? 1 : 0;
        p->q_pos_offset = a->analytic.q_pos_offset;
        p->window = a->analytic.window;
        p->q_positions = a->q_positions;
    }
    p->kv_lens = a->kv_lens;
    if (a->mask_kind != FHIP_MASK_NONE) {
        p->mask = (const char *)a->mask.ptr + a->mask.offset * (uint64_t)bytes_of(a->dtype);
        p->ms0 = a->mask.stride[0], p->ms1 = a->mask.stride[1];
        p->mask_kind = a->mask_kind;
    }
    p->scale = a->scale;
    p->cus = cus > 0 ? cus : 256;
}

// Few columns ((query row, head of the group) pairs) per KV head: the kernel that streams the codes into registers (32 rows at a time).  It takes 16 columns
// per workgroup and the codes once for each of them (us, few and many, recorded calls: 8 sequences of 4096 keys, 32/8 heads at 128, f16, 16 columns 22 and
// 32, 32 columns 31 and 33, 48 columns 49 and 35; 8 of 4001, 16/4 at 256, bf16, 32 columns 28 and 47, 48 columns 51 and 49; 16 of 2000, 32/32 at 64, 48
// columns 66 and 121).
static Q8AttnPlan attention_plan(const Q8AttnParams &p) {
    return (int64_t)p.G * p.Sq <= 32 && p.Skv >= 32 ? q8_decode_plan(p) : q8_prefill_plan(p);
}

}  // namespace fhip

using namespace fhip;

extern "C" {

int fhip_q8_append(fhip_stream *s, const fhip_q8_append_args *args) {
    if (!s || !args) return invalid("q8_append: NULL argument");
    AppendShape sh;
    int rc = check_new_rows(args, &sh);
    if (rc || (rc = check_pair(&args->k, &args->v, true))) return rc;
    if (args->k.shape[0] != sh.B || args->k.shape[1] != sh.Hkv || args->k.shape[3] != sh.D) {
        set_error("q8_append: [%u, %u, _, %u] does not match the cache's [%u, %u, _, %u]", sh.B, sh.Hkv, sh.D, args->k.shape[0],
                  args->k.shape[1], args->k.shape[3]);
        return FHIP_ERR_INVALID_ARG;
    }
    if (args->row > 0x7fffffffull || (!args->lens && args->row + sh.n > args->k.shape[2])) {
        set_error("q8_append: rows %llu..%llu exceed the %u rows of the cache", (unsigned long long)args->row,
                  (unsigned long long)(args->row + sh.n), args->k.shape[2]);
        return FHIP_ERR_INVALID_ARG;
    }
    if (empty(args->k.shape)) return FHIP_OK;  // (lens: no room for any row)
    FHIP_HIP_CHECK(hipSetDevice(s->dev->ordinal));
    return append_rows(s->s, args, sh, args->k, args->v, args->row, 0);
}

int fhip_q8_dequantize(fhip_stream *s, const fhip_q8_tensor *x, uint64_t row, const int32_t *lens, const fhip_tensor4 *out,
                       fhip_dtype out_dtype) {
    if (!s || !x || !out || !known(out_dtype)) return invalid("q8_dequantize: NULL argument or bad dtype");
    int rc = check_view(x, "x", false);
    if (rc) return rc;
    const uint32_t *os = out->shape;
    if (os[0] != x->shape[0] || os[1] != x->shape[1] || os[3] != x->shape[3] || os[2] > 0x7fffffffu) {
        set_error("q8_dequantize: output shape [%u, %u, %u, %u] does not match [%u, %u, _, %u]", os[0], os[1], os[2], os[3], x->shape[0],
                  x->shape[1], x->shape[3]);
        return FHIP_ERR_INVALID_ARG;
    }
    if (row > 0x7fffffffull || (!lens && row + os[2] > x->shape[2])) {
        set_error("q8_dequantize: rows %llu..%llu exceed the %u rows of the cache", (unsigned long long)row, (unsigned long long)(row + os[2]),
                  x->shape[2]);
        return FHIP_ERR_INVALID_ARG;
    }
    if (empty(os) || empty(x->shape)) return FHIP_OK;
    if (!out->ptr) return invalid("q8_dequantize: out needs a device pointer");
    for (int i = 0; i < 4; i++)
        if (os[i] > 1 && out->stride[i] == 0) {
            set_error("output stride %d is 0 (overlapping writes)", i);
            return FHIP_ERR_INVALID_ARG;
        }
    if ((uint64_t)os[1] * (os[3] / 8) > 0x7fffffffull) {  // (the heads of a row go in one launch)
        set_error("q8_dequantize: 2^34 elements or more in a row of all heads");
        return FHIP_ERR_UNSUPPORTED;
    }
    Q8ReadParams p;
    memset(&p, 0, sizeof(p));
    p.x = view_of(*x);
    p.out = (char *)out->ptr + out->offset * (uint64_t)bytes_of(out_dtype);
    for (int i = 0; i < 4; i++) p.os[i] = out->stride[i];
    p.out_dtype = out_dtype;
    p.vec = fours(*out, bytes_of(out_dtype));
    p.B = (int)os[0], p.H = (int)os[1], p.n = (int)os[2], p.D = (int)os[3];
    p.format = x->format;
    p.row = (int64_t)row;
    p.lens = lens;
    FHIP_HIP_CHECK(hipSetDevice(s->dev->ordinal));
    return launch_q8_dequantize(p, s->s);
}

int fhip_q8_attention_validate(const fhip_q8_attn_args *args) { return validate_attention(args); }

int fhip_q8_attention_workspace_bytes(const fhip_q8_attn_args *args, int32_t compute_units, size_t *bytes) {
    if (!bytes) return invalid("bytes is NULL");
    *bytes = 0;
    int rc = validate_attention(args);
    if (rc || empty(args->q.shape) || args->k.shape[2] == 0) return rc;
    Q8AttnParams p;
    fill_attention(args, compute_units, &p);
    *bytes = attention_plan(p).bytes;
    return FHIP_OK;
}

int fhip_q8_attention(fhip_stream *s, const fhip_q8_attn_args *args) {
    if (!s) return invalid("stream is NULL");
    int rc = validate_attention(args);
    if (rc || empty(args->q.shape)) return rc;
    FHIP_HIP_CHECK(hipSetDevice(s->dev->ordinal));
    if (args->k.shape[2] == 0) {  // no keys at all: zeros, as fhip_flash_attention
        char *out = (char *)args->out.ptr + args->out.offset * (uint64_t)bytes_of(args->out_dtype);
        return launch_fill_zero_rows(out, args->out.stride, args->out.shape, bytes_of(args->out_dtype), s->s);
    }
    Q8AttnParams p;
    fill_attention(args, s->dev->prop.multiProcessorCount, &p);
    const Q8AttnPlan plan = attention_plan(p);
    if (plan.bytes && (!args->workspace || ((uintptr_t)args->workspace & 15) != 0 || args->workspace_bytes < plan.bytes)) {
        set_error("q8_attention: needs %zu bytes of 16-byte aligned workspace, got %zu", plan.bytes, args->workspace ? args->workspace_bytes : 0);
        return FHIP_ERR_WORKSPACE;
    }
    p.nsplit = plan.nsplit;
    p.min_chunk = plan.min_chunk;
    p.partials = (float *)args->workspace;
    return plan.prefill ? launch_q8_prefill(p, plan, s->s) : launch_q8_decode(p, plan, s->s);
}

}  // extern "C"

// ---- the growable cache -----------------------------------------------------------------------------------------------------------------

struct fhip_q8_cache {
    fhip_device *dev;
    fhip_q8_format format;
    uint32_t T;
    uint64_t max_len;
    uint32_t B, Hkv, D;           // fixed by the first append
    uint64_t current, allocated;  // as the wide cache reports them
    bool sliding;
    uint64_t start;               // first valid row while sliding
    uint64_t rows;                // rows that `buf` has room for, whole blocks
    void *buf, *spare;            // keys' codes, values' codes, keys' scales, values' scales; what the last reset left
    size_t bytes, spare_bytes;
};

static size_t q8_codes_bytes(const fhip_q8_cache *c, uint64_t rows) { return (size_t)c->B * c->Hkv * rows * pitch_of(c->D); }
static size_t q8_scales_bytes(const fhip_q8_cache *c, uint64_t rows) { return ((size_t)c->B * c->Hkv * (rows / c->T) * 4 + 15) & ~(size_t)15; }
static size_t q8_cache_bytes(const fhip_q8_cache *c, uint64_t rows) { return 2 * (q8_codes_bytes(c, rows) + q8_scales_bytes(c, rows)); }

// rows [at, at + len) of a buffer with room for `rows`
static fhip_q8_tensor q8_cache_view(const fhip_q8_cache *c, void *buf, uint64_t rows, int side, uint64_t at, uint64_t len) {
    fhip_q8_tensor t;
    memset(&t, 0, sizeof(t));
    const size_t codes = q8_codes_bytes(c, rows), scales = q8_scales_bytes(c, rows);
    t.codes = (char *)buf + side * codes;
    t.scales = (char *)buf + 2 * codes + side * scales;
    t.offset = at * pitch_of(c->D);
    t.scale_offset = at / c->T;
    t.shape[0] = c->B, t.shape[1] = c->Hkv, t.shape[2] = (uint32_t)len, t.shape[3] = c->D;
    t.stride[2] = pitch_of(c->D);
    t.stride[1] = (int64_t)rows * t.stride[2];
    t.stride[0] = (int64_t)c->Hkv * t.stride[1];
    t.scale_stride[1] = (int64_t)(rows / c->T);
    t.scale_stride[0] = (int64_t)c->Hkv * t.scale_stride[1];
    t.block_tokens = c->T;
    t.first = (uint32_t)(at % c->T);
    t.format = c->format;
    return t;
}

// whole blocks from row `from` (a multiple of T) of one buffer to row 0 of another (or the same, further on), `count` rows
static int q8_move_rows(const fhip_q8_cache *c, hipStream_t st, void *src, uint64_t src_rows, uint64_t from, void *dst, uint64_t dst_rows,
                        uint64_t count) {
    const uint64_t blocks = (count + c->T - 1) / c->T;
    for (int side = 0; side < 2; side++) {
        const fhip_q8_tensor x = q8_cache_view(c, src, src_rows, side, from, count), y = q8_cache_view(c, dst, dst_rows, side, 0, count);
        const int64_t xs[4] = {x.stride[0] / 4, x.stride[1] / 4, x.stride[2] / 4, 1}, ys[4] = {y.stride[0] / 4, y.stride[1] / 4, y.stride[2] / 4, 1};
        const uint32_t shape[4] = {c->B, c->Hkv, (uint32_t)count, pitch_of(c->D) / 4};
        int rc = launch_copy_rows((char *)x.codes + x.offset, xs, y.codes, ys, shape, 4, st);
        if (rc) return rc;
        const int64_t xb[4] = {x.scale_stride[0], x.scale_stride[1], 1, 1}, yb[4] = {y.scale_stride[0], y.scale_stride[1], 1, 1};
        const uint32_t sshape[4] = {c->B, c->Hkv, 1, (uint32_t)blocks};
        rc = launch_copy_rows((float *)x.scales + x.scale_offset, xb, y.scales, yb, sshape, 4, st);
        if (rc) return rc;
    }
    return FHIP_OK;
}

static int q8_release(fhip_q8_cache *c, bool keep) {
    int rc = hipSetDevice(c->dev->ordinal) == hipSuccess ? FHIP_OK : FHIP_ERR_HIP;
    if (keep && c->buf && c->bytes > c->spare_bytes) {
        std::swap(c->buf, c->spare);
        std::swap(c->bytes, c->spare_bytes);
    }
    if (c->buf && hipFree(c->buf) != hipSuccess) rc = FHIP_ERR_HIP;
    c->buf = nullptr, c->bytes = 0;
    if (!keep) {
        if (c->spare && hipFree(c->spare) != hipSuccess) rc = FHIP_ERR_HIP;
        c->spare = nullptr, c->spare_bytes = 0;
    }
    c->current = c->allocated = c->rows = c->start = 0;
    c->sliding = false;
    c->B = c->Hkv = c->D = 0;
    if (rc) set_error("q8_cache: hipFree failed");
    return rc;
}

extern "C" {

int fhip_q8_cache_create(fhip_device *dev, fhip_q8_format format, uint32_t block_tokens, uint64_t max_sequence_len, fhip_q8_cache **out) {
    if (!dev || !out) return invalid("q8_cache_create: NULL argument");
    *out = nullptr;
    int rc = check_format(format, block_tokens);
    if (rc) return rc;
    // (the window slides through whole blocks of twice as many rows and two blocks, numbered in 31 bits)
    if (max_sequence_len == 0 || max_sequence_len > (1ull << 30) - 2 * Q8_MAX_BLOCK)
        return invalid("q8_cache_create: max_sequence_len must be in 1..2^30-128");
    fhip_q8_cache *c = new (std::nothrow) fhip_q8_cache();
    if (!c) {
        set_error("out of host memory");
        return FHIP_ERR_HIP;
    }
    c->dev = dev, c->format = format, c->T = block_tokens, c->max_len = max_sequence_len;
    *out = c;
    return FHIP_OK;
}

int fhip_q8_cache_destroy(fhip_q8_cache *c) {
    if (!c) return FHIP_OK;
    const int rc = q8_release(c, false);
    delete c;
    return rc;
}

int fhip_q8_cache_reset(fhip_q8_cache *c) { return c ? q8_release(c, true) : invalid("cache is NULL"); }

int fhip_q8_cache_current_seq_len(const fhip_q8_cache *c, uint64_t *len) {
    if (!c || !len) return invalid("cache/len is NULL");
    *len = c->current;
    return FHIP_OK;
}
int fhip_q8_cache_allocated_seq_len(const fhip_q8_cache *c, uint64_t *len) {
    if (!c || !len) return invalid("cache/len is NULL");
    *len = c->allocated;
    return FHIP_OK;
}

int fhip_q8_cache_append(fhip_q8_cache *c, fhip_stream *s, const fhip_q8_append_args *args, fhip_q8_tensor *k_all, fhip_q8_tensor *v_all) {
    if (!c || !s || !args || !k_all || !v_all) return invalid("q8_cache_append: NULL argument");
    if (args->lens || args->counts) return invalid("q8_cache_append: lens and counts are for fhip_q8_append (one length holds for the whole batch here)");
    AppendShape sh;
    int rc = check_new_rows(args, &sh);
    if (rc) return rc;
    const bool first = c->buf == nullptr;
    if (!first && (sh.B != c->B || sh.Hkv != c->Hkv || sh.D != c->D)) {
        set_error("q8_cache_append: [%u, %u, _, %u] does not match the cached [%u, %u, _, %u]", sh.B, sh.Hkv, sh.D, c->B, c->Hkv, c->D);
        return FHIP_ERR_INVALID_ARG;
    }
    FHIP_HIP_CHECK(hipSetDevice(c->dev->ordinal));
    if (first) c->B = sh.B, c->Hkv = sh.Hkv, c->D = sh.D;
    const uint64_t required = c->current + sh.n, T = c->T;
    auto whole = [&](uint64_t rows) { return (rows + T - 1) / T * T; };

    // where the rows will be: room, the rows kept of the old ones, where the first of them moves, and the new ones that stay
    uint64_t alloc = c->allocated, rows = c->rows, keep = c->current, from = c->start, start = c->start;
    uint32_t skip = 0;
    bool move = false, fresh = false;
    bool sliding = c->sliding;
    if (required > c->max_len) {
        const uint64_t mx = c->max_len, dropped = required - mx;
        keep = c->current > dropped ? c->current - dropped : 0;
        skip = (uint32_t)(sh.n - (mx - keep));
        from = c->start + (c->current - keep);
        // room for the window to slide; moved back, it starts at its own place in a block, and whole blocks are moved: two
        // blocks more keep their old and new places apart
        rows = whole(2 * mx) + 2 * T;
        fresh = !c->sliding;
        move = fresh || c->start + c->current + sh.n > rows || keep == 0;
        start = move ? (keep ? from % T : 0) : from;
        alloc = mx;
        sliding = true;
    } else if (first || required > c->allocated) {
        uint64_t pow2 = 1;
        while (pow2 < required) pow2 <<= 1;
        alloc = first ? required : pow2;
        rows = whole(alloc);
        fresh = move = rows != c->rows;
    }
    void *buf = c->buf;
    size_t bytes = c->bytes;
    if (fresh) {
        const size_t need = q8_cache_bytes(c, rows);
        if (c->spare && c->spare_bytes >= need) {  // what the last reset left
            buf = c->spare, bytes = c->spare_bytes;
            c->spare = nullptr, c->spare_bytes = 0;
        } else {
            const hipError_t e = hipMalloc(&buf, need);
            if (e != hipSuccess) {
                if (first) c->B = c->Hkv = c->D = 0;
                return hip_fail(e, "hipMalloc (8-bit KV cache buffers)");
            }
            bytes = need;
        }
        // the bytes between head_dim and the end of a row's last piece are zero
        if (c->D % 16 != 0) rc = launch_fill_bytes(buf, 0, 2 * q8_codes_bytes(c, rows), s->s);
    }
    if (!rc && move && keep) rc = q8_move_rows(c, s->s, c->buf, c->rows, from - start % T, buf, rows, start % T + keep);
    if (!rc) {
        const fhip_q8_tensor k = q8_cache_view(c, buf, rows, 0, 0, rows), v = q8_cache_view(c, buf, rows, 1, 0, rows);
        rc = append_rows(s->s, args, sh, k, v, start + keep, skip);
    }
    if (rc) {
        if (fresh) {
            (void)hipStreamSynchronize(s->s);  // nothing queued may still write into the buffer being dropped
            (void)hipFree(buf);
        }
        if (first) c->B = c->Hkv = c->D = 0;
        return rc;
    }
    if (fresh && c->buf) (void)hipFree(c->buf);  // waits for the copies out of it
    c->buf = buf, c->bytes = bytes, c->rows = rows;
    c->allocated = alloc, c->sliding = sliding, c->start = start;
    c->current = sliding ? c->max_len : required;
    *k_all = q8_cache_view(c, buf, rows, 0, c->start, c->current);
    *v_all = q8_cache_view(c, buf, rows, 1, c->start, c->current);
    return FHIP_OK;
}

}  // extern "C"
