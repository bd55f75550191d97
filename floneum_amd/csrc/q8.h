// Internal declarations of the 8-bit key / value cache: what its kernels receive and their launchers.
#pragma once
#include "common.h"

namespace fhip {

constexpr int Q8_MAX_DIM = 256;
constexpr int Q8_MAX_BLOCK = 64;
constexpr int Q8_MAX_SHARES = 512;  // of the keys of a call

// A view of codes and scales: pointers with the offsets applied, strides in bytes / elements.
struct Q8View {
    uint8_t *codes;
    float *scales;
    int64_t cs[3];   // batch, head, row
    int64_t ss[2];   // batch, head
    int64_t rows;
    int32_t log2_block;
    int32_t first;   // place of row 0 in its block
};

// One row-wise job of an append: new keys or values into the cache, or q into q_out.
struct Q8Rows {
    const void *src;
    int64_t s[4];            // of the source, elements
    int32_t src_dtype;
    int32_t vec;             // source (and destination) rows in pieces of four elements
    int32_t heads;
    int32_t n;               // new rows per sequence
    int64_t pos0;            // position of the first of them in the tables (before lens)
    int32_t mode;            // 0 pairs (i, i + D/2), 1 pairs (2i, 2i + 1), 2 no rotation
    const void *norm_w, *norm_b;
    int32_t norm_dtype;
    float eps;
    int32_t is_q;
    int32_t dst_dtype;       // q only
    void *dst;               // q only
    int64_t d[4];            // q only
    Q8View out;              // keys and values; of q only `rows`, which bounds the places of its rows
    uint32_t span;           // row slots per (batch, head): n, or whole blocks for any place of the first row in its own
    uint32_t total;          // slots of the job (both are counted in groups of rows by the launcher of rows on their own)
    uint32_t by_heads[2], by_rows[2];  // factor and shift that divide numbers below 2^31 by heads and span (factor 0: by 1), set by the launcher
};
struct Q8AppendParams {
    Q8Rows job[3];
    uint32_t first_wg[3];    // a job's first workgroup
    int32_t jobs;
    int32_t D, format;
    int64_t row;
    const int32_t *lens, *counts;
    const float *cos, *sin;
    int64_t table_rows;
};
// max_block: the cache's block_tokens; rows_alone: no two new rows share a block, and the jobs' slots are their rows; normed: some job has a norm
int launch_q8_append(Q8AppendParams &p, int max_block, bool rows_alone, bool normed, hipStream_t stream);

struct Q8ReadParams {
    Q8View x;
    void *out;
    int64_t os[4];
    int32_t out_dtype, vec;
    int32_t B, H, n, D, format;
    int64_t row;
    const int32_t *lens;
};
struct Q8ReadDivisors {
    uint32_t pieces[2], rows[2], heads[2];  // as Q8Rows::by_heads
};
int launch_q8_dequantize(const Q8ReadParams &p, hipStream_t stream);

// Attention over the cache.
struct Q8AttnParams {
    const void *q;
    void *out;
    int64_t qs[4], os[4];
    int32_t q_dtype, out_dtype;
    int32_t q_vec, out_vec;  // query / output rows in pieces of four elements
    Q8View k, v;
    int32_t B, H, Hkv, G, Sq, Skv, D, format;
    int32_t causal;
    int64_t q_pos_offset, window;
    const int32_t *kv_lens, *q_positions;
    const void *mask;
    int64_t ms0, ms1;
    int32_t mask_kind;
    float scale;
    // keys in shares: `nsplit` per (batch, kv head, column block), each of at least `min_chunk` keys
    int32_t nsplit, min_chunk;
    float *partials;   // [B * Hkv][nsplit][G * Sq][padded D] means of the shares' values, then as many (m, l): largest score and sum of the weights
    int32_t cus;
};
struct Q8AttnPlan {
    bool prefill;  // the kernel for many rows (attn_q8_prefill.hip), else the one for few (attn_q8_decode.hip)
    int waves;     // per workgroup of the former
    int nsplit, min_chunk;
    size_t bytes;  // of workspace
};
Q8AttnPlan q8_decode_plan(const Q8AttnParams &p);
int launch_q8_decode(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream);
Q8AttnPlan q8_prefill_plan(const Q8AttnParams &p);
int launch_q8_prefill(const Q8AttnParams &p, const Q8AttnPlan &plan, hipStream_t stream);
int launch_q8_merge(const Q8AttnParams &p, hipStream_t stream);  // joins the shares in p.partials

}  // namespace fhip
