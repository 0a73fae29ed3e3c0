// jl_kv_attention and jl_kv_attention_scored: what they check, and which kernel takes a call.
#include <algorithm>
#include <climits>
#include <cmath>

#include "jl_attention.h"

namespace {

constexpr size_t kArrivedBytes = kAttentionMostGroups * sizeof(uint32_t);
constexpr size_t kTakenBytes = 32768;             // a byte for each block of rows, two rows at least
// (Row block, head of k and v) pairs to a compute unit from which rows go in blocks: each is a workgroup's, whole, and the other
// kernel cuts what it has among all.  (4-bit cache, 8 query heads over 4 of 128: 700 rows of one request, 88 pairs: 22.7 us in
// blocks, 21.0 without; 1400, 176 pairs: 34.6 and 52.5; 4 requests of 175 ... 700, 220 pairs: 27.1 and 39.9.  32 over 8: 256 rows
// after 4000 tokens, 128 pairs: 83 and 70; 512 after 30 000, 256 pairs, binary16: 570 and 1062.)
constexpr float kPromptShare = 0.625f;

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Everything that a call takes but the scores' shape, which is null for jl_kv_attention.
struct Shaping {
    float cap;
    const float *slopes;
    const int32_t *first_tokens, *end_tokens;
};

int attention(const char *who, jl_context *ctx, const jl_kv_cache *cache, const float *q, int heads, int64_t ldq, int64_t rows,
              const int32_t *positions, const int32_t *row_requests, const int32_t *block_table, int64_t requests,
              int64_t table_stride, float scale, int64_t window, const Shaping *shaping, void *out, int out_f16, int64_t ldo,
              void *workspace, size_t workspace_bytes) {
    JL_REQUIRE(ctx && cache && q && positions && block_table && out && workspace, "%s: null argument", who);
    JL_REQUIRE(cache->ctx->device == ctx->device, "%s: the cache lies on device %d, the context's is %d", who,
               cache->ctx->device, ctx->device);
    const int dim = cache->head_dim;
    JL_REQUIRE(heads > 0 && heads <= 65536 && heads % cache->kv_heads == 0, "%s: %d query heads over %d of k and v", who,
               heads, cache->kv_heads);
    JL_REQUIRE(rows >= 0 && rows <= 65535, "%s: %lld rows (at most 65535)", who, (long long)rows);
    JL_REQUIRE(requests >= 0 && requests <= INT32_MAX && (row_requests || requests >= rows),
               "%s: %lld rows of %lld requests", who, (long long)rows, (long long)requests);
    JL_REQUIRE(table_stride > 0 && table_stride <= INT32_MAX, "%s: block table rows of %lld entries", who, (long long)table_stride);
    // (a row's list of tiles of 32 tokens, times its heads, all rows together: a 32-bit number)
    const int64_t table_tokens = std::min(table_stride * cache->page_tokens, (int64_t)INT_MAX - 64);
    const int64_t lists = rows * cache->kv_heads * ((heads / cache->kv_heads + 15) / 16);
    JL_REQUIRE(lists <= 0 || table_tokens / 32 + 2 + kAttentionStart <= (int64_t)(UINT32_MAX - 2 * kAttentionMostGroups) / lists,
               "%s: %lld rows of %d heads over %lld tokens in one call", who, (long long)rows, heads, (long long)table_tokens);
    const float scale_of_powers = scale * 1.44269504088896340736f;   // weights are powers of two
    JL_REQUIRE(std::isfinite(scale_of_powers), "%s: scale %g", who, (double)scale);
    JL_REQUIRE(window >= 0, "%s: window %lld", who, (long long)window);
    const int64_t width = (int64_t)heads * dim;
    JL_REQUIRE(ldq >= width && ldo >= width, "%s: rows closer together (%lld, %lld) than they are long (%lld)", who,
               (long long)ldq, (long long)ldo, (long long)width);
    JL_REQUIRE(aligned(q, 16) && aligned(out, 16) && aligned(workspace, 16) && ldq % 4 == 0 && ldo % (out_f16 ? 8 : 4) == 0,
               "%s: q, out and the workspace must be 16-byte aligned, ldq a multiple of 4 and ldo of %d", who, out_f16 ? 8 : 4);
    const size_t needed = jl_kv_attention_workspace_bytes(heads, cache->kv_heads, dim);
    if (workspace_bytes < needed)
        return jl_fail(JL_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, needed);
    if (rows == 0) return JL_OK;
    JL_REQUIRE(out != q, "%s: out in place of q", who);
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    JlScoredArgs a;
    a.cache = jl_kv_view(cache);
    a.q = q, a.ldq = ldq, a.ldo = ldo;
    a.positions = positions, a.row_requests = row_requests, a.table = block_table;
    a.requests = (int)requests, a.table_stride = table_stride, a.table_tokens = (int)table_tokens;
    a.scale = scale_of_powers;
    a.window = window > INT32_MAX ? 0 : (int)window;   // one that reaches behind every position
    a.group = heads / cache->kv_heads;
    a.blocks_of_16 = (a.group + 15) / 16;
    // Twice as many rows as requests, or more: some are of one, unless they are padding.  (32 heads over 8 of 128, one request,
    // each row alone and together: a prompt of 2048 tokens 753 and 187 us, of 512 64 and 27; 4 rows after 30 000 tokens 79 and
    // 44, after 1000 11.8 and 14.0.  32 heads over 32, 512 tokens: 224 and 32.  64 rows of 64 requests of up to 8192 tokens
    // padded to 512 rows: 118 and 124; to 72, which are too few: 105 and 118.)
    a.rows_each = 1;
    if (row_requests && rows >= 2 * requests)
        while (2 * a.rows_each * a.group <= 16) a.rows_each *= 2;
    a.rows = (int)rows;
    a.out = out, a.out_f16 = out_f16 != 0;
    a.arrived = (uint32_t *)workspace;
    a.parts = (float *)((uint8_t *)workspace + kArrivedBytes);
    // Blocks of rows, where they are many: 64 columns to a workgroup, a (row, query head) each.
    a.taken_rows = 64 / a.group & -a.rows_each, a.taken = nullptr, a.taken_out = nullptr;
    const bool prompts = row_requests && rows >= 2 * requests && (shaping || cache->type == JL_KV_Q4_0) && a.taken_rows > 1 &&
                         rows / a.taken_rows * cache->kv_heads >= ctx->compute_units * kPromptShare;
    if (prompts) a.taken_out = (uint8_t *)workspace + needed - kTakenBytes;
    const Shaping nothing{0.f, nullptr, nullptr, nullptr};
    if (prompts && !shaping) shaping = &nothing;
    JlAttentionArgs &plain = a;
    if (shaping) {
        a.cap = shaping->cap * 1.44269504088896340736f, a.one_over_cap = shaping->cap > 0.f ? 1.f / a.cap : 0.f;
        a.slopes = shaping->slopes, a.first_tokens = shaping->first_tokens, a.end_tokens = shaping->end_tokens;
        if (prompts) {
            JL_HIP((cache->type == JL_KV_Q8_0   ? jl_launch_attention_prompt_q8
                    : cache->type == JL_KV_Q4_0 ? jl_launch_attention_prompt_q4
                                                : jl_launch_attention_prompt_f16)(a, dim, ctx->compute_units, ctx->device, ctx->stream));
            a.taken = a.taken_out;
        }
        JL_HIP((cache->type == JL_KV_Q8_0   ? jl_launch_attention_scored_q8
                : cache->type == JL_KV_Q4_0 ? jl_launch_attention_scored_q4
                                            : jl_launch_attention_scored_f16)(a, dim, ctx->compute_units, ctx->stream));
    } else {
        JL_HIP((cache->type == JL_KV_Q8_0   ? jl_launch_attention_q8
                : cache->type == JL_KV_Q4_0 ? jl_launch_attention_q4
                                            : jl_launch_attention_f16)(plain, dim, ctx->compute_units, ctx->stream));
    }
    return JL_OK;
}

}  // namespace

extern "C" {

size_t jl_kv_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
    return kArrivedBytes + (size_t)2 * kAttentionMostGroups * 16 * ((size_t)head_dim + 2) * sizeof(float) + kTakenBytes;
}

int jl_kv_attention_workspace_init(jl_context *ctx, void *workspace, size_t workspace_bytes) {
    JL_REQUIRE(ctx && workspace, "jl_kv_attention_workspace_init: null argument");
    JL_REQUIRE(aligned(workspace, 16), "jl_kv_attention_workspace_init: the workspace must be 16-byte aligned");
    if (workspace_bytes < kArrivedBytes)
        return jl_fail(JL_ERR_WORKSPACE, "jl_kv_attention_workspace_init: workspace of %zu bytes", workspace_bytes);
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    return jl_launch_fill(ctx, (float *)workspace, 0.f, kArrivedBytes / sizeof(float));
}

int jl_kv_attention(jl_context *ctx, const jl_kv_cache *cache, const float *q, int heads, int64_t ldq, int64_t rows,
                    const int32_t *positions, const int32_t *row_requests, const int32_t *block_table,
                    int64_t requests, int64_t table_stride, float scale, int64_t window, void *out, int out_f16,
                    int64_t ldo, void *workspace, size_t workspace_bytes) {
    return attention("jl_kv_attention", ctx, cache, q, heads, ldq, rows, positions, row_requests, block_table, requests, table_stride,
                     scale, window, nullptr, out, out_f16, ldo, workspace, workspace_bytes);
}

int jl_kv_attention_scored(jl_context *ctx, const jl_kv_cache *cache, const float *q, int heads, int64_t ldq, int64_t rows,
                           const int32_t *positions, const int32_t *row_requests, const int32_t *block_table,
                           int64_t requests, int64_t table_stride, float scale, int64_t window, float cap,
                           const float *slopes, const int32_t *first_tokens, const int32_t *end_tokens, void *out,
                           int out_f16, int64_t ldo, void *workspace, size_t workspace_bytes) {
    const Shaping shaping{cap, slopes, first_tokens, end_tokens};
    // (its inverse, of powers of two, is finite)
    JL_REQUIRE(cap == 0.f || (cap >= 1e-30f && cap <= 1e30f), "jl_kv_attention_scored: cap %g (0, or 1e-30 ... 1e30)", (double)cap);
    JL_REQUIRE(aligned(slopes, 4) && aligned(first_tokens, 4) && aligned(end_tokens, 4), "jl_kv_attention_scored: unaligned slopes, first_tokens or end_tokens");
    return attention("jl_kv_attention_scored", ctx, cache, q, heads, ldq, rows, positions, row_requests, block_table, requests,
                     table_stride, scale, window, &shaping, out, out_f16, ldo, workspace, workspace_bytes);
}

}  // extern "C"
