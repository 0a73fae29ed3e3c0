// The paged key-value cache: its memory, the pages of a step (jl_kv_plan), and what is written to and read from
// pages (jl_kv_append, jl_kv_read).  The attention over it is in jl_attention.hip.
#include <climits>
#include <new>

#include "jl_kv.h"

namespace {

// ---- jl_kv_plan ----------------------------------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxRequests = 8192, kPlanMaxRows = 1 << 17;

struct PlanArgs {
    const int32_t *past, *fresh, *free_in;
    int32_t *ring, *free_out, *table, *lengths, *row_starts, *slots, *positions, *row_requests;
    int requests, pages, page_shift, table_stride, max_rows;
};

// Inclusive sums over the workgroup's threads of three values at once; `sums` [3][waves] in LDS.
__device__ __forceinline__ void scan3(int (&v)[3], int (&total)[3], int (*sums)[kPlanThreads / JL_WAVE]) {
    const int lane = threadIdx.x & (JL_WAVE - 1), wave = threadIdx.x / JL_WAVE;
#pragma unroll
    for (int off = 1; off < JL_WAVE; off <<= 1) {
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const int other = __shfl_up(v[i], off, JL_WAVE);
            if (lane >= off) v[i] += other;
        }
    }
    if (lane == JL_WAVE - 1)
        for (int i = 0; i < 3; i++) sums[i][wave] = v[i];
    __syncthreads();
    for (int i = 0; i < 3; i++) {
        int before = 0;
        total[i] = 0;
        for (int w = 0; w < kPlanThreads / JL_WAVE; w++) {
            if (w < wave) before += sums[i][w];
            total[i] += sums[i][w];
        }
        v[i] += before;
    }
    __syncthreads();
}

// One workgroup, a thread a request: sums over the requests (rows, pages taken, pages returned) give each its place.
__global__ void __launch_bounds__(kPlanThreads) jl_kv_plan_kernel(PlanArgs p) {
    __shared__ int sums[3][kPlanThreads / JL_WAVE];
    const int tid = threadIdx.x, page = 1 << p.page_shift;
    int head = p.free_in[0], count = p.free_in[1];
    if (head < 0 || head >= p.pages || count < 0 || count > p.pages) head = count = 0;
    const int64_t table_tokens = min((int64_t)p.table_stride << p.page_shift, (int64_t)INT_MAX);   // positions are int32
    int carry[3] = {0, 0, 0}, granted_pages = 0;
    for (int base = 0; base < p.requests; base += kPlanThreads) {
        const int r = base + tid;
        const bool real = r < p.requests;
        const int past = real ? p.past[r] : 0, fresh = real ? p.fresh[r] : 0;
        const int wanted = min(max(fresh, 0), p.max_rows + 1);
        const bool held = past >= 0 && past <= table_tokens;
        const int had = held ? (int)(((int64_t)past + page - 1) >> p.page_shift) : 0;
        // rows first: whether a request's rows fit decides whether it asks for pages
        int v[3] = {wanted, 0, 0}, total[3];
        scan3(v, total, sums);
        const int row_end = carry[0] + v[0];
        const bool fits = held && wanted == max(fresh, 0) && row_end <= p.max_rows && (int64_t)past + wanted <= table_tokens;
        const int need = fits ? (int)(((int64_t)past + wanted + page - 1) >> p.page_shift) - had : 0;
        const int back = fresh < 0 ? had : 0;
        v[0] = 0, v[1] = need, v[2] = back;
        const int rows_here = total[0];
        scan3(v, total, sums);
        const int need_end = carry[1] + v[1];
        const bool granted = fits && wanted > 0 && (need == 0 || need_end <= count);
        if (real) {
            p.lengths[r] = fresh < 0 ? 0 : granted ? past + wanted : past;
            p.row_starts[r + 1] = min(row_end, p.max_rows);
            if (r == 0) p.row_starts[0] = 0;
            for (int i = 0; i < wanted; i++) {
                const int row = row_end - wanted + i;
                if (row < p.max_rows) {
                    p.row_requests[row] = r;
                    p.positions[row] = granted ? past + i : -1;
                    int slot = -1;
                    if (granted) {
                        const int b = (past + i) >> p.page_shift;
                        const int at = b < had ? p.table[(int64_t)r * p.table_stride + b]
                                               : p.ring[(int)(((int64_t)head + need_end - need + b - had) % p.pages)];
                        if (at >= 0 && at < p.pages) slot = (at << p.page_shift) + ((past + i) & (page - 1));
                    }
                    p.slots[row] = slot;
                }
            }
            if (granted)
                for (int i = 0; i < need; i++)
                    p.table[(int64_t)r * p.table_stride + had + i] = p.ring[(int)(((int64_t)head + need_end - need + i) % p.pages)];
            if (back) {
                for (int i = 0; i < back; i++) {
                    const int64_t behind = (int64_t)carry[2] + v[2] - back + i;
                    if (behind < p.pages - count)
                        p.ring[(int)((head + count + behind) % p.pages)] = p.table[(int64_t)r * p.table_stride + i];
                }
            }
        }
        int g[3] = {granted ? need : 0, 0, 0}, gt[3];
        scan3(g, gt, sums);
        granted_pages += gt[0];
        carry[0] += rows_here;
        carry[1] += total[1];
        carry[2] += total[2];
    }
    for (int row = carry[0] + tid; row < p.max_rows; row += kPlanThreads) p.slots[row] = p.positions[row] = p.row_requests[row] = -1;
    if (tid == 0) {
        if (p.requests == 0) p.row_starts[0] = 0;
        const int returned = min(carry[2], p.pages - count);
        p.free_out[0] = (int)(((int64_t)head + granted_pages) % p.pages);
        p.free_out[1] = count - granted_pages + returned;
    }
}

// ---- jl_kv_append --------------------------------------------------------------------------------

constexpr int kAppendThreads = 256;

struct AppendArgs {
    JlKvView cache;
    const float *q, *k, *v;
    float *q_out;
    int64_t ldq, ldk, ldv, ldq_out;
    const int32_t *positions, *slots;
    const double *frequencies;
    const float *q_norm, *k_norm;
    float eps;
    int heads, head_dim, rotated;   // heads: 0 without q
    bool halves;
};

// LANES consecutive lanes have a head, eight values each (those past head_dim / 8 idle); a wave has 64 / LANES heads at
// a time, a workgroup the q, k and v heads [blockIdx.y * 256 / LANES, ...) of a token.
template <bool Q8, int LANES>
__global__ void __launch_bounds__(kAppendThreads) jl_kv_append_kernel(AppendArgs p) {
    __shared__ float2 turn[128];    // (cos, sin) of the token's pairs
    const int row = blockIdx.x, tid = threadIdx.x;
    const int position = p.positions[row];
    if (position < 0) return;
    for (int i = tid; i < p.rotated / 2; i += kAppendThreads) {
        // whole turns are dropped in double precision; what is left needs 24 bits
        const double turns = (double)position * p.frequencies[i] * 0.15915494309189533577;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();
    const int unit = blockIdx.y * (kAppendThreads / LANES) + tid / LANES, chunk = tid % LANES;
    const int kv_heads = p.cache.kv_heads;
    if (unit >= p.heads + 2 * kv_heads) return;
    const bool live = chunk < p.head_dim / 8;
    const bool is_q = unit < p.heads, is_v = unit >= p.heads + kv_heads;
    const float *x = is_q ? p.q + row * p.ldq + unit * p.head_dim
                   : is_v ? p.v + row * p.ldv + (unit - p.heads - kv_heads) * p.head_dim
                          : p.k + row * p.ldk + (unit - p.heads) * p.head_dim;
    const float *norm = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
    const int rotated = is_v ? 0 : p.rotated;
    float a[8], b[8];               // the lane's values, and those they turn with (halves)
    // where the partners of this lane's values lie: half the turned part on, or back
    const int half_chunks = rotated / 16;
    const int partner = !p.halves || 8 * chunk >= rotated ? chunk : chunk < half_chunks ? chunk + half_chunks : chunk - half_chunks;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = live ? x[8 * chunk + i] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) b[i] = live ? x[8 * partner + i] : 0.f;
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(a[i], a[i], ss);
        ss = jl_group_sum<LANES>(ss);
        const float root = sqrtf(ss / (float)p.head_dim + p.eps);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            a[i] = live ? a[i] / root * norm[8 * chunk + i] : 0.f;
            b[i] = live ? b[i] / root * norm[8 * partner + i] : 0.f;
        }
    }
    if (live && 8 * chunk < rotated) {
        if (p.halves) {
            const bool first = chunk < half_chunks;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 t = turn[8 * (first ? chunk : partner) + i];
                a[i] = first ? a[i] * t.x - b[i] * t.y : b[i] * t.y + a[i] * t.x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 t = turn[4 * chunk + i / 2];
                const float even = a[i], odd = a[i + 1];
                a[i] = even * t.x - odd * t.y;
                a[i + 1] = even * t.y + odd * t.x;
            }
        }
    }
    if (is_q) {
        float *out = p.q_out + row * p.ldq_out + unit * p.head_dim + 8 * chunk;
        if (live) {
            *(float4 *)out = make_float4(a[0], a[1], a[2], a[3]);
            *(float4 *)(out + 4) = make_float4(a[4], a[5], a[6], a[7]);
        }
        return;
    }
    const int slot = p.slots[row];
    if (slot < 0 || (slot >> p.cache.page_shift) >= p.cache.pages) return;
    const int page = slot >> p.cache.page_shift, token = slot & ((1 << p.cache.page_shift) - 1);
    uint8_t *part = p.cache.k + (is_v ? p.cache.v_offset : 0) +
                    ((int64_t)page * kv_heads + (is_v ? unit - p.heads - kv_heads : unit - p.heads)) * p.cache.part_bytes;
    if constexpr (!Q8) {
        jl_half8 h;
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = (_Float16)a[i];
        if (live) *(jl_half8 *)(part + (token * p.head_dim + 8 * chunk) * 2) = h;
    } else {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(a[i]));
        most = fmaxf(most, __shfl_xor(most, 1, JL_WAVE));   // a block is four lanes' values
        most = fmaxf(most, __shfl_xor(most, 2, JL_WAVE));
        const _Float16 d16 = (_Float16)fminf(most / 127.f, 65504.f);
        const float d = (float)d16;
        uint32_t word[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // (NaN: both comparisons fall to the other operand's side, so it is taken out first)
            const float y = d > 0.f && a[i] == a[i] ? fminf(fmaxf(rintf(a[i] / d), -127.f), 127.f) : 0.f;
            word[i / 4] |= (uint32_t)((int)y & 255) << (8 * (i % 4));
        }
        if (live) {
            *(uint2 *)(part + token * p.head_dim + 8 * chunk) = make_uint2(word[0], word[1]);
            if (chunk % 4 == 0) {
                _Float16 *scales = (_Float16 *)(part + ((int64_t)p.head_dim << p.cache.page_shift));
                scales[((chunk / 4) << p.cache.page_shift) + token] = d16;
            }
        }
    }
}

// ---- jl_kv_read ----------------------------------------------------------------------------------

template <bool Q8, bool HALF>
__global__ void __launch_bounds__(256) jl_kv_read_kernel(JlKvView cache, int head_dim, const int32_t *slots, int64_t rows,
                                                         void *k_out, void *v_out) {
    const int per_head = head_dim / 8, per_row = cache.kv_heads * per_head;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= rows * per_row) return;
    const int64_t row = at / per_row;
    const int head = (int)(at % per_row) / per_head, chunk = (int)(at % per_row) % per_head;
    const int slot = slots[row], page = slot >> cache.page_shift, token = slot & ((1 << cache.page_shift) - 1);
    const uint8_t *part = cache.k + ((int64_t)page * cache.kv_heads + head) * cache.part_bytes;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        void *out = which ? v_out : k_out;
        if (!out) continue;
        jl_half8 h = {0, 0, 0, 0, 0, 0, 0, 0};
        if (slot >= 0 && page < cache.pages) h = jl_kv_load8<Q8>(part + (which ? cache.v_offset : 0), cache.page_shift, head_dim, token, chunk);
        if constexpr (HALF) {
            ((jl_half8 *)out)[at] = h;
        } else {
            ((float4 *)out)[2 * at] = make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
            ((float4 *)out)[2 * at + 1] = make_float4((float)h[4], (float)h[5], (float)h[6], (float)h[7]);
        }
    }
}

int cache_check(const char *who, int kv_type, int64_t pages, int kv_heads, int head_dim, int page_tokens) {
    if (kv_type != JL_KV_F16 && kv_type != JL_KV_Q8_0)
        return jl_fail(JL_ERR_UNSUPPORTED, "%s: no key-value cache of type %d (JL_KV_F16 or JL_KV_Q8_0)", who, kv_type);
    if (head_dim != 64 && head_dim != 96 && head_dim != 128 && head_dim != 192 && head_dim != 256)
        return jl_fail(JL_ERR_UNSUPPORTED, "%s: no kernel for heads of %d values (64, 96, 128, 192 or 256)", who, head_dim);
    JL_REQUIRE(page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || page_tokens == 128 || page_tokens == 256,
               "%s: pages of %d tokens (16, 32, 64, 128 or 256)", who, page_tokens);
    JL_REQUIRE(kv_heads > 0 && kv_heads <= 1024, "%s: %d heads of k and v (1 ... 1024)", who, kv_heads);
    JL_REQUIRE(pages > 0 && pages <= INT32_MAX / page_tokens, "%s: %lld pages of %d tokens (at most 2^31 - 1 tokens)", who,
               (long long)pages, page_tokens);
    return JL_OK;
}

int cache_make(const char *who, jl_context *ctx, void *memory, int kv_type, int64_t pages, int kv_heads, int head_dim,
               int page_tokens, jl_kv_cache **out) {
    JL_REQUIRE(ctx && out, "%s: null argument", who);
    *out = nullptr;
    const int st = cache_check(who, kv_type, pages, kv_heads, head_dim, page_tokens);
    if (st != JL_OK) return st;
    const size_t bytes = jl_kv_cache_bytes(kv_type, pages, kv_heads, head_dim, page_tokens);
    const bool owns = memory == nullptr;
    if (owns) {
        const int got = jl_malloc(ctx, bytes, &memory);
        if (got != JL_OK) return got;
    }
    jl_kv_cache *c = new (std::nothrow) jl_kv_cache{ctx, kv_type, pages, kv_heads, head_dim, page_tokens, bytes, (uint8_t *)memory, owns};
    if (!c) {
        if (owns) (void)jl_free(ctx, memory);
        return jl_fail(JL_ERR_INVALID, "%s: host allocation failed", who);
    }
    *out = c;
    return JL_OK;
}

template <bool Q8>
void launch_append(const AppendArgs &a, unsigned rows, hipStream_t stream) {
    const int lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32;
    const int units = a.heads + 2 * a.cache.kv_heads, per = kAppendThreads / lanes;
    const dim3 grid(rows, (unsigned)((units + per - 1) / per)), block(kAppendThreads);
    if (lanes == 8) hipLaunchKernelGGL((jl_kv_append_kernel<Q8, 8>), grid, block, 0, stream, a);
    else if (lanes == 16) hipLaunchKernelGGL((jl_kv_append_kernel<Q8, 16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((jl_kv_append_kernel<Q8, 32>), grid, block, 0, stream, a);
}

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

extern "C" {

size_t jl_kv_cache_bytes(int kv_type, int64_t pages, int kv_heads, int head_dim, int page_tokens) {
    if (cache_check("jl_kv_cache_bytes", kv_type, pages, kv_heads, head_dim, page_tokens) != JL_OK) return 0;
    return 2 * (size_t)pages * kv_heads * jl_kv_part_bytes(kv_type, head_dim, page_tokens);
}

int jl_kv_cache_create(jl_context *ctx, int kv_type, int64_t pages, int kv_heads, int head_dim, int page_tokens,
                       jl_kv_cache **out) {
    return cache_make("jl_kv_cache_create", ctx, nullptr, kv_type, pages, kv_heads, head_dim, page_tokens, out);
}

int jl_kv_cache_wrap(jl_context *ctx, void *device_memory, int kv_type, int64_t pages, int kv_heads, int head_dim,
                     int page_tokens, jl_kv_cache **out) {
    if (out) *out = nullptr;
    JL_REQUIRE(device_memory != nullptr, "jl_kv_cache_wrap: null argument");
    JL_REQUIRE(aligned(device_memory, 16), "jl_kv_cache_wrap: the pages must be 16-byte aligned in device memory");
    return cache_make("jl_kv_cache_wrap", ctx, device_memory, kv_type, pages, kv_heads, head_dim, page_tokens, out);
}

int jl_kv_cache_free(jl_kv_cache *cache) {
    if (!cache) return JL_OK;
    const int st = cache->owns_memory ? jl_free(cache->ctx, cache->memory) : JL_OK;
    delete cache;
    return st;
}

void *jl_kv_cache_memory(const jl_kv_cache *cache) { return cache ? cache->memory : nullptr; }

int jl_kv_plan(jl_context *ctx, const int32_t *past, const int32_t *fresh, int64_t requests, int64_t pages,
               int page_tokens, int32_t *page_ring, const int32_t *free_in, int32_t *free_out, int32_t *block_table,
               int64_t table_stride, int32_t *lengths, int32_t *row_starts, int32_t *slots, int32_t *positions,
               int32_t *row_requests, int64_t max_rows) {
    JL_REQUIRE(ctx && past && fresh && page_ring && free_in && free_out && block_table && lengths && row_starts && slots &&
                   positions && row_requests, "jl_kv_plan: null argument");
    JL_REQUIRE(page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || page_tokens == 128 || page_tokens == 256,
               "jl_kv_plan: pages of %d tokens (16, 32, 64, 128 or 256)", page_tokens);
    JL_REQUIRE(pages > 0 && pages <= INT32_MAX / page_tokens, "jl_kv_plan: %lld pages of %d tokens (at most 2^31 - 1 tokens)",
               (long long)pages, page_tokens);
    JL_REQUIRE(requests >= 0 && requests <= kPlanMaxRequests, "jl_kv_plan: %lld requests (at most %d)", (long long)requests,
               kPlanMaxRequests);
    JL_REQUIRE(max_rows >= 0 && max_rows <= kPlanMaxRows, "jl_kv_plan: max_rows %lld (at most %d)", (long long)max_rows, kPlanMaxRows);
    JL_REQUIRE(table_stride > 0 && table_stride <= INT32_MAX / (requests > 0 ? requests : 1),
               "jl_kv_plan: a block table of %lld x %lld entries", (long long)requests, (long long)table_stride);
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    PlanArgs p;
    p.past = past, p.fresh = fresh, p.free_in = free_in;
    p.ring = page_ring, p.free_out = free_out, p.table = block_table, p.lengths = lengths, p.row_starts = row_starts;
    p.slots = slots, p.positions = positions, p.row_requests = row_requests;
    p.requests = (int)requests, p.pages = (int)pages, p.page_shift = __builtin_ctz((unsigned)page_tokens);
    p.table_stride = (int)table_stride, p.max_rows = (int)max_rows;
    hipLaunchKernelGGL(jl_kv_plan_kernel, dim3(1), dim3(kPlanThreads), 0, ctx->stream, p);
    JL_HIP(hipGetLastError());
    return JL_OK;
}

int jl_kv_append(jl_context *ctx, jl_kv_cache *cache, const float *q, int heads, int64_t ldq, const float *k,
                 int64_t ldk, const float *v, int64_t ldv, float *q_out, int64_t ldq_out, const int32_t *positions,
                 const int32_t *slots, int64_t rows, const double *frequencies, int rotated, int rope_style,
                 const float *q_norm, const float *k_norm, float eps) {
    JL_REQUIRE(ctx && cache && k && v && positions && slots && (!q || q_out), "jl_kv_append: null argument");
    const int dim = cache->head_dim;
    JL_REQUIRE(cache->ctx->device == ctx->device, "jl_kv_append: the cache lies on device %d, the context's is %d",
               cache->ctx->device, ctx->device);
    JL_REQUIRE(rows >= 0 && rows <= INT32_MAX, "jl_kv_append: %lld rows", (long long)rows);
    JL_REQUIRE(rotated >= 0 && rotated <= dim && rotated % 16 == 0, "jl_kv_append: %d values turned of heads of %d (a multiple of 16)",
               rotated, dim);
    JL_REQUIRE(rotated == 0 || frequencies, "jl_kv_append: null frequencies for %d turned values", rotated);
    JL_REQUIRE(rope_style == JL_ROPE_PAIRS || rope_style == JL_ROPE_HALVES, "jl_kv_append: rotation style %d", rope_style);
    JL_REQUIRE(!q || (heads > 0 && heads <= 65536), "jl_kv_append: %d query heads", heads);
    const int64_t kv_width = (int64_t)cache->kv_heads * dim, q_width = q ? (int64_t)heads * dim : 0;
    JL_REQUIRE(ldk >= kv_width && ldv >= kv_width && (!q || (ldq >= q_width && ldq_out >= q_width)),
               "jl_kv_append: rows closer together (%lld, %lld, %lld, %lld) than they are long", (long long)ldq, (long long)ldk,
               (long long)ldv, (long long)ldq_out);
    JL_REQUIRE(aligned(k, 16) && aligned(v, 16) && ldk % 4 == 0 && ldv % 4 == 0 &&
                   (!q || (aligned(q, 16) && aligned(q_out, 16) && ldq % 4 == 0 && ldq_out % 4 == 0)),
               "jl_kv_append: q, k, v and q_out must be 16-byte aligned, with row strides that are multiples of 4");
    JL_REQUIRE(q != q_out || !q || ldq == ldq_out, "jl_kv_append: q turned in place with another row stride");
    JL_REQUIRE(aligned(q_norm, 16) && aligned(k_norm, 16) && aligned(frequencies, 8), "jl_kv_append: unaligned norm weights or frequencies");
    if (rows == 0) return JL_OK;
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    AppendArgs a;
    a.cache = jl_kv_view(cache);
    a.q = q, a.k = k, a.v = v, a.q_out = q_out;
    a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldq_out = ldq_out;
    a.positions = positions, a.slots = slots, a.frequencies = frequencies;
    a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.heads = q ? heads : 0, a.head_dim = dim, a.rotated = rotated, a.halves = rope_style == JL_ROPE_HALVES;
    if (cache->type == JL_KV_Q8_0) launch_append<true>(a, (unsigned)rows, ctx->stream);
    else launch_append<false>(a, (unsigned)rows, ctx->stream);
    JL_HIP(hipGetLastError());
    return JL_OK;
}

int jl_kv_read(jl_context *ctx, const jl_kv_cache *cache, const int32_t *slots, int64_t rows, void *k_out,
               void *v_out, int out_f16) {
    JL_REQUIRE(ctx && cache && slots, "jl_kv_read: null argument");
    JL_REQUIRE(cache->ctx->device == ctx->device, "jl_kv_read: the cache lies on device %d, the context's is %d",
               cache->ctx->device, ctx->device);
    JL_REQUIRE(rows >= 0 && rows <= INT32_MAX, "jl_kv_read: %lld rows", (long long)rows);
    JL_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16), "jl_kv_read: k_out and v_out must be 16-byte aligned");
    if (rows == 0 || (!k_out && !v_out)) return JL_OK;
    const int64_t threads = rows * cache->kv_heads * (cache->head_dim / 8);
    JL_REQUIRE(threads <= (int64_t)INT32_MAX * 256, "jl_kv_read: %lld rows", (long long)rows);
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
    const JlKvView c = jl_kv_view(cache);
    const int dim = cache->head_dim;
    if (cache->type == JL_KV_Q8_0) {
        if (out_f16) hipLaunchKernelGGL((jl_kv_read_kernel<true, true>), grid, block, 0, ctx->stream, c, dim, slots, rows, k_out, v_out);
        else hipLaunchKernelGGL((jl_kv_read_kernel<true, false>), grid, block, 0, ctx->stream, c, dim, slots, rows, k_out, v_out);
    } else {
        if (out_f16) hipLaunchKernelGGL((jl_kv_read_kernel<false, true>), grid, block, 0, ctx->stream, c, dim, slots, rows, k_out, v_out);
        else hipLaunchKernelGGL((jl_kv_read_kernel<false, false>), grid, block, 0, ctx->stream, c, dim, slots, rows, k_out, v_out);
    }
    JL_HIP(hipGetLastError());
    return JL_OK;
}

}  // extern "C"
