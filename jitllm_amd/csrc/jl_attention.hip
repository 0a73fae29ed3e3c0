// jl_kv_attention: attention of one new token a row over its request's pages.
#include <climits>
#include <cmath>

#include "jl_kv.h"

namespace {

constexpr int kThreads = 256;

struct AttentionArgs {
    JlKvView cache;
    const float *q;
    int64_t ldq, ldo;
    const int32_t *positions, *row_requests, *table;
    int64_t requests, table_stride;
    float scale;          // times log2(e): weights are powers of two
    int window;           // 0: none
    int group;            // query heads to a head of k and v
    void *out;
    bool out_f16;
};

// A workgroup has a row and a query head: 256 tokens at a time, their scores by a thread each, then the weighted sum of
// their values by a thread per element, with the running maximum and sum of the softmax.
template <bool Q8, int DIM>
__global__ void __launch_bounds__(kThreads) jl_kv_attention_kernel(AttentionArgs p) {
    __shared__ float q[DIM], weight[kThreads];
    __shared__ float fold[kThreads / JL_WAVE];
    const int head = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const int kv_head = head / p.group;
    if (tid < DIM) q[tid] = p.q[row * p.ldq + head * DIM + tid] * p.scale;
    const int request = p.row_requests ? p.row_requests[row] : row;
    const int position = p.positions[row];
    const int64_t held = min((int64_t)p.table_stride << p.cache.page_shift, (int64_t)INT_MAX);
    const bool real = request >= 0 && request < p.requests && position >= 0;
    const int end = real ? (int)min((int64_t)position + 1, held) : 0;
    const int first = p.window > 0 ? max(position - p.window + 1, 0) : 0;
    const int32_t *table = p.table + (real ? request * p.table_stride : 0);
    float most = -INFINITY, total = 0.f, sum = 0.f;
    for (int base = first; base < end; base += kThreads) {
        const int token = base + tid;
        float score = -INFINITY;
        const int page = token < end ? table[token >> p.cache.page_shift] : -1;
        const uint8_t *part = p.cache.k + ((int64_t)page * p.cache.kv_heads + kv_head) * p.cache.part_bytes;
        const int in_page = token & ((1 << p.cache.page_shift) - 1);
        __syncthreads();
        if (page >= 0 && page < p.cache.pages) {
            score = 0.f;
            for (int c = 0; c < DIM / 8; c++) {
                const jl_half8 k = jl_kv_load8<Q8>(part, p.cache.page_shift, DIM, in_page, c);
#pragma unroll
                for (int i = 0; i < 8; i++) score = fmaf((float)k[i], q[8 * c + i], score);
            }
        }
        float m = score;
        for (int off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, JL_WAVE));
        if (tid % JL_WAVE == 0) fold[tid / JL_WAVE] = m;
        __syncthreads();
        m = fmaxf(most, fmaxf(fmaxf(fold[0], fold[1]), fmaxf(fold[2], fold[3])));
        const float from = m == -INFINITY ? 0.f : m;
        weight[tid] = score == -INFINITY ? 0.f : exp2f(score - from);
        const float keep = exp2f(most - from);
        most = m;
        total *= keep;
        sum *= keep;
        __syncthreads();
        for (int t = 0; t < kThreads && base + t < end; t++) {
            total += weight[t];
            if (tid < DIM) {
                const int other = table[(base + t) >> p.cache.page_shift];
                if (other < 0 || other >= p.cache.pages) continue;
                const uint8_t *v = p.cache.k + p.cache.v_offset + ((int64_t)other * p.cache.kv_heads + kv_head) * p.cache.part_bytes;
                const jl_half8 h = jl_kv_load8<Q8>(v, p.cache.page_shift, DIM, (base + t) & ((1 << p.cache.page_shift) - 1), tid / 8);
                sum = fmaf(weight[t], (float)h[tid % 8], sum);
            }
        }
    }
    if (tid < DIM) {
        const float r = total > 0.f || total != total ? sum / total : 0.f;
        if (p.out_f16) ((_Float16 *)p.out)[row * p.ldo + head * DIM + tid] = (_Float16)r;
        else ((float *)p.out)[row * p.ldo + head * DIM + tid] = r;
    }
}

template <bool Q8>
void launch(const AttentionArgs &a, int heads, int rows, int head_dim, hipStream_t stream) {
    const dim3 grid((unsigned)heads, (unsigned)rows), block(kThreads);
    switch (head_dim) {
        case 64: hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, 64>), grid, block, 0, stream, a); break;
        case 96: hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, 96>), grid, block, 0, stream, a); break;
        case 128: hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, 128>), grid, block, 0, stream, a); break;
        case 192: hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, 192>), grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, 256>), grid, block, 0, stream, a); break;
    }
}

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

extern "C" {

size_t jl_kv_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
    return 256;
}

int jl_kv_attention(jl_context *ctx, const jl_kv_cache *cache, const float *q, int heads, int64_t ldq, int64_t rows,
                    const int32_t *positions, const int32_t *row_requests, const int32_t *block_table,
                    int64_t requests, int64_t table_stride, float scale, int64_t window, void *out, int out_f16,
                    int64_t ldo, void *workspace, size_t workspace_bytes) {
    JL_REQUIRE(ctx && cache && q && positions && block_table && out && workspace, "jl_kv_attention: null argument");
    JL_REQUIRE(cache->ctx->device == ctx->device, "jl_kv_attention: the cache lies on device %d, the context's is %d",
               cache->ctx->device, ctx->device);
    const int dim = cache->head_dim;
    JL_REQUIRE(heads > 0 && heads <= 65536 && heads % cache->kv_heads == 0, "jl_kv_attention: %d query heads over %d of k and v",
               heads, cache->kv_heads);
    JL_REQUIRE(rows >= 0 && rows <= 65535, "jl_kv_attention: %lld rows (at most 65535)", (long long)rows);
    JL_REQUIRE(requests >= 0 && requests <= INT32_MAX && (row_requests || requests >= rows),
               "jl_kv_attention: %lld rows of %lld requests", (long long)rows, (long long)requests);
    JL_REQUIRE(table_stride > 0 && table_stride <= INT32_MAX, "jl_kv_attention: block table rows of %lld entries", (long long)table_stride);
    JL_REQUIRE(std::isfinite(scale), "jl_kv_attention: scale %g", (double)scale);
    JL_REQUIRE(window >= 0, "jl_kv_attention: window %lld", (long long)window);
    const int64_t width = (int64_t)heads * dim;
    JL_REQUIRE(ldq >= width && ldo >= width, "jl_kv_attention: rows closer together (%lld, %lld) than they are long (%lld)",
               (long long)ldq, (long long)ldo, (long long)width);
    JL_REQUIRE(aligned(q, 16) && aligned(out, 16) && aligned(workspace, 16) && ldq % 4 == 0 && ldo % (out_f16 ? 8 : 4) == 0,
               "jl_kv_attention: q, out and the workspace must be 16-byte aligned, ldq a multiple of 4 and ldo of %d", out_f16 ? 8 : 4);
    const size_t needed = jl_kv_attention_workspace_bytes(heads, cache->kv_heads, dim);
    if (workspace_bytes < needed)
        return jl_fail(JL_ERR_WORKSPACE, "jl_kv_attention: workspace of %zu bytes, %zu needed", workspace_bytes, needed);
    if (rows == 0) return JL_OK;
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    AttentionArgs a;
    a.cache = jl_kv_view(cache);
    a.q = q, a.ldq = ldq, a.ldo = ldo;
    a.positions = positions, a.row_requests = row_requests, a.table = block_table;
    a.requests = requests, a.table_stride = table_stride;
    a.scale = scale * 1.44269504088896340736f;
    a.window = window > INT32_MAX ? 0 : (int)window;   // one that reaches behind every position
    a.group = heads / cache->kv_heads;
    a.out = out, a.out_f16 = out_f16 != 0;
    if (cache->type == JL_KV_Q8_0) launch<true>(a, heads, (int)rows, dim, ctx->stream);
    else launch<false>(a, heads, (int)rows, dim, ctx->stream);
    JL_HIP(hipGetLastError());
    return JL_OK;
}

}  // extern "C"
