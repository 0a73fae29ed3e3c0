// jl_logprobs: log probabilities of given tokens, the entropy and the most probable tokens, of rows of logits.
//
// Mathematics.  x = l, or cap tanh(l / cap); m = max x; S = sum e^(scale (x - m)); T = sum e^(scale (x - m)) scale (x - m).
// Then log p(t) = scale (x_t - m) - log S and the entropy is log S - T / S.  The list is by l, equal ones by their index.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "jl_device.h"
#include "jl_internal.h"
#include "jl_kv.h"
#include "jl_math.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / JL_WAVE;
constexpr int kMostTop = 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

struct LogprobsArgs {
    const float *logits;
    int64_t stride;
    int n;
    float scale;
    float cap, one_over_cap;      // 0: none
    const int32_t *tokens;
    int tokens_per_row;
    float *logprobs, *entropy;
    int top;
    int32_t *top_tokens;
    float *top_logprobs;
};

// A logit of -infinity is a token that is left out, and stays one.
__device__ __forceinline__ float capped(const LogprobsArgs &p, float l) {
    return p.cap > 0.f && l != -INFINITY ? p.cap * jl_tanh(l * p.one_over_cap) : l;
}

// Larger logits are larger numbers, and of equal ones the earlier is; NaN is 0 and in no list.
__device__ __forceinline__ uint64_t key_of(float l, int at) {
    const uint32_t b = __float_as_uint(l + 0.f);              // (-0 is 0)
    const uint32_t order = b & 0x80000000u ? ~b : b | 0x80000000u;
    return l == l ? (uint64_t)order << 32 | (uint32_t)~at : 0;
}

__global__ void __launch_bounds__(kThreads) jl_logprobs_kernel(LogprobsArgs p) {
    __shared__ float part[3][kWaves];
    __shared__ uint64_t best_of[kWaves];
    const int tid = threadIdx.x, lane = tid % JL_WAVE, wave = tid / JL_WAVE;
    const int64_t row = blockIdx.x;
    const float *l = p.logits + row * p.stride;
    float most = -FLT_MAX;
    for (int i = tid; i < p.n; i += kThreads) most = fmaxf(most, capped(p, l[i]));
    for (int off = JL_WAVE / 2; off; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, JL_WAVE));
    if (lane == 0) part[0][wave] = most;
    __syncthreads();
    for (int w = 0; w < kWaves; w++) most = fmaxf(most, part[0][w]);
    float s = 0.f, t = 0.f;
    for (int i = tid; i < p.n; i += kThreads) {
        const float below = (capped(p, l[i]) - most) * (p.scale * kLog2e), a = below < -200.f ? -200.f : below;
        const float e = __builtin_amdgcn_exp2f(a);
        s += e, t += e * a;
    }
    for (int off = JL_WAVE / 2; off; off >>= 1) s += __shfl_xor(s, off, JL_WAVE), t += __shfl_xor(t, off, JL_WAVE);
    if (lane == 0) part[1][wave] = s, part[2][wave] = t;
    __syncthreads();
    s = t = 0.f;
    for (int w = 0; w < kWaves; w++) s += part[1][w], t += part[2][w];
    const float log_sum = logf(s);
    auto logprob = [&](float logit) { return s == 0.f ? -INFINITY : (capped(p, logit) - most) * p.scale - log_sum; };
    if (tid == 0 && p.entropy) p.entropy[row] = s == 0.f ? 0.f : log_sum - t / s * kLn2;
    for (int i = tid; i < p.tokens_per_row; i += kThreads) {
        const int token = p.tokens[row * p.tokens_per_row + i];
        p.logprobs[row * p.tokens_per_row + i] = (unsigned)token < (unsigned)p.n ? logprob(l[token]) : 0.f;
    }
    uint64_t before = UINT64_MAX;
    for (int k = 0; k < p.top; k++) {
        uint64_t best = 0;
        for (int i = tid; i < p.n; i += kThreads) {
            const uint64_t key = key_of(l[i], i);
            if (key < before && key > best) best = key;
        }
        for (int off = JL_WAVE / 2; off; off >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, off, JL_WAVE);
            best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) best_of[wave] = best;
        __syncthreads();
        for (int w = 0; w < kWaves; w++) best = best_of[w] > best ? best_of[w] : best;
        before = best;
        if (tid == 0) {
            const int at = (int)~(uint32_t)best;
            p.top_tokens[row * p.top + k] = best ? at : -1;
            p.top_logprobs[row * p.top + k] = best ? logprob(l[at]) : -INFINITY;
        }
    }
}

constexpr size_t kArrivedBytes = 16;

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

extern "C" {

size_t jl_logprobs_workspace_bytes(int64_t n, int top) {
    if (n <= 0 || n > INT32_MAX || top < 0 || top > kMostTop) return 0;
    return kArrivedBytes;
}

int jl_logprobs_workspace_init(jl_context *ctx, void *workspace, size_t workspace_bytes) {
    JL_REQUIRE(ctx && workspace, "jl_logprobs_workspace_init: null argument");
    JL_REQUIRE(aligned(workspace, 16), "jl_logprobs_workspace_init: the workspace must be 16-byte aligned");
    if (workspace_bytes < kArrivedBytes)
        return jl_fail(JL_ERR_WORKSPACE, "jl_logprobs_workspace_init: workspace of %zu bytes", workspace_bytes);
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    return jl_launch_fill(ctx, (float *)workspace, 0.f, kArrivedBytes / sizeof(float));
}

int jl_logprobs(jl_context *ctx, const float *logits, int64_t rows, int64_t n, int64_t row_stride, float scale, float cap,
                const int32_t *tokens, int64_t tokens_per_row, float *logprobs, float *entropy, int top,
                int32_t *top_tokens, float *top_logprobs, void *workspace, size_t workspace_bytes) {
    JL_REQUIRE(ctx && logits && workspace, "jl_logprobs: null argument");
    JL_REQUIRE(rows >= 0 && rows <= INT32_MAX, "jl_logprobs: %lld rows", (long long)rows);
    JL_REQUIRE(n > 0 && n <= INT32_MAX, "jl_logprobs: rows of %lld logits", (long long)n);
    JL_REQUIRE(row_stride >= n, "jl_logprobs: rows closer together (%lld) than they are long (%lld)", (long long)row_stride, (long long)n);
    JL_REQUIRE(std::isfinite(scale * kLog2e) && scale * kLog2e >= FLT_MIN, "jl_logprobs: scale %g (positive and finite)", (double)scale);
    JL_REQUIRE(cap == 0.f || (cap >= 1e-30f && cap <= 1e30f), "jl_logprobs: cap %g (0, or 1e-30 ... 1e30)", (double)cap);
    JL_REQUIRE(tokens_per_row >= 0 && tokens_per_row <= 65536, "jl_logprobs: %lld tokens a row (at most 65536)", (long long)tokens_per_row);
    JL_REQUIRE(tokens_per_row == 0 || (tokens && logprobs), "jl_logprobs: null tokens or logprobs for %lld a row", (long long)tokens_per_row);
    JL_REQUIRE(top >= 0 && top <= kMostTop && top <= n, "jl_logprobs: the %d most probable of %lld (at most %d)", top, (long long)n, kMostTop);
    JL_REQUIRE(top == 0 || (top_tokens && top_logprobs), "jl_logprobs: null top_tokens or top_logprobs for %d", top);
    JL_REQUIRE(aligned(logits, 4) && aligned(tokens, 4) && aligned(logprobs, 4) && aligned(entropy, 4) && aligned(top_tokens, 4) &&
                   aligned(top_logprobs, 4) && aligned(workspace, 16),
               "jl_logprobs: an unaligned array, or a workspace that is not 16-byte aligned");
    const size_t needed = jl_logprobs_workspace_bytes(n, top);
    if (workspace_bytes < needed)
        return jl_fail(JL_ERR_WORKSPACE, "jl_logprobs: workspace of %zu bytes, %zu needed", workspace_bytes, needed);
    if (rows == 0) return JL_OK;
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    LogprobsArgs a;
    a.logits = logits, a.stride = row_stride, a.n = (int)n;
    a.scale = scale, a.cap = cap, a.one_over_cap = cap > 0.f ? 1.f / cap : 0.f;
    a.tokens = tokens, a.tokens_per_row = (int)tokens_per_row, a.logprobs = logprobs, a.entropy = entropy;
    a.top = top, a.top_tokens = top_tokens, a.top_logprobs = top_logprobs;
    hipLaunchKernelGGL(jl_logprobs_kernel, dim3((unsigned)rows), dim3(kThreads), 0, ctx->stream, a);
    JL_HIP(hipGetLastError());
    return JL_OK;
}

}  // extern "C"
