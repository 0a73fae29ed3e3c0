// The paged key-value cache as its kernels see it (layout: jitllm_hip.h).
#pragma once

#include "jl_device.h"
#include "jl_internal.h"

struct jl_kv_cache {
    jl_context *ctx;
    int type;
    int64_t pages;
    int kv_heads;
    int head_dim;
    int page_tokens;
    size_t bytes;
    uint8_t *memory;
    bool owns_memory;
};

// Bytes of one head's part of a page.
static inline int64_t jl_kv_part_bytes(int type, int head_dim, int page_tokens) {
    const int64_t values = (int64_t)head_dim * page_tokens;
    return type == JL_KV_F16 ? 2 * values : values + values / 16;
}

// A cache by value, for kernels' arguments.
struct JlKvView {
    uint8_t *k;
    int64_t v_offset;     // bytes from a key's part of a page to its value's
    int64_t part_bytes;
    int pages;
    int kv_heads;
    int page_shift;       // page_tokens == 1 << page_shift
};

static inline JlKvView jl_kv_view(const jl_kv_cache *c) {
    JlKvView v;
    v.k = c->memory;
    v.v_offset = (int64_t)(c->bytes / 2);
    v.part_bytes = jl_kv_part_bytes(c->type, c->head_dim, c->page_tokens);
    v.pages = (int)c->pages;
    v.kv_heads = c->kv_heads;
    v.page_shift = __builtin_ctz((unsigned)c->page_tokens);
    return v;
}

typedef _Float16 jl_half8 __attribute__((ext_vector_type(8)));
typedef _Float16 jl_half4v __attribute__((ext_vector_type(4)));
typedef _Float16 jl_half2v __attribute__((ext_vector_type(2)));

// Four signed bytes as binary16: a byte b of 0 ... 255 under 0x64 is the binary16 of 1024 + b, so with the sign bit
// turned over (b = q + 128) one subtraction of 1152 leaves q, exactly.
__device__ __forceinline__ void jl_bytes_to_half(uint32_t q, jl_half2v &lo, jl_half2v &hi) {
    const uint32_t b = q ^ 0x80808080u;
    const jl_half2v bias = {(_Float16)1152.f, (_Float16)1152.f};
    lo = __builtin_bit_cast(jl_half2v, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - bias;
    hi = __builtin_bit_cast(jl_half2v, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - bias;
}

// Eight consecutive values, from element 8 * chunk of a token's, of the part of a page at `part`.
template <bool Q8>
__device__ __forceinline__ jl_half8 jl_kv_load8(const uint8_t *part, int page_shift, int head_dim, int token, int chunk) {
    if constexpr (!Q8) {
        return *(const jl_half8 *)(part + ((int64_t)token * head_dim + 8 * chunk) * 2);
    } else {
        const uint2 q = *(const uint2 *)(part + token * head_dim + 8 * chunk);
        const _Float16 *scales = (const _Float16 *)(part + ((int64_t)head_dim << page_shift));
        const _Float16 d = scales[((chunk >> 2) << page_shift) + token];
        jl_half2v h[4];
        jl_bytes_to_half(q.x, h[0], h[1]);
        jl_bytes_to_half(q.y, h[2], h[3]);
        jl_half8 r;
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = h[i / 2][i % 2] * d;
        return r;
    }
}

// Kernels of a context run on its device whichever is the current one, and leave the caller's as it was.
struct JlOnDevice {
    int before = -1;
    hipError_t status;
    explicit JlOnDevice(const jl_context *ctx) {
        status = hipGetDevice(&before);
        if (status == hipSuccess && before == ctx->device) before = -1;
        else if (status == hipSuccess) status = hipSetDevice(ctx->device);
    }
    ~JlOnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
