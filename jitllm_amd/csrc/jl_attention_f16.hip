// jl_kv_attention's and jl_kv_attention_scored's kernels over a cache of JL_KV_F16.
#include "jl_attention_kernel.h"

hipError_t jl_launch_attention_f16(const JlAttentionArgs &a, int head_dim, int compute_units, hipStream_t stream) {
    return launch_dim<JL_KV_F16>(a, head_dim, compute_units, stream);
}
hipError_t jl_launch_attention_scored_f16(const JlScoredArgs &a, int head_dim, int compute_units, hipStream_t stream) {
    return launch_dim<JL_KV_F16>(a, head_dim, compute_units, stream);
}
