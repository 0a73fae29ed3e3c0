// jl_kv_attention's and jl_kv_attention_scored's kernels over a cache of JL_KV_Q8_0.
#include "jl_attention_kernel.h"

hipError_t jl_launch_attention_q8(const JlAttentionArgs &a, int head_dim, int compute_units, hipStream_t stream) {
    return launch_dim<JL_KV_Q8_0>(a, head_dim, compute_units, stream);
}
hipError_t jl_launch_attention_scored_q8(const JlScoredArgs &a, int head_dim, int compute_units, hipStream_t stream) {
    return launch_dim<JL_KV_Q8_0>(a, head_dim, compute_units, stream);
}
