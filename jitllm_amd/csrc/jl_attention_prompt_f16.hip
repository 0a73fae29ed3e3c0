// The kernel for blocks of rows, over a cache of JL_KV_F16.
#include "jl_attention_prompt.h"

hipError_t jl_launch_attention_prompt_f16(const JlScoredArgs &a, int head_dim, int compute_units, int device, hipStream_t stream) {
    return launch_prompt_dim<JL_KV_F16>(a, head_dim, compute_units, device, stream);
}
