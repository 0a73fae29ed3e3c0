// What the attention's kernels take, for the sources that they are built in.
#pragma once

#include <type_traits>

#include "jl_kv.h"

constexpr int kAttentionMostGroups = 512, kAttentionStart = 4;   // (what they are: jl_attention_kernel.h)

struct JlAttentionArgs {
    JlKvView cache;
    const float *q;
    int64_t ldq, ldo;
    const int32_t *positions, *row_requests, *table;
    int64_t table_stride;
    int requests;
    int table_tokens;     // of a row of the table, at most 2^31 - 64
    float scale;          // times log2(e): weights are powers of two
    int window;           // 0: none
    int group;            // query heads to a head of k and v
    int blocks_of_16;     // ... in sixteens
    int rows;
    void *out;
    bool out_f16;
    uint32_t *arrived;    // [kAttentionMostGroups], all 0 between calls
    float *parts;         // [2 * spans][16 * (DIM + 2)]
    // Rows of one request that go together: a power of two, at most 16 / group; 1: each alone.  (The last argument: among the
    // others it moved some to another load, and every call took 0.1 ... 0.2 us longer.)
    int rows_each;
};

// ... with scores that are capped or lowered by distance, and rows that see other tokens than those up to their own.
struct JlScoredArgs : JlAttentionArgs {
    float cap, one_over_cap;                     // of scores that are powers of two; 0: none
    const float *slopes;                         // [heads], or null
    const int32_t *first_tokens, *end_tokens;    // [rows], or null
    // Blocks of this many rows, a multiple of rows_each, that jl_kv_attention_prompt_kernel has taken: what it says, and what the
    // other kernel reads (null: there was no such launch).
    int taken_rows;
    uint8_t *taken_out;
    const uint8_t *taken;
};
template <typename ARGS>
inline constexpr bool kScored = std::is_same_v<ARGS, JlScoredArgs>;

hipError_t jl_launch_attention_prompt_f16(const JlScoredArgs &a, int head_dim, int compute_units, int device, hipStream_t stream);
hipError_t jl_launch_attention_prompt_q8(const JlScoredArgs &a, int head_dim, int compute_units, int device, hipStream_t stream);
hipError_t jl_launch_attention_prompt_q4(const JlScoredArgs &a, int head_dim, int compute_units, int device, hipStream_t stream);
hipError_t jl_launch_attention_f16(const JlAttentionArgs &a, int head_dim, int compute_units, hipStream_t stream);
hipError_t jl_launch_attention_q8(const JlAttentionArgs &a, int head_dim, int compute_units, hipStream_t stream);
hipError_t jl_launch_attention_q4(const JlAttentionArgs &a, int head_dim, int compute_units, hipStream_t stream);
hipError_t jl_launch_attention_scored_f16(const JlScoredArgs &a, int head_dim, int compute_units, hipStream_t stream);
hipError_t jl_launch_attention_scored_q8(const JlScoredArgs &a, int head_dim, int compute_units, hipStream_t stream);
hipError_t jl_launch_attention_scored_q4(const JlScoredArgs &a, int head_dim, int compute_units, hipStream_t stream);
