// The kernel of attention over pages for blocks of rows of few requests: a prompt's.
//
// Mathematics and layouts are those of jl_attention_kernel.h.  There the waves of a workgroup share 16 columns, a (row,
// query head) each, and take the tokens in turn: every 16 columns read all tokens.  Here a workgroup has 64 columns, 16 a
// wave, that go through the same tokens.  Two tiles of 32 tokens at a time, each wave loads a half of one, decodes it, turns v
// as the second product wants it, and leaves the matrix instructions' operands in LDS, as they are; all waves then
// take both tiles from there, while the next two go on to the other buffer and two more are on their way.  What a tile costs to
// load and decode is paid once for 64 columns.
//
// Bound: the matrix instructions, four for a 16 x 16 x 32 piece (q and P are two binary16 parts each), and, as much, the
// powers and conversions of P.
//
// Work.  A workgroup has a block of rows beside each other and a head of k and v.  Rows of one request whose
// ranges touch go together, one run after the other.  A block with a run that is long and has few rows is left, whole, to the
// other kernel, which cuts long ranges among workgroups; `taken` says to it which are not.
#pragma once

#include "jl_attention_kernel.h"

namespace {

constexpr int kLongRun = 32;                      // tiles of a run that has to have a quarter of the block's rows
constexpr int kLongPrompt = 2000;                 // rows a request
constexpr int kColumnWaves = 4, kTilesAtATime = 2;   // waves beside each other, and the tiles that one takes at a time

// WAVES: four, or eight, the second four of which take every other two tiles, and are joined with the first through LDS: where there are
// no more workgroups than compute units, each of which would have one wave a SIMD (4-bit cache, 8 query heads over 4 of 128: 1400
// rows of a prompt, 176 workgroups, 44.0 -> 34.6 us; 4 prompts of 175 ... 700 with a cap and a prefix, 220, 42.3 -> 37.6; 512 rows after
// 30 000 tokens, 32 over 8, binary16, 256: 750 -> 570); and up to twice as many of prompts of kLongPrompt rows or more, the last of whose
// blocks would else go on alone (8 heads over 4 of 128, 2400 rows, 300: 73 -> 57; 4096, 512: 115 -> 97; 16 over 8 of 64, 2000 rows,
// 504: 46 -> 42; but 900 rows of 32 over 8, 456: 34.5 and 36.1, 8 prompts of 512, 512: 29.9 and 36.1, 3200 with a window of 300, 400: 26.4
// and 33.6).  Their LDS holds up to 128 values a head.
template <int DIM, int WAVES>
struct PromptShape {
    static constexpr int kFragments = DIM / 16 + DIM / 16;                 // of a tile, 1 KB each: k's, v's
    static constexpr int kTilesStaged = WAVES / kHalves;                   // a half by each wave
    static constexpr int kBufferBytes = kTilesStaged * kFragments * 1024, kLdsBytes = 2 * kBufferBytes;
    static constexpr int kWavesASimd = DIM <= 128 ? 2 : 1;
};

// over the sixteen lanes of a row of lanes, and over all, in all of them
__device__ __forceinline__ int over_16_min(int x) {
#define JL_MIN_FROM(N) x = min(x, __builtin_amdgcn_update_dpp(0, x, 0x120 + N, 0xF, 0xF, true));
    JL_MIN_FROM(8) JL_MIN_FROM(4) JL_MIN_FROM(2) JL_MIN_FROM(1)
#undef JL_MIN_FROM
    return x;
}
__device__ __forceinline__ int over_lanes_min(int x) {
    x = over_16_min(x);
    const auto f = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
    x = min((int)f[0], (int)f[1]);
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
    return min((int)h[0], (int)h[1]);
}

template <int TYPE, int DIM, int WAVES>
__global__ void __launch_bounds__(WAVES * JL_WAVE, (PromptShape<DIM, WAVES>::kWavesASimd)) jl_kv_attention_prompt_kernel(JlScoredArgs p) {
    typedef PromptShape<DIM, WAVES> Its;
    constexpr int kSteps = DIM / 32, kBlocks = DIM / 16, kFragments = Its::kFragments, kTilesStaged = Its::kTilesStaged;
    extern __shared__ __align__(16) uint8_t fragments[];       // [2][kTilesStaged][kFragments][64 lanes][16 bytes]
    __shared__ int half_info[2][WAVES];
    const int tid = threadIdx.x, lane = tid % JL_WAVE, wave = uniform(tid / JL_WAVE);
    const int column_wave = WAVES > kColumnWaves ? wave % kColumnWaves : wave;
    const int own_tiles = WAVES > kColumnWaves ? wave / kColumnWaves * kTilesAtATime : 0;   // of those that are staged
    const int g = lane / 16, m = lane % 16;
    const int kv_heads = p.cache.kv_heads, kv_head = blockIdx.x % kv_heads;
    const int block = gridDim.x / kv_heads - 1 - blockIdx.x / kv_heads;    // (the last rows first: a prompt's longest)
    const int row0 = block * p.taken_rows, rows = min(p.taken_rows, p.rows - row0);
    const int page_shift = p.cache.page_shift, in_page_mask = (1 << page_shift) - 1;

    // ---- the rows' ranges, one a lane, and the runs that they make; rows without tokens make runs of their own
    Range in_lane{0, -1, -1};
    int position_in_lane;
    {
        const int row = row0 + min(lane, rows - 1);
        position_in_lane = p.positions[row];
        const Range r = range_at(p, row, position_in_lane, p.row_requests[row]);
        if (lane < rows && r.end > r.first) in_lane = r;
    }
    const Range before{__shfl_up(in_lane.first, 1, JL_WAVE), __shfl_up(in_lane.end, 1, JL_WAVE), __shfl_up(in_lane.request, 1, JL_WAVE)};
    const bool goes = lane > 0 && (in_lane.request < 0 ? before.request < 0 : goes_on(before, in_lane));
    const uint64_t starts = __ballot(lane < rows && !goes);
    auto run_end = [&](int from) {                            // of the run that begins at row `from`
        const uint64_t behind = from < JL_WAVE - 1 ? starts >> (from + 1) : 0;
        return behind ? from + 1 + (int)__builtin_ctzll(behind) : rows;
    };
    auto run_range = [&](int from, int to) {
        const bool is = lane >= from && lane < to;
        return Range{uniform(over_lanes_min(is ? in_lane.first : INT_MAX)), uniform(-over_lanes_min(is ? -in_lane.end : INT_MAX)),
                     __builtin_amdgcn_readlane(in_lane.request, from)};
    };
    bool some = false, takes = true;
    for (int from = 0, to; from < rows; from = to) {
        to = run_end(from);
        const int tiles = run_range(from, to).tiles();
        some |= tiles > 0;
        takes &= tiles <= kLongRun || 4 * (to - from) >= p.taken_rows;
    }
    takes &= some;
    if (kv_head == 0 && tid == 0) p.taken_out[block] = takes;
    if (!takes) return;

    Raw<TYPE, DIM, 1> raw[2];                                 // two tiles' and the next two's
    for (int from = 0, to; from < rows; from = to) {
        to = run_end(from);
        const int columns = (to - from) * p.group;
        const Range run = run_range(from, to);
        const int tile_begin = run.first / kTile, tile_end = run.end > run.first ? (run.end + kTile - 1) / kTile : tile_begin;

        // a half of a tile of this wave's: its page, and the loads
        const int its_tile = wave / kHalves, its_half = wave % kHalves;
        bool paged[2];
        auto issue = [&](auto which, int t) {
            constexpr int W = decltype(which)::value;
            paged[W] = false;
            if (t >= tile_end) return;
            typedef const __attribute__((address_space(4))) int32_t constant_int;
            constant_int *table = (constant_int *)(uintptr_t)(p.table + run.request * p.table_stride);
            const int token = t * kTile + 16 * its_half;
            const int page = token < run.end ? table[token >> page_shift] : -1;
            paged[W] = (unsigned)page < (unsigned)p.cache.pages;
            const uint8_t *part = p.cache.k + ((int64_t)(paged[W] ? page : 0) * kv_heads + kv_head) * p.cache.part_bytes;
            raw[W].template load_k<true>(0, part, token & in_page_mask, page_shift, g, m);
            raw[W].template load_v<true>(0, part + p.cache.v_offset, token & in_page_mask, page_shift, g, m);
        };
        // what was loaded, into a buffer; a half behind the last tile, or with no page, as tokens that nobody sees
        auto stage = [&](auto which, int t) {
            constexpr int W = decltype(which)::value;
            const int token0 = min(t, tile_end) * kTile + 16 * its_half;
            if (token0 < run.first || token0 + 16 > run.end || !paged[W]) {
                bool seen[1][4];
#pragma unroll
                for (int i = 0; i < 4; i++) seen[0][i] = token0 + 4 * g + i >= run.first && token0 + 4 * g + i < run.end && paged[W];
                raw[W].mask_v(seen);
            }
            const bool bad = __any(raw[W].any_not_finite());
            if (lane == 0) half_info[W][wave] = (paged[W] ? 1 : 0) | (bad ? 2 : 0);
            uint8_t *to_fragment = fragments + W * Its::kBufferBytes + its_tile * (kFragments * 1024) + lane * 16;
#pragma unroll
            for (int s = 0; s < kSteps; s++) *(jl_half8 *)(to_fragment + (its_half * kSteps + s) * 1024) = raw[W].k_operand(0, s);
#pragma unroll
            for (int b = 0; b < kBlocks; b += 2) {
                uintx2 v[2];
                raw[W].v_pairs(b, v);
#pragma unroll
                for (int c = 0; c < 2; c++) *(uintx2 *)(to_fragment + (kBlocks + b + c) * 1024 + 8 * its_half) = v[c];
            }
        };
        const std::integral_constant<int, 0> even{};
        const std::integral_constant<int, 1> odd{};
        issue(even, tile_begin + its_tile);
        issue(odd, tile_begin + kTilesStaged + its_tile);

        // ---- this wave's columns: the query heads of one row after the other; lanes past the last one double it
        const bool works = column_wave * 16 < columns;
        const int column = min(column_wave * 16 + m, columns - 1), in_run = column / p.group;
        const int row = row0 + from + in_run, head = kv_head * p.group + column - in_run * p.group;
        const int position = __shfl(position_in_lane, from + in_run, JL_WAVE);
        const int first_seen = __shfl(in_lane.first, from + in_run, JL_WAVE), end_seen = __shfl(in_lane.end, from + in_run, JL_WAVE);
        // of all columns, and of any
        const int all_first = uniform(-over_16_min(-first_seen)), all_end = uniform(over_16_min(end_seen));
        const int any_first = uniform(over_16_min(first_seen)), any_end = uniform(-over_16_min(-end_seen));
        const float slope = p.slopes ? 1.44269504088896340736f * p.slopes[head] : 0.f;
        float undo = 0.f, top = kNone, sum = 0.f;
        jl_half8 q_hi[kSteps], q_lo[kSteps];
        floatx4 o[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) o[b] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (works) {
            const float *x_from = p.q + row * p.ldq + (int64_t)head * DIM;
            floatx4 x[kSteps][2];
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; s++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    x[s][e] = *(const floatx4 *)(x_from + Raw<TYPE, DIM>::element(s, g) + 4 * e);
                    x[s][e] *= p.scale;
#pragma unroll
                    for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(x[s][e][i]));
                }
            most = over_groups_max(most);
            JL_SPLIT_Q(TYPE, DIM, x, most, q_hi, q_lo, undo);
        }

        __syncthreads();                                      // (all have read what the run before left)
        stage(even, tile_begin + its_tile);
        issue(even, tile_begin + 2 * kTilesStaged + its_tile);
        auto step = [&](auto which, auto other, int staged) {
            const int base = staged + own_tiles;              // this wave's two
            constexpr int buffer = decltype(which)::value;
            __syncthreads();                                  // (this buffer is written, and the other one read, by all)
            const uint8_t *fragment = fragments + buffer * Its::kBufferBytes + own_tiles * (kFragments * 1024) + lane * 16;
            auto operand = [&](int i) { return *(const jl_half8 *)(fragment + (i / (2 * kBlocks) * kFragments + i % (2 * kBlocks)) * 1024); };
            int info = 0, bad = 0;                            // bit i: half i has a page; one has values that are not finite
#pragma unroll
            for (int i = 0; i < WAVES; i++) bad |= half_info[buffer][i];
            bad = uniform(bad) & 2;
#pragma unroll
            for (int i = 0; i < kTilesAtATime * kHalves; i++) info |= (uniform(half_info[buffer][own_tiles * kHalves + i]) & 1) << i;
            const bool reads = works && base * kTile < any_end && (base + kTilesAtATime) * kTile > any_first;
            auto sees = [&](int i) {                          // token i of the lane's sixteen
                const int token = base * kTile + i / 4 * 16 + 4 * g + i % 4;
                return token >= first_seen && token < end_seen && (info >> i / 4 & 1);
            };
            if (bad) {
                // An infinity or NaN among the values: NaN to the columns that see it (2^127 in its place times 2^127, and times
                // -2^127), and 0 where it lay.
                if (reads) {
#pragma unroll 1
                    for (int t = 0; t < kTilesAtATime; t++) {
                        uintx4 plus;
#pragma unroll
                        for (int i = 0; i < 8; i += 2) plus[i / 2] = (sees(8 * t + i) ? 0x7f00u : 0u) | (sees(8 * t + i + 1) ? 0x7f000000u : 0u);
                        const bfloat8 both[2] = {__builtin_bit_cast(bfloat8, plus), __builtin_bit_cast(bfloat8, plus ^ 0x80008000u)};
#pragma unroll
                        for (int b = 0; b < kBlocks; b++) {
                            uintx4 its = __builtin_bit_cast(uintx4, operand(2 * kBlocks * t + kBlocks + b));
#pragma unroll
                            for (int i = 0; i < 4; i++) its[i] = not_finite(its[i]) & 0x7f007f00u;
#pragma unroll
                            for (int i = 0; i < 2; i++) o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloat8, its), both[i], o[b], 0, 0, 0);
                        }
                    }
                }
                __syncthreads();
                uint8_t *own_half = fragments + buffer * Its::kBufferBytes + its_tile * (kFragments * 1024) + lane * 16 + 8 * its_half;
#pragma unroll 1
                for (int b = 0; b < kBlocks; b++) {
                    uintx2 *at = (uintx2 *)(own_half + (kBlocks + b) * 1024);
                    const uintx2 v = *at;
                    *at = uintx2{v.x & ~not_finite(v.x), v.y & ~not_finite(v.y)};
                }
                __syncthreads();
            }
            if (reads) {
                // (operands come from LDS a step ahead of the matrix instructions that take them, the values' first ones before
                // the weights are worked out)
                constexpr int kAtOnce = kTilesAtATime * kHalves;
                floatx4 s[kAtOnce];
                jl_half8 k[2][kAtOnce];
                auto key_operand = [&](int step, int i) { return operand(2 * kBlocks * (i / kHalves) + i % kHalves * kSteps + step); };
#pragma unroll
                for (int i = 0; i < kAtOnce; i++) s[i] = floatx4{0.f, 0.f, 0.f, 0.f}, k[0][i] = key_operand(0, i);
#pragma unroll
                for (int step = 0; step < kSteps; step++) {
                    if (step + 1 < kSteps) {
#pragma unroll
                        for (int i = 0; i < kAtOnce; i++) k[(step + 1) % 2][i] = key_operand(step + 1, i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < kAtOnce; i++) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[step % 2][i], q_lo[step], s[i], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < kAtOnce; i++) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[step % 2][i], q_hi[step], s[i], 0, 0, 0);
                }
                constexpr int kAhead = 4;
                jl_half8 v[2][kAhead];
                auto value_operand = [&](int i) { return operand(i / kBlocks * 2 * kBlocks + kBlocks + i % kBlocks); };
#pragma unroll
                for (int i = 0; i < kAhead; i++) v[0][i] = value_operand(i);
                __builtin_amdgcn_sched_barrier(0);
                const bool all_seen = base * kTile >= all_first && (base + kTilesAtATime) * kTile <= all_end && info == (1 << kTilesAtATime * kHalves) - 1;
                const bool shaped = p.cap > 0.f || p.slopes;
                const float unit = shaped ? 1.f : undo;       // of a score, in powers of two
                float x[kTilesAtATime][8];
                float most = -INFINITY;
#pragma unroll
                for (int t = 0; t < kTilesAtATime; t++) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[t][i] = s[t * kHalves + i / 4][i % 4];
                    if (shaped) shape_scores(p, x[t], undo, slope, (base + t) * kTile + 4 * g - position);
                    if (!all_seen) {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[t][i] = sees(8 * t + i) ? x[t][i] : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) most = fmaxf(most, x[t][i]);
                }
                most = over_groups_max(most) * unit;
                if (__any(most > top + kSlack)) {
                    const float next_top = fmaxf(top, most);
                    const float keep = __builtin_amdgcn_exp2f(top - next_top);
                    top = next_top;
                    sum *= keep;
#pragma unroll
                    for (int b = 0; b < kBlocks; b++) o[b] *= keep;
                }
                jl_half8 p_hi[kTilesAtATime], p_lo[kTilesAtATime];
#pragma unroll
                for (int t = 0; t < kTilesAtATime; t++) weights_of(x[t], unit, kLift - top, sum, p_hi[t], p_lo[t]);
                constexpr int kValues = kTilesAtATime * kBlocks;
#pragma unroll
                for (int from = 0; from < kValues; from += kAhead) {
                    const int now = from / kAhead % 2;
                    if (from + kAhead < kValues) {
#pragma unroll
                        for (int i = 0; i < kAhead; i++)
                            if (from + kAhead + i < kValues) v[1 - now][i] = value_operand(from + kAhead + i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < kAhead; i++)
                        if (from + i < kValues) {
                            const int b = (from + i) % kBlocks, its = (from + i) / kBlocks;
                            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[now][i], p_lo[its], o[b], 0, 0, 0);
                        }
#pragma unroll
                    for (int i = 0; i < kAhead; i++)
                        if (from + i < kValues) {
                            const int b = (from + i) % kBlocks, its = (from + i) / kBlocks;
                            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[now][i], p_hi[its], o[b], 0, 0, 0);
                        }
                }
            }
            if (staged + kTilesStaged < tile_end) {
                stage(other, staged + kTilesStaged + its_tile);
                issue(other, staged + 3 * kTilesStaged + its_tile);
            }
        };
        for (int base = tile_begin; base < tile_end; base += 2 * kTilesStaged) {
            step(even, odd, base);
            if (base + kTilesStaged < tile_end) step(odd, even, base + kTilesStaged);
        }
        if constexpr (WAVES > kColumnWaves) {
            // the second four waves' parts, through LDS, to the first ones
            float *joined = (float *)fragments + column_wave * ((4 * kBlocks + 2) * JL_WAVE) + lane;
            __syncthreads();
            if (own_tiles > 0 && works) {
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) joined[(4 * b + i) * JL_WAVE] = o[b][i];
                joined[4 * kBlocks * JL_WAVE] = top, joined[(4 * kBlocks + 1) * JL_WAVE] = sum;
            }
            __syncthreads();
            if (own_tiles > 0) continue;
            if (works) {
                const float its_top = joined[4 * kBlocks * JL_WAVE], most = fmaxf(top, its_top);
                const float keep = __builtin_amdgcn_exp2f(top - most), share = __builtin_amdgcn_exp2f(its_top - most);
                sum = keep * sum + share * joined[(4 * kBlocks + 1) * JL_WAVE];
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[b][i] = keep * o[b][i] + share * joined[(4 * b + i) * JL_WAVE];
            }
        }
        if (!works) continue;
        const float l = over_groups_sum(sum);
        if (column_wave * 16 + m >= columns) continue;
        const int64_t at = row * p.ldo + (int64_t)head * DIM;
        auto put = [&](int element, floatx4 v) { store_out(p, at + element, l == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : v / l); };
        constexpr int wide = DIM / 128, mid = DIM % 128 / 64, thin = DIM % 64 / 32;
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int b = 0; b < 8 * wide; b += 4) put(128 * (b / 8) + 8 * (4 * g + i) + b % 8, floatx4{o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]});
            if constexpr (mid) {
                constexpr int b = 8 * wide;
                put(128 * wide + 4 * (4 * g + i), floatx4{o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]});
            }
            if constexpr (thin) {
                constexpr int b = 8 * wide + 4 * mid;
                if (i % 2 == 0) put(128 * wide + 64 * mid + 2 * (4 * g + i), floatx4{o[b][i], o[b + 1][i], o[b][i + 1], o[b + 1][i + 1]});
            }
        }
    }
}

template <int TYPE, int DIM, int WAVES>
hipError_t launch_prompt_waves(const JlScoredArgs &a, unsigned groups, int device, hipStream_t stream) {
    constexpr int lds = PromptShape<DIM, WAVES>::kLdsBytes;
    if (lds > 60 * 1024) {
        static jl_lds_limit_flags raised;
        if (jl_raise_lds_limit(raised, device, (const void *)jl_kv_attention_prompt_kernel<TYPE, DIM, WAVES>, lds) != JL_OK) return hipErrorInvalidValue;
    }
    hipLaunchKernelGGL((jl_kv_attention_prompt_kernel<TYPE, DIM, WAVES>), dim3(groups), dim3(WAVES * JL_WAVE), lds, stream, a);
    return hipGetLastError();
}
template <int TYPE, int DIM>
hipError_t launch_prompt(const JlScoredArgs &a, int compute_units, int device, hipStream_t stream) {
    const unsigned groups = (unsigned)((a.rows + a.taken_rows - 1) / a.taken_rows) * a.cache.kv_heads;
    const bool long_runs = a.window == 0 && !a.first_tokens && kLongPrompt * (int64_t)a.requests <= a.rows;
    if constexpr (DIM <= 128)
        if (groups <= (unsigned)compute_units * (long_runs ? 2 : 1)) return launch_prompt_waves<TYPE, DIM, 8>(a, groups, device, stream);
    return launch_prompt_waves<TYPE, DIM, 4>(a, groups, device, stream);
}
template <int TYPE>
hipError_t launch_prompt_dim(const JlScoredArgs &a, int head_dim, int compute_units, int device, hipStream_t stream) {
    switch (head_dim) {
        case 64: return launch_prompt<TYPE, 64>(a, compute_units, device, stream);
        case 96: return launch_prompt<TYPE, 96>(a, compute_units, device, stream);
        case 128: return launch_prompt<TYPE, 128>(a, compute_units, device, stream);
        case 192: return launch_prompt<TYPE, 192>(a, compute_units, device, stream);
        default: return launch_prompt<TYPE, 256>(a, compute_units, device, stream);
    }
}

}  // namespace
