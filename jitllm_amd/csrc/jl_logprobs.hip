// jl_logprobs: log probabilities of given tokens, the entropy and the most probable tokens, of rows of logits.
//
// Mathematics.  x = l, or cap tanh(l / cap); m = max x; with a = scale log2(e) (x - m), S = sum 2^a and T = sum 2^a a.  Then
// log p(t) = scale (x_t - m) - log S and the entropy is log S - log(2) T / S.  Two parts (m, S, T) of a row join by bringing
// both to the larger m: S by 2^d and T by (T + S d) 2^d, d = scale log2(e) (m - m').  The list is by l, equal ones by
// their index: one 64-bit key that is larger for the one that comes first.
//
// Bound: the bytes of the logits, once.  A wave goes through its part in steps of 16 values a lane, the next step's on their
// way; each lane has a running m, S and T.  For the list the wave keeps its largest keys so far, sorted, one a lane: a step
// none of whose values reaches the last one that is wanted costs one comparison.  From others those that do are gathered
// in LDS, and every 64 sorted and merged in.  The first step, and any that would gather more than 64, sorts its lanes'
// largest first: of the top ones of those there are as many as are wanted, so that nothing below the last of them is.
//
// Work.  A workgroup of four waves a row (one wave where rows are short); where rows are few each is cut into parts, and the
// workgroup that is done last with a row joins them, in their order whoever that is (nobody waits for anybody).
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "jl_device.h"
#include "jl_internal.h"
#include "jl_kv.h"
#include "jl_math.h"

// A product and a sum become one rounding where fmaf says so, and nowhere else: what a call leaves is the same whatever else it is
// asked for, which is another kernel.
#pragma clang fp contract(off)

namespace {

constexpr int kMostTop = JL_WAVE;                 // a lane each
constexpr int kEach = 4;                          // loads of four values a lane and step
constexpr int kStepFours = kEach * JL_WAVE;       // fours of a wave's step
constexpr int kMostParts = 32;                    // of a row
constexpr int kPartsRows = 512;                   // rows that are cut
// Workgroups that a launch of few rows has, about (256 rows of 128256, five alternatives: 66 us with 512, 44 with 1024, 50 with
// 2048; 64 of 151936, twenty: 25.7, 24.4 and 35.5).
constexpr int kGroups = 1024;
constexpr int kShortRow = 2048;                   // logits of a row that one wave has
constexpr int64_t kMostLogits = 1 << 30;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

struct Part {
    uint64_t keys[kMostTop];
    float most, sum, weighted, unused;
};

struct LogprobsArgs {
    const float *logits;
    int64_t stride;
    int n;
    int parts, fours_each;        // parts of a row, and fours of a part: whole steps of a workgroup
    float scale, power;           // power: scale log2(e)
    float cap, one_over_cap;      // 0: none
    // The quotient of jl_tanh_middle for logits of at most cap_middle, in powers of the logit's square: l (1 + ...) / (1 + ...) is
    // the capped logit, with no product in front and none behind.
    float cap_middle, over[3], under[3];
    // ... and Lambert's fraction up to 9, which is off by 6.2e-8 of the value at 1, for those of at most cap_near (2048 rows of
    // 32000, capped: as products around the longer one 69 us, as powers of the square 68, the shorter one 62).
    float cap_near, near_over[2], near_under[2];
    const int32_t *tokens;
    int tokens_per_row;
    float *logprobs, *entropy;
    int top;
    int32_t *top_tokens;
    float *top_logprobs;
    uint32_t *arrived;            // [kPartsRows], all 0 between calls
    Part *part;                   // [rows * parts]
};

// A logit of -infinity is a token that is left out, and stays one.
__device__ __forceinline__ float capped(const LogprobsArgs &p, float l) {
    return p.cap > 0.f && l != -INFINITY ? p.cap * jl_tanh(l * p.one_over_cap) : l;
}

// Larger logits are larger numbers (-0 is 0, NaN a 0), and back; in the key, of equal ones the earlier is the larger.
__device__ __forceinline__ uint32_t order_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return l == l ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0;
}
__device__ __forceinline__ float logit_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ uint64_t key_of(float l, uint32_t at) { return (uint64_t)order_of(l) << 32 | ~at; }

// The value of lane ^ N, by moves between lanes alone.
template <int N>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x, int lane) {
#define JL_MOVE(X, CONTROL) (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(X), CONTROL, 0xF, 0xF, true)
    if constexpr (N == 1) return JL_MOVE(x, 0xB1);                        // quad_perm 1 0 3 2
    if constexpr (N == 2) return JL_MOVE(x, 0x4E);                        // quad_perm 2 3 0 1
    if constexpr (N == 4) return JL_MOVE(JL_MOVE(x, 0x141), 0x1B);        // row_half_mirror (^ 7), quad_perm 3 2 1 0 (^ 3)
    if constexpr (N == 8) return JL_MOVE(x, 0x128);                       // row_ror 8
#undef JL_MOVE
    if constexpr (N == 16) {
        const auto f = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return lane & 16 ? f[0] : f[1];
    }
    if constexpr (N == 32) {
        const auto f = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return lane & 32 ? f[0] : f[1];
    }
    return x;
}
template <int N>
__device__ __forceinline__ uint64_t lane_xor(uint64_t x, int lane) {
    return (uint64_t)lane_xor<N>((uint32_t)(x >> 32), lane) << 32 | lane_xor<N>((uint32_t)x, lane);
}
template <int N>
__device__ __forceinline__ float lane_xor(float x, int lane) { return __uint_as_float(lane_xor<N>(__float_as_uint(x), lane)); }

// One step of a sorting network: of the pair (lane, lane ^ N) this lane keeps the larger key where `larger`.
template <int N, typename KEY>
__device__ __forceinline__ KEY keep_of_pair(KEY own, bool larger, int lane) {
    const KEY other = lane_xor<N>(own, lane);
    return (other > own) == larger ? other : own;
}
// A sequence over 2 FROM lanes that rises and then falls, or the other way round, into a falling (or rising) one.
template <int FROM, typename KEY>
__device__ __forceinline__ KEY bitonic_sorted(KEY key, bool falling, int lane) {
    key = keep_of_pair<FROM>(key, ((lane & FROM) == 0) == falling, lane);
    if constexpr (FROM > 1) return bitonic_sorted<FROM / 2>(key, falling, lane);
    else return key;
}
// Every W lanes sorted.
template <int W, typename KEY>
__device__ __forceinline__ KEY sorted(KEY key, bool falling, int lane) {
    if constexpr (W > 2) key = sorted<W / 2>(key, (lane & (W / 2)) == 0, lane);
    return bitonic_sorted<W / 2>(key, falling, lane);
}
// The W largest of a wave whose W lanes each are sorted, falling and rising in turn: falling (or rising) in every W lanes.
template <int W>
__device__ __forceinline__ uint64_t largest_of(uint64_t key, bool falling, int lane) {
    if constexpr (W <= 16) {
        const uint64_t other = lane_xor<16>(key, lane);
        key = bitonic_sorted<W / 2>(other > key ? other : key, (lane & 32) == 0, lane);
    }
    if constexpr (W <= 32) {
        const uint64_t other = lane_xor<32>(key, lane);
        key = bitonic_sorted<W / 2>(other > key ? other : key, falling, lane);
    }
    return key;
}
template <int W>
__device__ __forceinline__ bool falls(int lane) { return W == JL_WAVE || (lane & W) == 0; }   // in turn
// The W largest of a falling and a rising sequence of W, falling.
template <int W>
__device__ __forceinline__ uint64_t merged(uint64_t falling, uint64_t rising, int lane) {
    return bitonic_sorted<W / 2>(falling > rising ? falling : rising, true, lane);
}

// 2^it is 0, and 0 times it no NaN, as 0 times -infinity is.
constexpr float kFar = -200.f;

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct Sums {
    float most = -FLT_MAX, sum = 0.f, weighted = 0.f;
    __device__ __forceinline__ void bring_to(float other_most, float power) {
        const float d = (most - other_most) * power, share = __builtin_amdgcn_exp2f(d);
        weighted = fmaf(sum, fmaxf(d, kFar), weighted) * share;
        sum *= share;
        most = other_most;
    }
    __device__ __forceinline__ void join(Sums other, float power) {
        const float top = fmaxf(most, other.most);
        bring_to(top, power), other.bring_to(top, power);
        sum += other.sum, weighted += other.weighted;
    }
    template <int N>
    __device__ __forceinline__ Sums of_lane_xor(int lane) const {
        Sums s;
        s.most = lane_xor<N>(most, lane), s.sum = lane_xor<N>(sum, lane), s.weighted = lane_xor<N>(weighted, lane);
        return s;
    }
    // over the wave, in every lane
    __device__ __forceinline__ void join_lanes(float power, int lane) {
        join(of_lane_xor<1>(lane), power), join(of_lane_xor<2>(lane), power), join(of_lane_xor<4>(lane), power);
        join(of_lane_xor<8>(lane), power), join(of_lane_xor<16>(lane), power), join(of_lane_xor<32>(lane), power);
    }
};

// W: keys that the list has room for, 16, 32 or 64; 0: there is none.
// CUT: rows are.  Where they are not there are many, and registers for eight waves a SIMD bring the workgroups of 2048 rows onto
// the card at once (2048 rows of 32000, five alternatives: 76 -> 63 us, twenty: 80 -> 69; none, with nothing left of the
// parts: 52 -> 49); where they are, that gains nothing and costs a few spilled registers (64 rows of 151936, twenty: 24.3 and 26.3).
template <int WAVES, int W, bool CUT>
__global__ void __launch_bounds__(WAVES * JL_WAVE, (WAVES > 1 && !CUT ? 8 : 1)) jl_logprobs_kernel(LogprobsArgs p) {
    constexpr bool TOP = W > 0;
    constexpr int kWide = TOP ? W : JL_WAVE, kLists = JL_WAVE / kWide;   // lists that a register holds
    __shared__ uint2 gathered[WAVES][TOP ? 5 * JL_WAVE : 1];             // value, place
    __shared__ uint64_t lists[WAVES * kWide];
    __shared__ float sums_of[WAVES][3];
    __shared__ uint32_t arrived;
    const int tid = threadIdx.x, lane = tid % JL_WAVE, wave = __builtin_amdgcn_readfirstlane(tid / JL_WAVE);
    const int64_t row = CUT ? blockIdx.x / p.parts : blockIdx.x;
    const int part = CUT ? blockIdx.x % p.parts : 0;
    const float *l = p.logits + row * p.stride;
    const int off = (int)((uintptr_t)l / 4 % 4);              // fours lie on 16-byte boundaries: the first begins this many before the row
    const int fours = (p.n + off + 3) / 4, end = min((part + 1) * p.fours_each, fours);

    uint64_t list = 0;                                        // falling over the first W lanes
    bool full = false;                                        // it has as many keys as are wanted
    float bar = 0.f;                                          // then: the least value that is larger than its last
    int count = 0;                                            // values in `gathered`
    Sums own;

    auto is_whole = [&](int four) { return 4 * four - off >= 0 && 4 * (four + kStepFours) - off <= p.n; };
    auto load = [&](int four, float (&x)[4 * kEach]) {
        const bool whole = is_whole(four);
#pragma unroll
        for (int j = 0; j < kEach; j++) {
            const int first = 4 * (four + j * JL_WAVE + lane) - off;
            if (whole) {
                const float4 v = *(const float4 *)(l + first);
                x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++) x[4 * j + c] = (unsigned)(first + c) < (unsigned)p.n ? l[first + c] : -INFINITY;
            }
        }
    };
    // up to 64 of what is gathered, the last ones, into the list
    auto flush = [&]() {
        wave_fence();
        const int taken = min(count, JL_WAVE);
        count -= taken;
        const uint2 value = gathered[wave][count + min(lane, taken - 1)];
        uint64_t key = lane < taken ? key_of(__uint_as_float(value.x), value.y) : 0;
        if (taken <= kWide) key = sorted<kWide>(key, false, lane);
        else key = largest_of<kWide>(sorted<kWide>(key, kLists > 1 && falls<kWide>(lane), lane), false, lane);
        list = merged<kWide>(list, key, lane);
        const uint32_t last = __builtin_amdgcn_readlane((int)(list >> 32), p.top - 1);
        full = last != 0;
        bar = logit_of(last + 1);                             // (behind infinity: NaN, which nothing reaches)
    };
    auto gather = [&](int four, const float (&x)[4 * kEach], float most) {
        const bool whole = is_whole(four);
        int passing = 0;
        if (full) {
#pragma unroll
            for (int i = 0; i < 4 * kEach; i++) passing += __popcll(__ballot(x[i] >= bar));
        }
        float least = bar;
        if (!full || passing > JL_WAVE) {
            // (one that is wanted itself; without one, where NaN are many, any)
            const uint32_t last = __builtin_amdgcn_readlane((int)sorted<JL_WAVE>(order_of(most), false, lane), JL_WAVE - p.top);
            const float of_lanes = last ? logit_of(last) : -INFINITY;
            least = full ? fmaxf(bar, of_lanes) : of_lanes;
        }
#pragma unroll
        for (int j = 0; j < kEach; j++) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t at = 4 * (four + j * JL_WAVE + lane) - off + c;
                const bool wanted = x[4 * j + c] >= least && (whole || at < (uint32_t)p.n);
                const uint64_t mask = __ballot(wanted);
                if (mask == 0) continue;
                if (wanted) gathered[wave][count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = make_uint2(__float_as_uint(x[4 * j + c]), at);
                count += __popcll(mask);
            }
            if (count >= JL_WAVE) {
                while (count >= JL_WAVE) flush();
                if (full) least = fmaxf(least, bar);          // (what comes next lies behind)
            }
        }
        // (at once where the list is not full: all that is behind it would pass)
        while (!full && count > 0) flush();
    };

    float x[4 * kEach];
    int four = part * p.fours_each + wave * kStepFours;
    if (four < end) load(four, x);
    while (four < end) {
        float next[4 * kEach];
        const int next_four = four + WAVES * kStepFours;
        if (next_four < end) load(next_four, next);
        float most = x[0];
#pragma unroll
        for (int i = 1; i < 4 * kEach; i++) most = fmaxf(most, x[i]);
        if constexpr (TOP)
            if (!full || __any(most >= bar)) gather(four, x, most);
        own.bring_to(fmaxf(own.most, capped(p, most)), p.power);
        float least = x[0];
#pragma unroll
        for (int i = 1; i < 4 * kEach; i++) least = fminf(least, x[i]);
        // (one form of tanh where all of a step's are within its reach)
        const float size = fmaxf(most, -least);
        if (p.cap > 0.f && !__any(!(size <= p.cap_near))) {
#pragma unroll
            for (int i = 0; i < 4 * kEach; i++) {
                const float z = x[i] * x[i];
                const float over = fmaf(z, fmaf(z, p.near_over[1], p.near_over[0]), 1.f);
                const float under = fmaf(z, fmaf(z, p.near_under[1], p.near_under[0]), 1.f);
                x[i] *= over * __builtin_amdgcn_rcpf(under);
            }
        } else if (p.cap > 0.f && !__any(!(size <= p.cap_middle))) {
#pragma unroll
            for (int i = 0; i < 4 * kEach; i++) {
                const float z = x[i] * x[i];
                const float over = fmaf(z, fmaf(z, fmaf(z, p.over[2], p.over[1]), p.over[0]), 1.f);
                const float under = fmaf(z, fmaf(z, fmaf(z, p.under[2], p.under[1]), p.under[0]), 1.f);
                x[i] *= over * __builtin_amdgcn_rcpf(under);
            }
        } else if (p.cap > 0.f) {
#pragma unroll
            for (int i = 0; i < 4 * kEach; i++) x[i] = capped(p, x[i]);
        }
#pragma unroll
        for (int i = 0; i < 4 * kEach; i++) {
            const float a = (x[i] - own.most) * p.power, e = __builtin_amdgcn_exp2f(a);
            own.sum += e;
            own.weighted = fmaf(e, fmaxf(a, kFar), own.weighted);
        }
#pragma unroll
        for (int i = 0; i < 4 * kEach; i++) x[i] = next[i];
        four = next_four;
    }
    if constexpr (TOP)
        while (count > 0) flush();
    own.join_lanes(p.power, lane);

    // the lists that `from` says where they lie, `lists_left` of them, into `list`: kLists at a time, falling and rising in turn
    auto join_lists = [&](int lists_there, auto key_at) {
        list = 0;
#pragma unroll
        for (int j = 0; j < (kMostParts / WAVES + kLists - 1) / kLists; j++) {
            const int first = j * kLists, which = first + lane / kWide;
            if (first >= lists_there) break;
            const uint64_t key = which < lists_there ? key_at(which, j, falls<kWide>(lane) && kLists > 1 ? lane % kWide : kWide - 1 - lane % kWide) : 0;
            list = merged<kWide>(list, largest_of<kWide>(key, false, lane), lane);
        }
    };
    // the waves' parts into the first one's
    auto join_waves = [&]() {
        if constexpr (WAVES > 1) {
            if (lane == 0) sums_of[wave][0] = own.most, sums_of[wave][1] = own.sum, sums_of[wave][2] = own.weighted;
            if constexpr (TOP)
                if (lane < kWide) lists[wave * kWide + lane] = list;
            __syncthreads();
            if (wave == 0) {
                for (int w = 1; w < WAVES; w++) own.join(Sums{sums_of[w][0], sums_of[w][1], sums_of[w][2]}, p.power);
                if constexpr (TOP) join_lists(WAVES, [&](int which, int, int i) { return lists[which * kWide + i]; });
            }
        }
    };
    join_waves();
    if constexpr (CUT) {
        if (wave == 0) {
            Part *to = p.part + row * p.parts + part;
            if constexpr (TOP)
                if (lane < kWide) __hip_atomic_store(&to->keys[lane], list, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (lane < 3) __hip_atomic_store(&to->most + lane, lane == 0 ? own.most : lane == 1 ? own.sum : own.weighted, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores have arrived
            if (lane == 0) {
                const uint32_t before = __hip_atomic_fetch_add(p.arrived + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
                if (before == (uint32_t)p.parts) __hip_atomic_store(p.arrived + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                arrived = before;
            }
        }
        __syncthreads();
        if (arrived != (uint32_t)p.parts) return;
        // a wave has the parts from `first` on; a lane the sums of one
        const Part *from = p.part + row * p.parts;
        const int each = (p.parts + WAVES - 1) / WAVES, first = wave * each, mine = max(min(each, p.parts - first), 0);
        constexpr int kLoads = (kMostParts / WAVES + kLists - 1) / kLists;
        uint64_t keys[kLoads];
        if constexpr (TOP) {
#pragma unroll
            for (int j = 0; j < kLoads; j++) {
                const int which = j * kLists + lane / kWide, i = falls<kWide>(lane) && kLists > 1 ? lane % kWide : kWide - 1 - lane % kWide;
                keys[j] = which < mine ? __hip_atomic_load(&from[first + which].keys[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
            }
        }
        own = Sums();
        if (lane < mine) {
            own.most = __hip_atomic_load(&from[first + lane].most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            own.sum = __hip_atomic_load(&from[first + lane].sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            own.weighted = __hip_atomic_load(&from[first + lane].weighted, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if constexpr (TOP) join_lists(mine, [&](int, int j, int) { return keys[j]; });
        own.join_lanes(p.power, lane);
        join_waves();
    }
    if (wave != 0) return;

    const float log_sum = logf(own.sum);
    auto logprob = [&](float logit) { return own.sum == 0.f ? -INFINITY : fmaf(capped(p, logit) - own.most, p.scale, -log_sum); };
    if (lane == 0 && p.entropy) p.entropy[row] = own.sum == 0.f ? 0.f : fmaf(own.weighted / own.sum, -kLn2, log_sum);
    for (int i = lane; i < p.tokens_per_row; i += JL_WAVE) {
        const int token = p.tokens[row * p.tokens_per_row + i];
        p.logprobs[row * p.tokens_per_row + i] = (unsigned)token < (unsigned)p.n ? logprob(l[token]) : 0.f;
    }
    if constexpr (TOP) {
        if (lane < p.top) {
            const bool is = list >> 32 != 0;
            p.top_tokens[row * p.top + lane] = is ? (int)~(uint32_t)list : -1;
            p.top_logprobs[row * p.top + lane] = is ? logprob(logit_of((uint32_t)(list >> 32))) : -INFINITY;
        }
    }
}

constexpr size_t kArrivedBytes = kPartsRows * sizeof(uint32_t);
constexpr size_t kWorkspaceBytes = kArrivedBytes + (size_t)kGroups * sizeof(Part);

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

template <int WAVES, bool CUT>
void launch(const LogprobsArgs &a, int64_t rows, hipStream_t stream) {
    const dim3 grid((unsigned)(rows * a.parts)), block(WAVES * JL_WAVE);
    if (a.top > 32) hipLaunchKernelGGL((jl_logprobs_kernel<WAVES, 64, CUT>), grid, block, 0, stream, a);
    else if (a.top > 16) hipLaunchKernelGGL((jl_logprobs_kernel<WAVES, 32, CUT>), grid, block, 0, stream, a);
    else if (a.top > 0) hipLaunchKernelGGL((jl_logprobs_kernel<WAVES, 16, CUT>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((jl_logprobs_kernel<WAVES, 0, CUT>), grid, block, 0, stream, a);
}

}  // namespace

extern "C" {

size_t jl_logprobs_workspace_bytes(int64_t n, int top) {
    if (n <= 0 || n > kMostLogits || top < 0 || top > kMostTop) return 0;
    return kWorkspaceBytes;
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
    // (a launch has fewer than 2^32 threads along a side)
    JL_REQUIRE(rows >= 0 && rows < 1 << 24, "jl_logprobs: %lld rows (fewer than 2^24)", (long long)rows);
    JL_REQUIRE(n > 0 && n <= kMostLogits, "jl_logprobs: rows of %lld logits (1 ... 2^30)", (long long)n);
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
    // (of a cap whose sixth power is a number and whose square's products are: else each logit on its own)
    const double y = cap >= 1e-5f && cap <= 1e5f ? 1. / ((double)cap * cap) : 0.;
    a.cap_middle = y > 0. ? kTanhMiddle * cap : 0.f;
    a.over[0] = (float)(17325. / 135135. * y), a.over[1] = (float)(378. / 135135. * y * y), a.over[2] = (float)(y * y * y / 135135.);
    a.under[0] = (float)(62370. / 135135. * y), a.under[1] = (float)(3150. / 135135. * y * y), a.under[2] = (float)(28. / 135135. * y * y * y);
    a.cap_near = y > 0. ? cap : 0.f;
    a.near_over[0] = (float)(105. / 945. * y), a.near_over[1] = (float)(y * y / 945.);
    a.near_under[0] = (float)(420. / 945. * y), a.near_under[1] = (float)(15. / 945. * y * y);
    a.tokens = tokens, a.tokens_per_row = (int)tokens_per_row, a.logprobs = logprobs, a.entropy = entropy;
    a.top = top, a.top_tokens = top_tokens, a.top_logprobs = top_logprobs;
    a.power = scale * kLog2e;
    a.arrived = (uint32_t *)workspace, a.part = (Part *)((uint8_t *)workspace + kArrivedBytes);
    const int waves = n <= kShortRow ? 1 : 4;
    const int64_t steps = ((n + 3 + 3) / 4 + waves * kStepFours - 1) / (waves * kStepFours);   // of a workgroup, in a row that begins between two fours
    a.parts = waves == 1 ? 1 : (int)std::max<int64_t>(std::min<int64_t>({steps, kMostParts, kGroups / rows}), 1);
    a.fours_each = (int)((steps + a.parts - 1) / a.parts) * waves * kStepFours;
    waves == 1 ? launch<1, false>(a, rows, ctx->stream) : a.parts == 1 ? launch<4, false>(a, rows, ctx->stream) : launch<4, true>(a, rows, ctx->stream);
    JL_HIP(hipGetLastError());
    return JL_OK;
}

}  // extern "C"
