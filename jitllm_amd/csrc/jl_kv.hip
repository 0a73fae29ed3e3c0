// The paged key-value cache: its memory, the pages of a step (jl_kv_plan), and what is written to and read from
// pages (jl_kv_append, jl_kv_read).  The attention over it is in jl_attention.hip.
#include <algorithm>
#include <climits>
#include <new>
#include <type_traits>

#include "jl_kv.h"

namespace {

// ---- jl_kv_plan ----------------------------------------------------------------------------------

constexpr int kPlanMaxRequests = 8192, kPlanMaxRows = 1 << 17;
// Workgroups of a launch: one for each 512 rows, or 64 requests, begun, so that a step with prompts in it is one element of
// its list a thread (64 requests, 512 rows: 5.6 us with one workgroup, 4.8 with two; 512, 8192 rows and pages short: 18.3,
// 7.6 with 8, 5.1 with 17; 4096 and 65 536: 125, 14 with 64, 9.4 with 128).
constexpr int kPlanRowsEach = 512, kPlanRequestsEach = 64, kPlanMostGroups = 128;
// Where lengths are past or free_out is free_in, several workgroups need a second launch, for those two: one workgroup does
// up to this many rows (512 requests that all decode: 3.9 us with one workgroup, 7.0 with two launches; 4096 of them in
// 4096 rows 9.6 and 12.1, in 65 536 rows 17.4 and 12.3, with prompts 125 and 14).
constexpr int kPlanRowsInPlace = 4096;

struct PlanArgs {
    const int32_t *past, *fresh, *free_in;
    int32_t *ring, *free_out, *table, *lengths, *row_starts, *slots, *positions, *row_requests;
    int requests, pages, page_shift, table_stride, max_rows, parts;
};

// Inclusive sum over a wave's lanes: within rows of sixteen, then rows' last lanes handed on.
__device__ __forceinline__ int wave_sum_through(int v) {
#define JL_ADD_DPP(CONTROL, ROWS) v += __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xF, false)
    JL_ADD_DPP(0x111, 0xF);   // row_shr 1, 2, 4, 8
    JL_ADD_DPP(0x112, 0xF);
    JL_ADD_DPP(0x114, 0xF);
    JL_ADD_DPP(0x118, 0xF);
    JL_ADD_DPP(0x142, 0xA);   // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    JL_ADD_DPP(0x143, 0xC);
#undef JL_ADD_DPP
    return v;
}

// The sum of `v` over the threads before this one, and over all; `sums` [waves] in LDS, one per call.
template <int THREADS>
__device__ __forceinline__ int sum_before(int v, int &total, int *sums) {
    const int lane = threadIdx.x % JL_WAVE, wave = threadIdx.x / JL_WAVE;
    const int through = wave_sum_through(v);
    if (lane == JL_WAVE - 1) sums[wave] = through;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / JL_WAVE; w++) {
        if (w < wave) before += sums[w];
        total += sums[w];
    }
    return before + through - v;
}

// The first of n ascending sums that is larger than x[j], for K numbers side by side; `most`: the smallest power of two
// above n.  (Their steps wait for LDS together.)
template <int K>
__device__ __forceinline__ void first_above(const int *const (&through)[K], int n, int most, const int (&x)[K], int (&at)[K]) {
#pragma unroll
    for (int j = 0; j < K; j++) at[j] = 0;
    for (int step = most >> 1; step > 0; step >>= 1) {
#pragma unroll
        for (int j = 0; j < K; j++) {
            const int to = at[j] + step;
            if (to <= n && through[j][to - 1] <= x[j]) at[j] = to;
        }
    }
}
__device__ __forceinline__ int power_above(int n) { return n > 0 ? 2 << (31 - __clz(n)) : 1; }

__device__ __forceinline__ int wrapped(int64_t at, int pages) { return (int)(at < pages ? at : at - pages); }   // 0 <= at < 2 pages

__device__ __forceinline__ int slot_in(const PlanArgs &p, int page, int position) {
    return (unsigned)page < (unsigned)p.pages ? (page << p.page_shift) + (position & ((1 << p.page_shift) - 1)) : -1;
}

// A thread's ITEMS consecutive elements of an array of n: four at a time where there are four (0 behind the last one).
typedef int int4_of_ints __attribute__((ext_vector_type(4), aligned(4)));
template <int ITEMS>
__device__ __forceinline__ void load_items(const int32_t *from, int n, int (&to)[ITEMS]) {
    constexpr int W = ITEMS % 4 == 0 ? 4 : 1;
#pragma unroll
    for (int j = 0; j < ITEMS; j += W) {
        const int at = (int)threadIdx.x * ITEMS + j;
        if constexpr (W == 4) {
            if (at + 4 <= n) {
                const int4_of_ints four = *(const int4_of_ints *)(from + at);
#pragma unroll
                for (int i = 0; i < 4; i++) to[j + i] = four[i];
                continue;
            }
        }
#pragma unroll
        for (int i = 0; i < W; i++) to[j + i] = at + i < n ? from[at + i] : 0;
    }
}
template <int ITEMS>
__device__ __forceinline__ void store_items(int32_t *to, int n, const int (&from)[ITEMS]) {
#pragma unroll
    for (int j = 0; j < ITEMS; j++)
        if ((int)threadIdx.x * ITEMS + j < n) to[(int)threadIdx.x * ITEMS + j] = from[j];
}

// What a launch writes: everything but lengths and free_out, those two, or all.
constexpr int kPlanMoves = 1, kPlanLengths = 2;

// ITEMS consecutive requests a thread.  Sums over the requests give each its rows and pages; what a request has many
// of -- rows of a prompt, pages of one that begins or ends -- is dealt to all threads of all workgroups alike, each
// finding its request by bisection in LDS.  Every workgroup takes the sums over all requests for itself: they come out
// of the caches, and nobody waits for anybody.  Latency: of the lengths' loads, two sums over the workgroup, and the
// loads of page numbers that hang on them.
template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) jl_kv_plan_kernel(PlanArgs p) {
    extern __shared__ int lds[];
    int *rows_through = lds, *taken_through = lds + p.requests, *back_through = lds + 2 * p.requests, *first_position = lds + 3 * p.requests;
    __shared__ int sums[3][THREADS / JL_WAVE], granted_pages, most_rows;
    const int tid = threadIdx.x, page = 1 << p.page_shift;
    const bool moves = p.parts & kPlanMoves, its_lengths = p.parts & kPlanLengths;
    // the workgroup that writes what this wave's requests have one of
    const bool mine = min((unsigned)tid / JL_WAVE, gridDim.x - 1) == blockIdx.x;
    if (tid == 0) granted_pages = most_rows = 0;
    int head = p.free_in[0], count = p.free_in[1];
    if (head < 0 || head >= p.pages || count < 0 || count > p.pages) head = count = 0;
    const int table_tokens = (int)min((int64_t)p.table_stride << p.page_shift, (int64_t)INT_MAX);   // positions are int32
    int past[ITEMS], fresh[ITEMS], wanted[ITEMS], need[ITEMS], back[ITEMS];
    load_items(p.past, p.requests, past), load_items(p.fresh, p.requests, fresh);
    int rows = 0;
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        wanted[j] = min(max(fresh[j], 0), p.max_rows + 1);
        rows += wanted[j];
    }
    int all_rows, all_need, all_back;
    int row = sum_before<THREADS>(rows, all_rows, sums[0]);
    // whether its rows fit decides whether a request asks for pages
    int needs = 0, backs = 0, at = row;
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        at += wanted[j];
        const bool held = past[j] >= 0 && past[j] <= table_tokens;
        const int had = held ? (int)(((int64_t)past[j] + page - 1) >> p.page_shift) : 0;
        const bool fits = held && wanted[j] == max(fresh[j], 0) && at <= p.max_rows && (int64_t)past[j] + wanted[j] <= table_tokens;
        need[j] = fits ? (int)(((int64_t)past[j] + wanted[j] + page - 1) >> p.page_shift) - had : -1;    // -1: does not fit
        back[j] = fresh[j] < 0 ? had : 0;
        needs += max(need[j], 0), backs += back[j];
    }
    int asked = sum_before<THREADS>(needs, all_need, sums[1]);
    int returned = sum_before<THREADS>(backs, all_back, sums[2]);
    int granted_through = 0, widest = 0;
    int first_row[ITEMS], first_at[ITEMS], first_page[ITEMS], lengths[ITEMS], starts[ITEMS];   // (row -1: none)
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        const int r = tid * ITEMS + j;
        const int take = max(need[j], 0), had = need[j] >= 0 ? (int)(((int64_t)past[j] + page - 1) >> p.page_shift) : 0;
        asked += take, returned += back[j];
        const bool granted = need[j] >= 0 && wanted[j] > 0 && (take == 0 || asked <= count);
        if (granted && take > 0) granted_through = asked;
        widest = max(widest, wanted[j]);
        if (r < p.requests) {
            rows_through[r] = row + wanted[j];
            taken_through[r] = granted ? asked : min(asked, count);      // (nothing behind the last one granted is taken)
            back_through[r] = returned;
            first_position[r] = granted ? past[j] : -1;
        }
        lengths[j] = fresh[j] < 0 ? 0 : granted ? past[j] + wanted[j] : past[j];
        starts[j] = min(row + wanted[j], p.max_rows);
        // its first row (others are in the list below): the loads of their pages are under way together
        first_row[j] = mine && moves && wanted[j] > 0 && row < p.max_rows ? row : -1;
        first_at[j] = granted ? past[j] : -1, first_page[j] = -1;
        if (first_row[j] >= 0 && granted) {
            const int b = past[j] >> p.page_shift;
            first_page[j] = b < had ? p.table[(int64_t)r * p.table_stride + b] : p.ring[wrapped((int64_t)head + asked - take + b - had, p.pages)];
        }
        row += wanted[j];
    }
    if (granted_through > 0) atomicMax(&granted_pages, granted_through);
    if (widest > 1) atomicMax(&most_rows, widest);
    __syncthreads();
    const int taken = granted_pages, put_back = min(all_back, p.pages - count);
    if (its_lengths) {
        if (mine) store_items(p.lengths, p.requests, lengths);
        if (tid == 0 && blockIdx.x == 0) {
            p.free_out[0] = wrapped((int64_t)head + taken, p.pages);
            p.free_out[1] = count - taken + put_back;
        }
    }
    if (!moves) return;
    // Everything that is moved is one list -- pages taken, pages returned, rows -- dealt to the threads: all searches run
    // together, and then all loads.
    const int most = power_above(p.requests), behind = wrapped((int64_t)head + count, p.pages);
    const int used = min(all_rows, p.max_rows), rows_listed = most_rows > 1 ? used : 0;
    const int listed = taken + put_back + rows_listed;             // (at most twice 2^27 pages and 2^17 rows)
    const int threads = THREADS * gridDim.x, me = blockIdx.x * THREADS + tid;
    auto move = [&](auto batch, int base) {
        constexpr int K = decltype(batch)::value;
        int kind[K], i[K], r[K], of[K], position[K], into[K];
        const int *through[K];
#pragma unroll
        for (int j = 0; j < K; j++) {
            const int e = min(base + j * threads + me, listed - 1);
            kind[j] = e < taken ? 0 : e < taken + put_back ? 1 : 2;
            i[j] = e - (kind[j] == 0 ? 0 : kind[j] == 1 ? taken : taken + put_back);
            through[j] = kind[j] == 0 ? taken_through : kind[j] == 1 ? back_through : rows_through;
        }
        first_above(through, p.requests, most, i, r);
#pragma unroll
        for (int j = 0; j < K; j++) {
            const int first = first_position[r[j]];
            const int had = (int)(((int64_t)first + page - 1) >> p.page_shift);
            int32_t *row_of_table = p.table + (int64_t)r[j] * p.table_stride;
            const int32_t *from;
            into[j] = i[j] - (r[j] > 0 ? through[j][r[j] - 1] : 0);
            if (kind[j] == 0) {
                from = p.ring + wrapped((int64_t)head + i[j], p.pages);
                position[j] = had + into[j];                  // the entry that it becomes
            } else if (kind[j] == 1) {
                from = row_of_table + into[j];
                position[j] = 0;
            } else {
                position[j] = first < 0 ? -1 : first + into[j];
                const int b = max(position[j], 0) >> p.page_shift;
                from = b < had ? row_of_table + b : p.ring + wrapped((int64_t)head + (r[j] > 0 ? taken_through[r[j] - 1] : 0) + b - had, p.pages);
            }
            of[j] = kind[j] == 2 && first < 0 ? -1 : *from;
        }
#pragma unroll
        for (int j = 0; j < K; j++) {
            if (base + j * threads + me >= listed) continue;
            if (kind[j] == 0) {
                p.table[(int64_t)r[j] * p.table_stride + position[j]] = of[j];
            } else if (kind[j] == 1) {
                // (places that no page is taken from: together with those they are at most the ring's)
                p.ring[wrapped((int64_t)behind + i[j], p.pages)] = of[j];
            } else if (into[j] > 0) {
                p.row_requests[i[j]] = r[j];
                p.positions[i[j]] = position[j];
                p.slots[i[j]] = slot_in(p, of[j], position[j]);
            }
        }
    };
    int base = 0;
    for (; listed - base > threads; base += 4 * threads) move(std::integral_constant<int, 4>{}, base);
    if (listed > base) move(std::integral_constant<int, 1>{}, base);
    for (int i = used + me; i < p.max_rows; i += threads) p.slots[i] = p.positions[i] = p.row_requests[i] = -1;
    if (mine) store_items(p.row_starts + 1, p.requests, starts);
    if (tid == 0 && blockIdx.x == 0) p.row_starts[0] = 0;
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        if (first_row[j] < 0) continue;
        p.row_requests[first_row[j]] = tid * ITEMS + j;
        p.positions[first_row[j]] = first_at[j];
        p.slots[first_row[j]] = slot_in(p, first_page[j], first_at[j]);
    }
}

template <int THREADS, int ITEMS>
int launch_plan(jl_context *ctx, PlanArgs p) {
    const int lds = std::max(4 * p.requests * (int)sizeof(int), 16);
    if (lds > 60 * 1024) {
        static jl_lds_limit_flags raised;
        const int st = jl_raise_lds_limit(raised, ctx->device, (const void *)jl_kv_plan_kernel<THREADS, ITEMS>, 4 * THREADS * ITEMS * (int)sizeof(int));
        if (st != JL_OK) return st;
    }
    const bool in_place = p.lengths == p.past || p.free_out == p.free_in;
    const int groups = in_place && p.max_rows <= kPlanRowsInPlace
                           ? 1
                           : std::min(std::max(p.max_rows / kPlanRowsEach, (p.requests - 1) / kPlanRequestsEach) + 1, kPlanMostGroups);
    // (several workgroups: none may write what another one has yet to read)
    const bool two = in_place && groups > 1;
    p.parts = two ? kPlanMoves : kPlanMoves | kPlanLengths;
    hipLaunchKernelGGL((jl_kv_plan_kernel<THREADS, ITEMS>), dim3((unsigned)groups), dim3(THREADS), lds, ctx->stream, p);
    JL_HIP(hipGetLastError());
    if (two) {
        p.parts = kPlanLengths;
        hipLaunchKernelGGL((jl_kv_plan_kernel<THREADS, ITEMS>), dim3(1), dim3(THREADS), lds, ctx->stream, p);
        JL_HIP(hipGetLastError());
    }
    return JL_OK;
}

// ---- jl_kv_append --------------------------------------------------------------------------------

constexpr int kAppendThreads = 256;
constexpr int kAppendPer = 2;   // heads a thread has (2048 tokens of 48 heads of 128: 18.8 us with one, 17.8 with two, 18.2 with four)

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
};

// (cosine, sine) of a number of whole turns, in double precision: whole turns and quarters come off exactly, and the Taylor
// series of what is left (an eighth of a turn at most, 0.79 radians) end where a term is below 2^-45.
__device__ __forceinline__ double2 cos_sin_of_turns(double turns) {
    const double part = turns - rint(turns), quarters = rint(4.0 * part);
    const double x = (part - 0.25 * quarters) * 6.283185307179586477, y = x * x;
    const double s = x * (1 + y * (-1.0 / 6 + y * (1.0 / 120 + y * (-1.0 / 5040 + y * (1.0 / 362880 + y * (-1.0 / 39916800 + y * (1.0 / 6227020800.0)))))));
    const double c = 1 + y * (-0.5 + y * (1.0 / 24 + y * (-1.0 / 720 + y * (1.0 / 40320 + y * (-1.0 / 3628800 + y * (1.0 / 479001600 + y * (-1.0 / 87178291200.0)))))));
    const int n = (int)quarters & 3;
    return make_double2(n == 0 ? c : n == 1 ? -s : n == 2 ? -c : s, n == 0 ? s : n == 1 ? c : n == 2 ? -s : -c);
}

// LANES consecutive lanes have a head, eight values each (those past head_dim / 8 idle); a workgroup has kAppendPer times
// 256 / LANES of a token's q, k and v heads, and all their loads are on their way before anything else is done.
// Bound: the bytes.  The angles' cosines and sines are worked out once per workgroup, in LDS, while the loads come in.
// Sums and products between the loads and the rounding to fp32 are in double precision, which the bytes hide; what the cache
// keeps is rounded from that fp32 value.
template <int TYPE, int LANES, bool HALVES>
__global__ void __launch_bounds__(kAppendThreads) jl_kv_append_kernel(AppendArgs p) {
    __shared__ double2 turn[128];   // (cos, sin) of the token's pairs
    constexpr bool kBlocks = TYPE != JL_KV_F16;
    __shared__ float turned[kBlocks && HALVES ? kAppendThreads / LANES : 1][kBlocks && HALVES ? 8 * LANES : 4];
    const int row = blockIdx.x, tid = threadIdx.x;
    const int position = p.positions[row];
    if (position < 0) return;
    const int slot = p.slots[row];
    const int kv_heads = p.cache.kv_heads, units = p.heads + 2 * kv_heads;
    const int first_unit = blockIdx.y * (kAppendPer * (kAppendThreads / LANES)) + tid / LANES, chunk = tid % LANES;
    const bool in_head = chunk < p.head_dim / 8, turns = 8 * chunk < p.rotated;
    // A lane's eight values are two fours: consecutive ones, or (halves) four and those they turn with.
    const int at0 = HALVES && turns ? 4 * chunk : 8 * chunk, at1 = HALVES && turns ? p.rotated / 2 + 4 * chunk : 8 * chunk + 4;
    float4 own[kAppendPer][2];
#pragma unroll
    for (int j = 0; j < kAppendPer; j++) {
        const int unit = first_unit + j * (kAppendThreads / LANES);
        if (unit < units && in_head) {
            const float *x = unit < p.heads              ? p.q + row * p.ldq + unit * p.head_dim
                             : unit < p.heads + kv_heads ? p.k + row * p.ldk + (unit - p.heads) * p.head_dim
                                                         : p.v + row * p.ldv + (unit - p.heads - kv_heads) * p.head_dim;
            own[j][0] = *(const float4 *)(x + at0), own[j][1] = *(const float4 *)(x + at1);
        }
    }
    for (int i = tid; i < p.rotated / 2; i += kAppendThreads)
        turn[i] = cos_sin_of_turns((double)position * p.frequencies[i] * 0.15915494309189533577);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kAppendPer; j++) {
        const int unit = first_unit + j * (kAppendThreads / LANES);
        if (unit >= units) return;                            // (a head's lanes together)
        const bool is_q = unit < p.heads, is_v = unit >= p.heads + kv_heads;
        const float *norm = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
        float a[8];
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = in_head ? (&own[j][i / 4].x)[i % 4] : 0.f;
        if (!is_v && (norm || p.rotated > 0)) {
            double x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = a[i];
            if (norm) {
                double ss = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fma(x[i], x[i], ss);
#pragma unroll
                for (int off = LANES / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, JL_WAVE);
                const double scale = 1 / sqrt(ss / p.head_dim + p.eps);
                if (in_head) {
                    const float4 w[2] = {*(const float4 *)(norm + at0), *(const float4 *)(norm + at1)};
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] *= scale * (&w[i / 4].x)[i % 4];
                }
            }
            if (in_head && turns) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const double2 t = turn[4 * chunk + i];
                    const int m = HALVES ? i : 2 * i, n = HALVES ? i + 4 : 2 * i + 1;
                    const double first = x[m], second = x[n];
                    x[m] = first * t.x - second * t.y;
                    x[n] = first * t.y + second * t.x;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) a[i] = (float)x[i];
        }
        if (is_q) {
            float *out = p.q_out + row * p.ldq_out + unit * p.head_dim;
            if (in_head) {
                *(float4 *)(out + at0) = make_float4(a[0], a[1], a[2], a[3]);
                *(float4 *)(out + at1) = make_float4(a[4], a[5], a[6], a[7]);
            }
            continue;
        }
        if (slot < 0 || (slot >> p.cache.page_shift) >= p.cache.pages) continue;
        const int page = slot >> p.cache.page_shift, token = slot & ((1 << p.cache.page_shift) - 1);
        uint8_t *part = p.cache.k + (is_v ? p.cache.v_offset : 0) +
                        ((int64_t)page * kv_heads + (is_v ? unit - p.heads - kv_heads : unit - p.heads)) * p.cache.part_bytes;
        if constexpr (!kBlocks) {
            _Float16 *to = (_Float16 *)part + token * p.head_dim;
            const jl_half4v low = {(_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3]};
            const jl_half4v high = {(_Float16)a[4], (_Float16)a[5], (_Float16)a[6], (_Float16)a[7]};
            if (in_head) *(jl_half4v *)(to + at0) = low, *(jl_half4v *)(to + at1) = high;
        } else {
            if constexpr (HALVES) {
                // blocks are of consecutive values: through LDS, inside the wave
                float *head = turned[tid / LANES];
                if (in_head) {
                    *(float4 *)(head + at0) = make_float4(a[0], a[1], a[2], a[3]);
                    *(float4 *)(head + at1) = make_float4(a[4], a[5], a[6], a[7]);
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                if (in_head) {
                    const float4 low = *(const float4 *)(head + 8 * chunk), high = *(const float4 *)(head + 8 * chunk + 4);
                    a[0] = low.x, a[1] = low.y, a[2] = low.z, a[3] = low.w, a[4] = high.x, a[5] = high.y, a[6] = high.z, a[7] = high.w;
                }
                __builtin_amdgcn_wave_barrier();
            }
            if constexpr (TYPE == JL_KV_Q4_0) {
                // the value of largest magnitude of the block, four lanes' values, the first of several; NaN is none
                float largest = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) largest = fabsf(a[i]) > fabsf(largest) ? a[i] : largest;
#pragma unroll
                for (int off = 1; off <= 2; off <<= 1) {
                    const float other = __shfl_xor(largest, off, JL_WAVE);
                    const bool takes = fabsf(other) > fabsf(largest) || (fabsf(other) == fabsf(largest) && (chunk & off));
                    largest = takes ? other : largest;
                }
                const _Float16 d16 = (_Float16)fminf(fmaxf(largest * -0.125f, -65504.f), 65504.f);
                const float d = (float)d16;
                uint32_t word = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = d != 0.f && a[i] == a[i] ? fminf(fmaxf(rintf(a[i] / d), -8.f), 7.f) : 0.f;
                    word |= (uint32_t)((int)y + 8) << 4 * i;
                }
                if (in_head) {
                    if (is_v) {
                        uint8_t *at = part + jl_q4_value_at(p.head_dim, token, chunk);
                        *(uint16_t *)at = (uint16_t)word, *(uint16_t *)(at + 8) = (uint16_t)(word >> 16);
                    } else {
                        *(uint32_t *)(part + jl_q4_key_at(p.head_dim, token, chunk)) = word;
                    }
                    if (chunk % 4 == 0) {
                        _Float16 *scales = (_Float16 *)(part + ((int64_t)(p.head_dim / 2) << p.cache.page_shift));
                        scales[((chunk / 4) << p.cache.page_shift) + token] = d16;
                    }
                }
                continue;
            }
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
            if (in_head) {
                *(uint2 *)(part + token * p.head_dim + 8 * chunk) = make_uint2(word[0], word[1]);
                if (chunk % 4 == 0) {
                    _Float16 *scales = (_Float16 *)(part + ((int64_t)p.head_dim << p.cache.page_shift));
                    scales[((chunk / 4) << p.cache.page_shift) + token] = d16;
                }
            }
        }
    }
}

// ---- jl_kv_read ----------------------------------------------------------------------------------

template <int TYPE, bool HALF>
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
        if (slot >= 0 && page < cache.pages) h = jl_kv_load8<TYPE>(part + (which ? cache.v_offset : 0), which, cache.page_shift, head_dim, token, chunk);
        if constexpr (HALF) {
            ((jl_half8 *)out)[at] = h;
        } else {
            ((float4 *)out)[2 * at] = make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
            ((float4 *)out)[2 * at + 1] = make_float4((float)h[4], (float)h[5], (float)h[6], (float)h[7]);
        }
    }
}

int cache_check(const char *who, int kv_type, int64_t pages, int kv_heads, int head_dim, int page_tokens) {
    if (kv_type != JL_KV_F16 && kv_type != JL_KV_Q8_0 && kv_type != JL_KV_Q4_0)
        return jl_fail(JL_ERR_UNSUPPORTED, "%s: no key-value cache of type %d (JL_KV_F16, JL_KV_Q8_0 or JL_KV_Q4_0)", who, kv_type);
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

template <int TYPE, int LANES, bool HALVES>
void launch_append_lanes(const AppendArgs &a, unsigned rows, hipStream_t stream) {
    const int units = a.heads + 2 * a.cache.kv_heads, per = kAppendPer * (kAppendThreads / LANES);
    hipLaunchKernelGGL((jl_kv_append_kernel<TYPE, LANES, HALVES>), dim3(rows, (unsigned)((units + per - 1) / per)), dim3(kAppendThreads), 0, stream, a);
}
template <int TYPE, bool HALVES>
void launch_append(const AppendArgs &a, unsigned rows, hipStream_t stream) {
    if (a.head_dim <= 64) launch_append_lanes<TYPE, 8, HALVES>(a, rows, stream);
    else if (a.head_dim <= 128) launch_append_lanes<TYPE, 16, HALVES>(a, rows, stream);
    else launch_append_lanes<TYPE, 32, HALVES>(a, rows, stream);
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
    if (requests <= 1024) return launch_plan<1024, 1>(ctx, p);
    if (requests <= 4096) return launch_plan<1024, 4>(ctx, p);
    return launch_plan<1024, 8>(ctx, p);
}

int jl_kv_append(jl_context *ctx, jl_kv_cache *cache, const float *q, int heads, int64_t ldq, const float *k,
                 int64_t ldk, const float *v, int64_t ldv, float *q_out, int64_t ldq_out, const int32_t *positions,
                 const int32_t *slots, int64_t rows, const double *frequencies, int rotated, int rope_style,
                 const float *q_norm, const float *k_norm, float eps) {
    JL_REQUIRE(ctx && cache && k && v && positions && slots && (!q || q_out), "jl_kv_append: null argument");
    const int dim = cache->head_dim;
    JL_REQUIRE(cache->ctx->device == ctx->device, "jl_kv_append: the cache lies on device %d, the context's is %d",
               cache->ctx->device, ctx->device);
    // (a launch has fewer than 2^32 threads along a side)
    JL_REQUIRE(rows >= 0 && rows < (1ll << 32) / kAppendThreads, "jl_kv_append: %lld rows (fewer than 2^24)", (long long)rows);
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
    a.heads = q ? heads : 0, a.head_dim = dim, a.rotated = rotated;
    const bool halves = rope_style == JL_ROPE_HALVES && rotated > 0;
    const unsigned n = (unsigned)rows;
    if (cache->type == JL_KV_Q8_0) halves ? launch_append<JL_KV_Q8_0, true>(a, n, ctx->stream) : launch_append<JL_KV_Q8_0, false>(a, n, ctx->stream);
    else if (cache->type == JL_KV_Q4_0) halves ? launch_append<JL_KV_Q4_0, true>(a, n, ctx->stream) : launch_append<JL_KV_Q4_0, false>(a, n, ctx->stream);
    else halves ? launch_append<JL_KV_F16, true>(a, n, ctx->stream) : launch_append<JL_KV_F16, false>(a, n, ctx->stream);
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
    JL_REQUIRE(threads < (1ll << 32) - 256, "jl_kv_read: %lld rows of %d values in one call (fewer than 2^35 values in all)", (long long)rows,
               cache->kv_heads * cache->head_dim);
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
    const JlKvView c = jl_kv_view(cache);
    const int dim = cache->head_dim;
    auto launch = [&](auto type, auto half) {
        hipLaunchKernelGGL((jl_kv_read_kernel<decltype(type)::value, decltype(half)::value>), grid, block, 0, ctx->stream, c, dim, slots, rows, k_out, v_out);
    };
    auto launch_type = [&](auto type) { out_f16 ? launch(type, std::true_type{}) : launch(type, std::false_type{}); };
    if (cache->type == JL_KV_Q8_0) launch_type(std::integral_constant<int, JL_KV_Q8_0>{});
    else if (cache->type == JL_KV_Q4_0) launch_type(std::integral_constant<int, JL_KV_Q4_0>{});
    else launch_type(std::integral_constant<int, JL_KV_F16>{});
    JL_HIP(hipGetLastError());
    return JL_OK;
}

}  // extern "C"
