// jl_kv_attention: attention of one new token a row over its request's pages.
//
// Mathematics.  For a row and a head of k and v, S = K Q^T over tiles of 32 tokens and up to 16 query heads (the heads
// that share k and v), P = 2^(S - m) with a running maximum m, O = O 2^(m_old - m) + V^T P^T, l the sum of P; the result
// is O / l, and two parts (m, l, O) of a row join by the same rule.  scale * log2(e) is folded into q; P, and with it l
// and O, are held 2^13 times as large, so that weights far below the largest keep their precision.
//
// Matrix instructions.  v_mfma_f32_16x16x32_f16 throughout, laid out so that nothing is exchanged between lanes but
// the maximum: S comes out with a query head per lane (lane % 16) and the tokens 4 g ... 4 g + 3 of both 16-token
// halves in the lanes of group g = lane / 16, which is the layout that the second product wants P in if its k index
// runs through the tokens in that order -- and V is simply loaded in that order.  O^T = V^T P^T keeps a query head per
// lane, so the rescaling by 2^(m_old - m) is lane-local too.  k and v go from memory to registers and on into the
// matrix instructions; V is transposed there, eight tokens of a column at a time, by byte permutes.  q and P enter as
// the sum of two binary16 values (22 bits), k and v as they are: the products are exact and everything else fp32.
//
// Bound: the bytes of k and v.  A tile is two matrix instructions per 16 x 32 piece of k and v, 16 flops a byte, a tenth
// of what the matrix units do in the time the bytes take.
//
// Work.  The tiles of all (row, head of k and v, 16 query heads) are one long list, cut into equal spans for the
// launch's workgroups whatever the rows' lengths are; a workgroup's four waves take a span's tiles in turn and
// join in LDS.  A head that a cut goes through leaves its parts in the workspace, and the workgroup that is done last
// with it joins them, in their order whoever that is (nobody waits for anybody).
//
// Rows of one request (a prompt's, a draft's) go through its pages together where there are twice as many rows as
// requests: 16 columns of the matrix instructions are the query heads of one row after the other, each with its own mask.
// Only rows whose ranges touch do, so that no token is read that none of them sees, and in tiles that some of them do not
// see all of, values of v that are not finite are kept from those.
#include <algorithm>
#include <climits>
#include <cmath>

#include "jl_kv.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / JL_WAVE;
constexpr int kMostGroups = 512;          // workgroups of a launch, and spans: two on each of 256 compute units
constexpr int kStart = 4;                 // what beginning a (row, head) pair takes, in tiles
// Parts of a head: 32 at most, up to 64 of 64 tiles and more (8 heads of 4000 tokens: 13.4 and 15.5 us; of 131072: 95.2
// and 93.4).
constexpr uint32_t kParts = 32, kMostParts = 64, kLargePart = 64;
constexpr int kDeviceScope = 16;          // a buffer load's policy: sc1
// Weights are 2^kLift at the running maximum, which may fall behind by 2^kSlack: 2^15 at most, and what binary16 keeps of
// one (2^-25 off, however small it is) is 2^-38 of the largest.
constexpr float kSlack = 2, kLift = 13;
constexpr float kNone = -3.0e38f;         // the running maximum of nothing: finite, so that differences are numbers

constexpr int kHalves = 2, kTile = 16 * kHalves;   // a wave's tile: tokens, in halves of 16

template <bool Q8, int DIM>
struct Shape {
    static constexpr int kPerUnit = DIM == 256 ? 1 : 2;   // workgroups that a compute unit holds at a time
    // Tiles that the whole chip reads (6 TB/s) in the time that a workgroup alone takes for one (half a microsecond).
    static constexpr int kTileBytes = Q8 ? 2 * kTile * (DIM + DIM / 16) : 2 * kTile * DIM * 2;
    static constexpr float kTilesAtOnce = 3.0e6f / kTileBytes;
};

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bfloat8 __attribute__((ext_vector_type(8)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

struct AttentionArgs {
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
    uint32_t *arrived;    // [kMostGroups], all 0 between calls
    float *parts;         // [2 * spans][16 * (DIM + 2)]
    // Rows of one request that go together: a power of two, at most 16 / group; 1: each alone.  (The last argument: among the
    // others it moved some to another load, and every call took 0.1 ... 0.2 us longer.)
    int rows_each;
};

// The tokens [first, end) of its request that a row sees.  A row without a position or a request has [0, -1), which touches no
// other's.
struct Range {
    int first, end, request, members = 1;
    __device__ int tiles() const { return end > first ? (end + kTile - 1) / kTile - first / kTile : 0; }
};
__device__ __forceinline__ Range range_at(const AttentionArgs &p, int position, int request) {
    Range r;
    r.request = request;
    r.end = position >= 0 && r.request >= 0 && r.request < p.requests ? min(position, p.table_tokens - 1) + 1 : -1;
    r.first = p.window > 0 ? max(position - p.window + 1, 0) : 0;
    return r;
}

__device__ __forceinline__ Range range_of(const AttentionArgs &p, int row) {
    return range_at(p, p.positions[row], p.row_requests ? p.row_requests[row] : row);
}

// Rows that go together (SHARED): a run among rows_each rows that begin at a multiple of it, of one request's, each of which
// has tokens in common with the one before it or begins or ends where that one does: what they see together is then one
// range, and no token between two windows is read.  The first of a run has the range of all; the others have nothing.
__device__ __forceinline__ bool goes_on(const Range &before, const Range &r) {
    return before.request == r.request && max(before.first, r.first) <= min(before.end, r.end);
}
__device__ __forceinline__ void join_ranges(Range &r, const Range &next) {
    r.first = min(r.first, next.first), r.end = max(r.end, next.end);
    r.members += next.members;
}
// Of the row in every lane (one behind the last row has nothing); sixteen lanes' first one has a row at such a multiple.
__device__ __forceinline__ Range run_in_lanes(const AttentionArgs &p, Range r, int lane) {
    const int in_block = lane & (p.rows_each - 1);
#define JL_ROW(X, CONTROL) __builtin_amdgcn_update_dpp(0, X, CONTROL, 0xF, 0xF, true)
    const Range before{JL_ROW(r.first, 0x111), JL_ROW(r.end, 0x111), JL_ROW(r.request, 0x111)};   // of the lane before, of sixteen
    const int goes = in_block != 0 && goes_on(before, r);
#define JL_JOIN_FROM(N)                                                                                                        \
    if (N < p.rows_each) {                                                                                                     \
        const Range other{JL_ROW(r.first, 0x100 + N), JL_ROW(r.end, 0x100 + N), 0, JL_ROW(r.members, 0x100 + N)};              \
        const int its = JL_ROW(goes, 0x100 + N);                                                                               \
        if (r.members == N && in_block + N < p.rows_each && its) join_ranges(r, other);                                        \
    }
    JL_JOIN_FROM(1)
    JL_JOIN_FROM(2)
    JL_JOIN_FROM(4)
    JL_JOIN_FROM(8)
#undef JL_JOIN_FROM
#undef JL_ROW
    if (goes) r.end = 0;
    return r;
}
// Calls work(row, range) for the runs that begin at rows begin ... end - 1, in order, until it returns false; `begin` is at
// such a multiple.
template <bool SHARED, typename WORK>
__device__ __forceinline__ void for_runs(const AttentionArgs &p, int begin, int end, WORK work) {
    if constexpr (!SHARED) {
        for (int r = begin; r < end; r++)
            if (!work(r, range_of(p, r))) return;
    } else {
        Range run, before;
        int first_row = -1;
        for (int r = begin; r < end; r += 4) {
            Range four[4];
#pragma unroll
            for (int j = 0; j < 4; j++) four[j] = range_of(p, min(r + j, p.rows - 1));
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (r + j >= end) break;
                const bool goes = first_row >= 0 && ((r + j) & (p.rows_each - 1)) && goes_on(before, four[j]);
                before = four[j];
                if (goes) {
                    join_ranges(run, four[j]);
                    continue;
                }
                if (first_row >= 0 && !work(first_row, run)) return;
                first_row = r + j, run = four[j];
            }
        }
        if (first_row >= 0) work(first_row, run);
    }
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Parts go to the workgroup that joins them through device scope: past the XCD's own second-level cache.
__device__ __forceinline__ void agent_store(float *to, float v) {
    __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_store4(float *to, floatx4 v) {
    uint64_t two[2];
    __builtin_memcpy(two, &v, 16);
    __hip_atomic_store((uint64_t *)to, two[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store((uint64_t *)to + 1, two[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// k and v pass once: loads that do not stay in the caches (512 MB in 16 KB pieces, nothing else done: 90 us with ordinary
// loads, 80 with these).
// Where rows of one request follow each other over the same pages, theirs stay.
template <typename T, bool STAY>
__device__ __forceinline__ T load_at(const uint8_t *base, uint32_t offset) {
    if constexpr (STAY) return *(const T *)(base + offset);
    else return __builtin_nontemporal_load((const T *)(base + offset));
}
__device__ __forceinline__ jl_half2v as_half2(uint32_t x) { return __builtin_bit_cast(jl_half2v, x); }
__device__ __forceinline__ uint32_t as_u32(jl_half2v x) { return __builtin_bit_cast(uint32_t, x); }

// Halves of a word that are binary16 infinities or NaN, all their bits set.
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
    return ((x & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}

// Bytes 0 and 2 of a word, signed, as binary16.  A byte b of 0 ... 255 under 0x64 is the binary16 of 1024 + b, so with the
// sign bit turned over (b = q + 128) a subtraction of 1152 leaves q, exactly.  One bit operation puts both in place; the
// kernel over 8-bit blocks is bound by its vector instructions, and those that permute bytes take twice as long as bit
// operations do (1.9 and 1.05 ns of a SIMD's time).
__device__ __forceinline__ jl_half2v even_bytes(uint32_t x) {
    const jl_half2v bias = {(_Float16)1152.f, (_Float16)1152.f};
    return as_half2((x & 0x00ff00ffu) ^ 0x64806480u) - bias;
}

// A tile's k and v as they lie in memory.  Lane (g, m) = (lane / 16, lane % 16) has, of k, token m of each 16-token half,
// and of v the tokens 4 g + i of each half at a few consecutive elements: head_dim is cut into pieces of 128, 64 and 32,
// and m has 8, 4 or 2 values of a piece.
template <bool Q8, int DIM>
struct Raw;

template <int DIM>
struct Raw<false, DIM> {
    static constexpr int kSteps = DIM / 32;
    static constexpr int kWide = DIM / 128, kMid = DIM % 128 / 64, kThin = DIM % 64 / 32;
    uintx4 k[kHalves][kSteps];
    uintx4 v4[kHalves][4][kWide ? kWide : 1];
    uintx2 v2[kHalves][4];
    uint32_t v1[kHalves][4];
    __device__ static int element(int step, int g) { return 32 * step + 8 * g; }   // first of the eight of k step `step`
    __device__ static constexpr int in_eight(int i) { return i; }                  // ... and their order
    template <bool STAY>
    __device__ void load_k(int half, const uint8_t *part, int in_page, int, int g, int m) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) k[half][s] = load_at<uintx4, STAY>(part, (in_page + m) * (2 * DIM) + 64 * s + 16 * g);
    }
    template <bool STAY>
    __device__ void load_v(int half, const uint8_t *part, int in_page, int, int g, int m) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t row = (in_page + 4 * g + i) * (2 * DIM);
#pragma unroll
            for (int w = 0; w < kWide; w++) v4[half][i][w] = load_at<uintx4, STAY>(part, row + 256 * w + 16 * m);
            if constexpr (kMid) v2[half][i] = load_at<uintx2, STAY>(part, row + 256 * kWide + 8 * m);
            if constexpr (kThin) v1[half][i] = load_at<uint32_t, STAY>(part, row + 256 * kWide + 128 * kMid + 4 * m);
        }
    }
    __device__ jl_half8 k_operand(int half, int step) const { return __builtin_bit_cast(jl_half8, k[half][step]); }
    // masked tokens' values are nothing, whatever lies there
    __device__ void mask_v(const bool (&seen)[kHalves][4]) {
#pragma unroll
        for (int h = 0; h < kHalves; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int w = 0; w < kWide; w++)
#pragma unroll
                    for (int c = 0; c < 4; c++) v4[h][i][w][c] = seen[h][i] ? v4[h][i][w][c] : 0;
                if constexpr (kMid) v2[h][i].x = seen[h][i] ? v2[h][i].x : 0, v2[h][i].y = seen[h][i] ? v2[h][i].y : 0;
                if constexpr (kThin) v1[h][i] = seen[h][i] ? v1[h][i] : 0;
            }
    }
    // whether any value is an infinity or NaN: nothing times it is no number
    __device__ bool any_not_finite() const {
        const jl_half2v nothing = {(_Float16)0.f, (_Float16)0.f};
        jl_half2v sum = nothing;
#pragma unroll
        for (int h = 0; h < kHalves; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int w = 0; w < kWide; w++)
#pragma unroll
                    for (int c = 0; c < 4; c++) sum = __builtin_elementwise_fma(as_half2(v4[h][i][w][c]), nothing, sum);
#pragma unroll
                for (int c = 0; c < 2 * kMid; c++) sum = __builtin_elementwise_fma(as_half2(v2[h][i][c]), nothing, sum);
                if constexpr (kThin) sum = __builtin_elementwise_fma(as_half2(v1[h][i]), nothing, sum);
            }
        return (as_u32(sum) & 0x7fff7fffu) != 0;
    }
    // those that are become 0
    __device__ void drop_not_finite() {
#pragma unroll
        for (int h = 0; h < kHalves; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int w = 0; w < kWide; w++)
#pragma unroll
                    for (int c = 0; c < 4; c++) v4[h][i][w][c] &= ~not_finite(v4[h][i][w][c]);
#pragma unroll
                for (int c = 0; c < 2 * kMid; c++) v2[h][i][c] &= ~not_finite(v2[h][i][c]);
                if constexpr (kThin) v1[h][i] &= ~not_finite(v1[h][i]);
            }
    }
    // eight tokens of the columns that output blocks `block` and `block` + 1 take of this lane
    __device__ void v_operands(int block, jl_half8 (&v)[2]) const {
        uintx4 r[2];
        const int word = block / 2;
#pragma unroll
        for (int pair = 0; pair < 4; pair++) {
            const int h = pair / 2, i = pair % 2 * 2;
            uint32_t a, b;
            if (word < 4 * kWide) a = v4[h][i][word / 4][word % 4], b = v4[h][i + 1][word / 4][word % 4];
            else if (word < 4 * kWide + 2 * kMid) a = v2[h][i][word % 2], b = v2[h][i + 1][word % 2];
            else a = v1[h][i], b = v1[h][i + 1];
            r[0][pair] = __builtin_amdgcn_perm(b, a, 0x05040100u), r[1][pair] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        }
        v[0] = __builtin_bit_cast(jl_half8, r[0]), v[1] = __builtin_bit_cast(jl_half8, r[1]);
    }
};

template <int DIM>
struct Raw<true, DIM> {
    static constexpr int kSteps = DIM / 32, kPairs = DIM / 64, kTail = DIM % 64 / 32;
    static constexpr int kWide = DIM / 128, kMid = DIM % 128 / 64, kThin = DIM % 64 / 32;
    static constexpr int kPieces = kWide + kMid + kThin;
    uintx4 k[kHalves][kPairs];
    uintx2 k_tail[kHalves];
    uint16_t k_scale[kHalves][kPairs + kTail];
    uintx2 v2[kHalves][4][kWide ? kWide : 1];
    uint32_t v1[kHalves][4];
    uint16_t v0[kHalves][4];
    uintx2 v_scale[kHalves][kPieces];
    // (16 consecutive bytes serve two steps: a lane's loads stay 16 bytes wide)
    __device__ static int element(int step, int g) {
        return step < 2 * kPairs ? 64 * (step / 2) + 16 * g + 8 * (step % 2) : 64 * kPairs + 8 * g;
    }
    // (0, 2), (1, 3), (4, 6), (5, 7): the pairs that one operation takes out of a word
    __device__ static constexpr int in_eight(int i) { return i / 4 * 4 + i % 4 / 2 + i % 2 * 2; }
    template <bool STAY>
    __device__ void load_k(int half, const uint8_t *part, int in_page, int page_shift, int g, int m) {
        const uint32_t row = (in_page + m) * DIM, scales = ((uint32_t)DIM << page_shift) + 2 * (in_page + m);
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            k[half][i] = load_at<uintx4, STAY>(part, row + 64 * i + 16 * g);
            k_scale[half][i] = load_at<uint16_t, STAY>(part, scales + ((2 * (2 * i + g / 2)) << page_shift));
        }
        if constexpr (kTail) {
            k_tail[half] = load_at<uintx2, STAY>(part, row + 64 * kPairs + 8 * g);
            k_scale[half][kPairs] = load_at<uint16_t, STAY>(part, scales + ((2 * 2 * kPairs) << page_shift));
        }
    }
    template <bool STAY>
    __device__ void load_v(int half, const uint8_t *part, int in_page, int page_shift, int g, int m) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t row = (in_page + 4 * g + i) * DIM;
#pragma unroll
            for (int w = 0; w < kWide; w++) v2[half][i][w] = load_at<uintx2, STAY>(part, row + 128 * w + 8 * m);
            if constexpr (kMid) v1[half][i] = load_at<uint32_t, STAY>(part, row + 128 * kWide + 4 * m);
            if constexpr (kThin) v0[half][i] = load_at<uint16_t, STAY>(part, row + 128 * kWide + 64 * kMid + 2 * m);
        }
        const uint32_t scales = ((uint32_t)DIM << page_shift) + 2 * (in_page + 4 * g);
#pragma unroll
        for (int w = 0; w < kWide; w++) v_scale[half][w] = load_at<uintx2, STAY>(part, scales + ((2 * (4 * w + m / 4)) << page_shift));
        if constexpr (kMid) v_scale[half][kWide] = load_at<uintx2, STAY>(part, scales + ((2 * (4 * kWide + m / 8)) << page_shift));
        if constexpr (kThin) v_scale[half][kWide + kMid] = load_at<uintx2, STAY>(part, scales + ((2 * (4 * kWide + 2 * kMid)) << page_shift));
    }
    __device__ jl_half8 k_operand(int half, int step) const {
        uint32_t lo, hi;
        uint32_t d;
        if (step < 2 * kPairs) lo = k[half][step / 2][step % 2 * 2], hi = k[half][step / 2][step % 2 * 2 + 1], d = k_scale[half][step / 2];
        else lo = k_tail[half].x, hi = k_tail[half].y, d = k_scale[half][kPairs + kTail - 1];
        const jl_half2v dd = as_half2(d | d << 16);
        return __builtin_bit_cast(jl_half8, uintx4{as_u32(even_bytes(lo) * dd), as_u32(even_bytes(lo >> 8) * dd),
                                                   as_u32(even_bytes(hi) * dd), as_u32(even_bytes(hi >> 8) * dd)});
    }
    // (a byte times a scale of 0; the scale alone can be an infinity or NaN)
    __device__ void mask_v(const bool (&seen)[kHalves][4]) {
#pragma unroll
        for (int h = 0; h < kHalves; h++)
#pragma unroll
            for (int w = 0; w < kPieces; w++)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    v_scale[h][w][c] &= (seen[h][2 * c] ? 0xffffu : 0u) | (seen[h][2 * c + 1] ? 0xffff0000u : 0u);
    }
    // whether any value may be an infinity or NaN: 128 times its scale is one
    __device__ bool any_not_finite() const {
        const jl_half2v nothing = {(_Float16)0.f, (_Float16)0.f}, most = {(_Float16)128.f, (_Float16)128.f};
        jl_half2v sum = nothing;
#pragma unroll
        for (int h = 0; h < kHalves; h++)
#pragma unroll
            for (int w = 0; w < kPieces; w++)
#pragma unroll
                for (int c = 0; c < 2; c++) sum = __builtin_elementwise_fma(as_half2(v_scale[h][w][c]) * most, nothing, sum);
        return (as_u32(sum) & 0x7fff7fffu) != 0;
    }
    // those that are become 0: bytes that a finite scale takes too far, and scales that are not finite
    __device__ void drop_not_finite() {
        auto drop = [](uint32_t x, uint32_t d) {
            const uint32_t even = not_finite(as_u32(even_bytes(x) * as_half2(d))), odd = not_finite(as_u32(even_bytes(x >> 8) * as_half2(d)));
            return x & ~((even & 0x00ff00ffu) | (odd & 0xff00ff00u));
        };
#pragma unroll
        for (int h = 0; h < kHalves; h++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                auto scale = [&](int piece) { return (v_scale[h][piece][i / 2] >> 16 * (i % 2) & 0xffffu) * 0x10001u; };
#pragma unroll
                for (int w = 0; w < kWide; w++)
#pragma unroll
                    for (int c = 0; c < 2; c++) v2[h][i][w][c] = drop(v2[h][i][w][c], scale(w));
                if constexpr (kMid) v1[h][i] = drop(v1[h][i], scale(kWide));
                if constexpr (kThin) v0[h][i] = (uint16_t)drop(v0[h][i], scale(kWide + kMid));
            }
#pragma unroll
            for (int w = 0; w < kPieces; w++)
#pragma unroll
                for (int c = 0; c < 2; c++) v_scale[h][w][c] &= ~not_finite(v_scale[h][w][c]);
        }
    }
    // Operands of two neighbouring blocks: their columns' bytes of two tokens come into one word, and out of it as pairs.
    __device__ void v_operands(int block, jl_half8 (&v)[2]) const {
        uintx4 r[2];
        const int piece = block < 8 * kWide ? block / 8 : block < 8 * kWide + 4 * kMid ? kWide : kWide + kMid;
#pragma unroll
        for (int pair = 0; pair < 4; pair++) {
            const int h = pair / 2, i = pair % 2 * 2;
            uint32_t a, b;
            int byte;
            if (block < 8 * kWide) a = v2[h][i][block / 8][block % 8 / 4], b = v2[h][i + 1][block / 8][block % 8 / 4], byte = block % 4;
            else if (block < 8 * kWide + 4 * kMid) a = v1[h][i], b = v1[h][i + 1], byte = block % 4;
            else a = v0[h][i], b = v0[h][i + 1], byte = 0;
            const uint32_t both = __builtin_amdgcn_perm(b, a, byte == 0 ? 0x05040100u : 0x07060302u);
            const jl_half2v d = as_half2(v_scale[h][piece][i / 2]);
            r[0][pair] = as_u32(even_bytes(both) * d), r[1][pair] = as_u32(even_bytes(both >> 8) * d);
        }
        v[0] = __builtin_bit_cast(jl_half8, r[0]), v[1] = __builtin_bit_cast(jl_half8, r[1]);
    }
};

// The output element that row 4 g + i of output block `block` is: 8, 4 or 2 consecutive blocks are consecutive elements.
template <int DIM>
__device__ __forceinline__ int out_element(int block, int index) {
    constexpr int wide = DIM / 128, mid = DIM % 128 / 64;
    if (block < 8 * wide) return 128 * (block / 8) + 8 * index + block % 8;
    if (block < 8 * wide + 4 * mid) return 128 * wide + 4 * index + block % 4;
    return 128 * wide + 64 * mid + 2 * index + block % 2;
}

__device__ __forceinline__ float over_groups_max(float x) {
    const auto f = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(f[0]), __uint_as_float(f[1]));
    const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float over_groups_sum(float x) {
    const auto f = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(f[0]) + __uint_as_float(f[1]);
    const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

__device__ __forceinline__ void store_out(const AttentionArgs &p, int64_t at, const floatx4 v) {
    if (p.out_f16) *(jl_half4v *)((_Float16 *)p.out + at) = jl_half4v{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
    else *(floatx4 *)((float *)p.out + at) = v;
}

// Units of a head in the list of all work: its tiles, and what beginning it takes.
__device__ __forceinline__ uint32_t units_of(int tiles) { return tiles > 0 ? tiles + kStart : 0; }

// A piece of a workgroup's list: tiles tile ... tile + count - 1 of a row's head, and what the row sees.
struct Piece {
    int row, head, tile, count, tiles;
    int first, end, request, members;
    int unit;         // where the piece begins in its head
    uint32_t left;    // units of the span, this piece's included; 0: no such piece
};

// A head that the workgroup has one of several parts of: those of spans group ... group + parts - 1.
struct Cut {
    int row, members, kv_head, block_of_16, group, parts;
};

// SHARED: rows of one request go through the tiles together, a (row, query head) a column.
template <bool Q8, int DIM, bool SHARED>
__global__ void __launch_bounds__(kThreads, (Shape<Q8, DIM>::kPerUnit)) jl_kv_attention_kernel(AttentionArgs p) {
    constexpr int kSteps = DIM / 32, kBlocks = DIM / 16;
    constexpr int kRound = DIM == 256 ? 128 : DIM;            // elements that are joined at a time: 64 KB of LDS at most
    constexpr int kStride = kRound + 4;                       // (four floats on: rows start on other banks)
    constexpr int kSlot = 16 * (DIM + 2);
    __shared__ float joined[kWaves][16][kStride];
    __shared__ float joined_max[kWaves][16], joined_sum[kWaves][16];
    __shared__ uint32_t scan[kWaves], scan_longest[kWaves], scan_dealt[kWaves], start_units, arrived[2];
    __shared__ int start_row;
    const int tid = threadIdx.x, lane = tid % JL_WAVE, wave = uniform(tid / JL_WAVE);
    const int g = lane / 16, m = lane % 16;
    const int heads = p.cache.kv_heads * p.blocks_of_16;      // of a row's list
    const int page_shift = p.cache.page_shift, in_page_mask = (1 << page_shift) - 1;

    // ---- the rows' ranges, 64 at a time in the lanes of every wave
    int window_row = 0;
    Range in_lane;
    int own_tiles = 0;                                        // without those of rows that go with the lane's
    auto load_window = [&](int from) {
        window_row = from;
        in_lane = from + lane < p.rows ? range_of(p, from + lane) : Range{0, -1, 0};
        own_tiles = in_lane.tiles();
        if constexpr (SHARED) in_lane = run_in_lanes(p, in_lane, lane);
    };

    // ---- this workgroup's share of the list: whole (row, head) pairs one after the other where all rows are short, else
    // an equal span of tiles.  (All tiles together are fewer than 2^32: jl_kv_attention.)
    load_window(0);
    const uint32_t mine = units_of(in_lane.tiles());
    uint32_t all, through = mine;                             // tiles of all rows; of those up to this lane's (this thread's last)
    uint32_t longest = mine, own = mine, longest_dealt = mine;   // ... of what is dealt whole
    int per = (p.rows + kThreads - 1) / kThreads;             // rows a thread, where a wave does not hold them all
    if constexpr (SHARED) per = (per + p.rows_each - 1) & -p.rows_each;
    if constexpr (SHARED)
        for (int off = 1; off < p.rows_each; off <<= 1) longest_dealt += __shfl_xor(longest_dealt, off, JL_WAVE);
    if (p.rows > JL_WAVE) {
        uint32_t dealt = 0;
        own = longest = longest_dealt = 0;
        for_runs<SHARED>(p, tid * per, min((tid + 1) * per, p.rows), [&](int r, const Range &range) {
            const uint32_t n = units_of(range.tiles());
            own += n;
            longest = max(longest, n);
            if constexpr (SHARED) {
                dealt = (r & (p.rows_each - 1)) ? dealt + n : n;
                longest_dealt = max(longest_dealt, dealt);
            }
            return true;
        });
        through = own;
    }
#pragma unroll
    for (int off = 1; off < JL_WAVE; off <<= 1) {
        const uint32_t other = __shfl_up(through, off, JL_WAVE);
        if (lane >= off) through += other;
    }
#pragma unroll
    for (int off = JL_WAVE / 2; off; off >>= 1) {
        longest = max(longest, (uint32_t)__shfl_xor(longest, off, JL_WAVE));
        if constexpr (SHARED) longest_dealt = max(longest_dealt, (uint32_t)__shfl_xor(longest_dealt, off, JL_WAVE));
    }
    all = __builtin_amdgcn_readlane(through, JL_WAVE - 1);
    if (p.rows > JL_WAVE) {
        if (lane == 0) scan[wave] = all, scan_longest[wave] = longest, scan_dealt[wave] = longest_dealt;
        __syncthreads();
        all = 0;
        for (int w = 0; w < kWaves; w++) {
            if (w < wave) through += scan[w];
            all += scan[w];
            longest = max(longest, scan_longest[w]);
            if constexpr (SHARED) longest_dealt = max(longest_dealt, scan_dealt[w]);
        }
    }
    all = uniform(all), longest = uniform(longest), longest_dealt = uniform(longest_dealt);
    // Pairs are not cut where a workgroup is done with its whole ones in the time that all take to read anyway, or in what
    // joining parts takes besides, ten tiles' worth.  (32 rows of 8 heads, 1000 tokens each: 27.8 us whole, 31.6 cut; 8 heads
    // of 1000 tokens: 20.2 whole, 10.2 cut; of 256 tokens: 9.1 and 9.7.)
    // (Rows that go together: what is dealt whole is rows_each rows, whose runs come one after the other.)
    const int each = SHARED ? p.rows_each : 1;
    const float rounds = ceilf((float)((p.rows + each - 1) / each) * heads / gridDim.x);
    // Rows that go together read from the caches: whole where that is at most twice an equal span (2048 tokens, 32 heads over 8
    // of 64: 118 us whole, 203 cut).
    const bool whole = SHARED ? ((float)longest_dealt * rounds - kStart - 10) * gridDim.x <= 2.f * (float)all * heads
                              : ((float)longest * rounds - kStart - 10) * Shape<Q8, DIM>::kTilesAtOnce <= (float)all * heads;
    const uint32_t total = all * heads;
    const uint32_t least = max((longest + kMostParts - 1) / kMostParts, min((longest + kParts - 1) / kParts, kLargePart));
    const uint32_t span = max((total + gridDim.x - 1) / gridDim.x, least);
    const uint32_t begin = whole ? 0 : span * blockIdx.x;
    if (p.rows > JL_WAVE) {
        const uint32_t from = begin / heads;
        if (!whole && begin < total && from >= through - own && from < through) {
            uint32_t before = through - own;
            for_runs<SHARED>(p, tid * per, min((tid + 1) * per, p.rows), [&](int r, const Range &range) {
                const uint32_t n = units_of(range.tiles());
                if (before + n > from) {
                    start_row = r, start_units = before;
                    return false;
                }
                before += n;
                return true;
            });
        }
        __syncthreads();
    }

    // rows with nothing to read (one that goes with others is zeros from them too)
    const int width = p.cache.kv_heads * p.group * DIM;
    for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const int n = p.rows <= JL_WAVE ? __builtin_amdgcn_readlane(own_tiles, r) : range_of(p, r).tiles();
        if (n == 0)
            for (int c = 4 * tid; c < width; c += 4 * kThreads) store_out(p, r * p.ldo + c, floatx4{0.f, 0.f, 0.f, 0.f});
    }

    const int row_step = gridDim.x / heads, head_step = gridDim.x % heads;    // from one whole pair of a workgroup to its next
    Piece next;
    if (whole) {
        next.row = blockIdx.x / heads * each, next.head = blockIdx.x % heads, next.unit = 0;
        next.left = 1;
    } else {
        if (begin >= total) return;
        const uint32_t from = begin / heads;
        uint32_t before;
        if (p.rows <= JL_WAVE) {
            next.row = __popcll(__ballot(through <= from));
            before = next.row == 0 ? 0 : __builtin_amdgcn_readlane(through, uniform(next.row - 1));
        } else {
            next.row = uniform(start_row), before = uniform(start_units);
        }
        next.head = begin - before * heads;                   // (its unit in the row's list, taken apart below)
        next.unit = -1;
        next.left = min(span, total - begin);
    }
    auto next_whole = [&]() {
        if (((next.row + 1) & (each - 1)) && next.row + 1 < p.rows) {
            next.row++;
        } else {
            next.row = (next.row & -each) + row_step * each, next.head += head_step;
            if (next.head >= heads) next.head -= heads, next.row += each;
        }
    };
    // Completes `next` from its row, head and tile, going on to the first row that has tiles.
    auto complete = [&]() {
        next.row = uniform(next.row), next.head = uniform(next.head), next.unit = uniform(next.unit), next.left = uniform(next.left);
        while (next.left > 0) {
            if (next.row >= p.rows) {
                next.left = 0;
                break;
            }
            if (next.row < window_row || next.row >= window_row + JL_WAVE) load_window(SHARED ? next.row & -16 : next.row);
            const int at = uniform(next.row - window_row);
            next.first = __builtin_amdgcn_readlane(in_lane.first, at);
            next.end = __builtin_amdgcn_readlane(in_lane.end, at);
            next.request = __builtin_amdgcn_readlane(in_lane.request, at);
            next.members = SHARED ? __builtin_amdgcn_readlane(in_lane.members, at) : 1;
            next.tiles = Range{next.first, next.end, 0}.tiles();
            if (next.tiles > 0) break;
            if (whole) next_whole();
            else next.row++;
        }
        if (next.unit < 0 && next.left > 0) {
            const int into = next.head, units = units_of(next.tiles);
            next.head = uniform((uint32_t)into / units);
            next.unit = into - next.head * units;
        }
        // (a head's first units are its beginning, not tiles: a span that ends there has none of it)
        const int until = whole ? next.tiles + kStart : min(next.unit + next.left, (uint32_t)next.tiles + kStart);
        next.tile = max(next.unit - kStart, 0);
        next.count = max(until - kStart, 0) - next.tile;
    };

    // k and v of a tile go from memory to `raw`; `page` are the pages of its halves, and one behind the last token, or one
    // outside the cache, is -1
    Raw<Q8, DIM> raw;
    bool loaded = false;          // it has, or waits for, the wave's first tile of the coming piece
    uint32_t paged = 0;           // bit h: half h of its tile has a page of the cache
    int page[kHalves];
    auto find_pages = [&](const Piece &c, int t) {
        // (scalar loads: vector loads come back in order, and these would wait for the tile that is under way)
        typedef const __attribute__((address_space(4))) int32_t constant_int;
        constant_int *table = (constant_int *)(uintptr_t)(p.table + c.request * p.table_stride);
#pragma unroll
        for (int h = 0; h < kHalves; h++) {
            const int token = t * kTile + 16 * h;
            page[h] = token < c.end ? table[token >> page_shift] : -1;
        }
    };
    auto issue = [&](int kv_head, int t, bool values) {
        if (values) paged = 0;
#pragma unroll
        for (int h = 0; h < kHalves; h++) {
            const bool real = (unsigned)page[h] < (unsigned)p.cache.pages;
            const uint8_t *part = p.cache.k + ((int64_t)(real ? page[h] : 0) * p.cache.kv_heads + kv_head) * p.cache.part_bytes;
            const int in_page = (t * kTile + 16 * h) & in_page_mask;
            if (values) {
                raw.template load_v<SHARED>(h, part + p.cache.v_offset, in_page, page_shift, g, m);
                paged |= real ? 1u << h : 0u;
            } else {
                raw.template load_k<SHARED>(h, part, in_page, page_shift, g, m);
            }
        }
    };
    const bool one_block = p.blocks_of_16 == 1;
    auto kv_head_of = [&](int head) { return one_block ? head : head / p.blocks_of_16; };

    // Of two workgroups on a compute unit the one that came first has the right of way, and is done with an equal span in
    // three quarters of the time (65 and 87 us); the other one then has the unit to itself and cannot fill it.  The later
    // half of the launch goes first in three of four tiles: 97.4 -> 94.6 us over 64 ragged rows, 68.9 -> 65.9 over 8-bit blocks.
    const bool second = 2 * blockIdx.x >= gridDim.x;
    Cut went_on, opened;
    went_on.parts = opened.parts = 0;
    for (complete(); next.left > 0;) {
        const Piece cur = next;
        // the piece behind this one: the loads of its first tiles go out with this one's last
        next.left = whole ? 1 : next.left - min(next.left, units_of(cur.tiles) - cur.unit);
        next.unit = 0;
        if (whole) next_whole();
        else if (++next.head >= heads) next.head -= heads, next.row++;
        complete();
        const int count = cur.count, row = cur.row;
        if (count == 0) continue;
        const int kv_head = kv_head_of(cur.head), block_of_16 = cur.head - kv_head * p.blocks_of_16;
        // (a row's tiles begin with the one of its first token)
        const int list_tile = cur.first / kTile + cur.tile, last = list_tile + count, from_tile = list_tile + wave;
        const int next_list = next.left > 0 ? next.first / kTile + next.tile : 0, next_last = next_list + next.count, next_tile = next_list + wave;
        const int next_head = next.left > 0 ? kv_head_of(next.head) : 0;
        // a first tile that is not on its way yet; a wave that this piece has none for goes on to the next one's at once
        const bool here = from_tile < last, there = !here && next.left > 0 && next_tile < next_last;
        if (here ? !loaded : there) {
            find_pages(here ? cur : next, here ? from_tile : next_tile);
            issue(here ? kv_head : next_head, here ? from_tile : next_tile, false);
            issue(here ? kv_head : next_head, here ? from_tile : next_tile, true);
        }
        loaded = there;
        // columns: query heads of a row, or of one row after the other
        const int q_head = kv_head * p.group + 16 * block_of_16, q_heads = SHARED ? cur.members * p.group : min(p.group - 16 * block_of_16, 16);
        int row_of_lane = row, head_of_lane = m < q_heads ? m : 0;
        int position = 0;
        if constexpr (SHARED) {
            row_of_lane += head_of_lane / p.group, head_of_lane %= p.group;
            position = p.positions[row_of_lane];
        }

        // ---- q, times a power of two that brings its largest value to 2^10 ... 2^11: both parts are then binary16
        // numbers of full precision however large or small the row is
        jl_half8 q_hi[kSteps], q_lo[kSteps];
        float undo;
        {
            floatx4 x[kSteps][2];
            const float *from = p.q + row_of_lane * p.ldq + (q_head + head_of_lane) * DIM;
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; s++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    x[s][c] = *(const floatx4 *)(from + Raw<Q8, DIM>::element(s, g) + 4 * c);
                    x[s][c] *= p.scale;
#pragma unroll
                    for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(x[s][c][i]));
                }
            most = over_groups_max(most);
            int exponent = (int)((__float_as_uint(most) >> 23) & 255) - 127;
            if (exponent < -100 || exponent == 128) exponent = 10;                  // zeros and the like, infinities, NaN
            const float to = __uint_as_float((uint32_t)(10 - exponent + 127) << 23);
            undo = __uint_as_float((uint32_t)(exponent - 10 + 127) << 23);
#pragma unroll
            for (int s = 0; s < kSteps; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int e = Raw<Q8, DIM>::in_eight(i);
                    const float y = x[s][e / 4][e % 4] * to;
                    q_hi[s][i] = (_Float16)y;
                    q_lo[s][i] = (_Float16)(y - (float)q_hi[s][i]);
                }
        }

        Range seen_here{cur.first, cur.end, 0}, seen_by_all = seen_here;      // what the lane's row sees, what all of them do
        if constexpr (SHARED) {
            seen_here = range_at(p, position, cur.request), seen_by_all = seen_here;
#define JL_SEEN_FROM(N)                                                                                                        \
    seen_by_all.first = max(seen_by_all.first, __builtin_amdgcn_update_dpp(0, seen_by_all.first, 0x120 + N, 0xF, 0xF, true));  \
    seen_by_all.end = min(seen_by_all.end, __builtin_amdgcn_update_dpp(0, seen_by_all.end, 0x120 + N, 0xF, 0xF, true));
            JL_SEEN_FROM(8) JL_SEEN_FROM(4) JL_SEEN_FROM(2) JL_SEEN_FROM(1)   // (round the sixteen lanes)
#undef JL_SEEN_FROM
            seen_by_all.first = uniform(seen_by_all.first), seen_by_all.end = uniform(seen_by_all.end);
        }

        floatx4 o[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) o[b] = floatx4{0.f, 0.f, 0.f, 0.f};
        float top = kNone, sum = 0.f;

        for (int t = from_tile; t < last; t += kWaves) {
            if (second) {
                if (t / kWaves % 4 != 0) __builtin_amdgcn_s_setprio(1);
                else __builtin_amdgcn_s_setprio(0);
            }
            const uint32_t with_page = paged;
            // what is loaded next: this piece's next tile of the wave, or the next piece's first
            const bool more = t + kWaves < last;
            loaded = more || (next.left > 0 && next_tile < next_last);
            const int load_tile = more ? t + kWaves : next_tile, load_head = more ? kv_head : next_head;
            if (loaded) find_pages(more ? cur : next, load_tile);
            // (the halves side by side: a product waits for the one before it of its own half only)
            floatx4 s[kHalves];
#pragma unroll
            for (int h = 0; h < kHalves; h++) s[h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                jl_half8 k[kHalves];
#pragma unroll
                for (int h = 0; h < kHalves; h++) {
                    k[h] = raw.k_operand(h, i);
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[h], q_lo[i], s[h], 0, 0, 0);
                }
#pragma unroll
                for (int h = 0; h < kHalves; h++) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[h], q_hi[i], s[h], 0, 0, 0);
            }
            if (loaded) issue(load_head, load_tile, false);   // k goes out as soon as this tile's is used
            const bool all_seen = t * kTile >= seen_by_all.first && t * kTile + kTile <= seen_by_all.end && with_page == (1u << kHalves) - 1;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = s[i / 4][i % 4];
            if (!all_seen) {
                bool seen[kHalves][4];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int token = t * kTile + 16 * (i / 4) + 4 * g + i % 4;
                    seen[i / 4][i % 4] = token >= cur.first && token < cur.end && (with_page >> (i / 4) & 1);
                    x[i] = seen[i / 4][i % 4] && (!SHARED || (token >= seen_here.first && token < seen_here.end)) ? x[i] : -INFINITY;
                }
                raw.mask_v(seen);
                if constexpr (SHARED) {
                    // An infinity or NaN that one row sees would reach one that does not, as nothing times it.  It is taken out
                    // of v, and NaN goes to those that see it: in bfloat16, 2^127 in its place times 2^127 and -2^127 for each
                    // such row, and zeros for all others.
                    if (__any(raw.any_not_finite())) {
                        uintx4 sees;
#pragma unroll
                        for (int i = 0; i < 8; i += 2) sees[i / 2] = (x[i] == -INFINITY ? 0u : 0x7f00u) | (x[i + 1] == -INFINITY ? 0u : 0x7f000000u);
                        const bfloat8 plus = __builtin_bit_cast(bfloat8, sees), minus = __builtin_bit_cast(bfloat8, sees ^ 0x80008000u);
#pragma unroll
                        for (int b = 0; b < kBlocks; b += 2) {
                            jl_half8 v[2];
                            raw.v_operands(b, v);
#pragma unroll
                            for (int c = 0; c < 2; c++) {
                                uintx4 its = __builtin_bit_cast(uintx4, v[c]);
#pragma unroll
                                for (int i = 0; i < 4; i++) its[i] = not_finite(its[i]) & 0x7f007f00u;
                                const bfloat8 bad = __builtin_bit_cast(bfloat8, its);
                                o[b + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bad, plus, o[b + c], 0, 0, 0);
                                o[b + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bad, minus, o[b + c], 0, 0, 0);
                            }
                        }
                        raw.drop_not_finite();
                    }
                }
            }
            float most = x[0];
#pragma unroll
            for (int i = 1; i < 8; i++) most = fmaxf(most, x[i]);
            most = over_groups_max(most) * undo;
            // The maximum may fall behind by a factor of 2^kSlack before everything is brought to the new one: after a
            // row's first tiles this is rare.
            if (__any(most > top + kSlack)) {
                const float next_top = fmaxf(top, most);
                const float keep = __builtin_amdgcn_exp2f(top - next_top);
                top = next_top;
                sum *= keep;
#pragma unroll
                for (int b = 0; b < kBlocks; b++) o[b] *= keep;
            }
            const float lift = kLift - top;
            uintx4 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float a = __builtin_amdgcn_exp2f(fmaf(x[i], undo, lift)), b = __builtin_amdgcn_exp2f(fmaf(x[i + 1], undo, lift));
                sum += a + b;
                const jl_half2v two = __builtin_convertvector(floatx2{a, b}, jl_half2v);
                hi[i / 2] = as_u32(two);
                lo[i / 2] = as_u32(__builtin_convertvector(floatx2{a - (float)two[0], b - (float)two[1]}, jl_half2v));
            }
            const jl_half8 p_hi = __builtin_bit_cast(jl_half8, hi), p_lo = __builtin_bit_cast(jl_half8, lo);
#pragma unroll
            for (int b = 0; b < kBlocks; b += 2) {
                jl_half8 v[2];
                raw.v_operands(b, v);
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[0], p_lo, o[b], 0, 0, 0);
                o[b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[1], p_lo, o[b + 1], 0, 0, 0);
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[0], p_hi, o[b], 0, 0, 0);
                o[b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[1], p_hi, o[b + 1], 0, 0, 0);
            }
            if (loaded) issue(load_head, load_tile, true);
        }

        // ---- the four waves' parts into one
        sum = over_groups_sum(sum);
        if (g == 0) joined_max[wave][m] = top, joined_sum[wave][m] = sum;
        const bool opens = cur.tile == 0, closes = cur.tile + count == cur.tiles;
        float *slot = p.parts + (int64_t)(2 * blockIdx.x + (opens ? 1 : 0)) * kSlot;
        auto finish = [&](int h, int d, floatx4 v, float l) {
            store_out(p, (SHARED ? (row + h / p.group) * p.ldo + (int64_t)(q_head + h % p.group) * DIM : row * p.ldo + (int64_t)(q_head + h) * DIM) + d, l == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : v / l);
        };
#pragma unroll
        for (int from = 0; from < DIM; from += kRound) {
            if (from > 0) __syncthreads();
            if (m < q_heads) {
#pragma unroll
                for (int b = from / 16; b < (from + kRound) / 16; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) joined[wave][m][out_element<DIM>(b, 4 * g + i) - from] = o[b][i];
            }
            __syncthreads();
            for (int c = 4 * tid; c < q_heads * kRound; c += 4 * kThreads) {
                const int h = c / kRound, d = c % kRound;
                const float most = fmaxf(fmaxf(joined_max[0][h], joined_max[1][h]), fmaxf(joined_max[2][h], joined_max[3][h]));
                floatx4 v = {0.f, 0.f, 0.f, 0.f};
                float l = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float share = __builtin_amdgcn_exp2f(joined_max[w][h] - most);
                    v += share * *(const floatx4 *)&joined[w][h][d];
                    l += share * joined_sum[w][h];
                }
                if (opens && closes) {
                    finish(h, from + d, v, l);
                } else {
                    agent_store4(slot + h * DIM + from + d, v);
                    if (from + d == 0) agent_store(slot + 16 * DIM + h, most), agent_store(slot + 16 * DIM + 16 + h, l);
                }
            }
        }
        if (!(opens && closes)) {
            const uint32_t head_begin = begin + min(span, total - begin) - cur.left - cur.unit;   // in the list of all units
            Cut &c = opens ? opened : went_on;
            c.row = row, c.members = cur.members, c.kv_head = kv_head, c.block_of_16 = block_of_16;
            // the spans that have tiles of it: from the one of its first tile on
            c.group = (head_begin + kStart) / span, c.parts = (head_begin + kStart + cur.tiles - 1) / span - c.group + 1;
        }
        __syncthreads();
    }

    // ---- heads that others have parts of: the workgroup that is the last to be done with its part joins all, in their
    // order.  (Two at most: one that the span begins in, one that it ends in.)
    if (went_on.parts == 0 && opened.parts == 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // this wave's stores have arrived
    __syncthreads();
    if (tid < 2) {
        const int group = tid ? opened.group : went_on.group, parts = tid ? opened.parts : went_on.parts;
        uint32_t before = 0;
        if (parts > 0) {
            before = __hip_atomic_fetch_add(p.arrived + group, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
            if (before == (uint32_t)parts) __hip_atomic_store(p.arrived + group, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        arrived[tid] = before;
    }
    __syncthreads();
#pragma unroll 1
    for (int which = 0; which < 2; which++) {
        const Cut c = which ? opened : went_on;
        if (c.parts == 0 || arrived[which] != (uint32_t)c.parts) continue;
        const int q_head = c.kv_head * p.group + 16 * c.block_of_16, parts = c.parts;
        const int q_heads = SHARED ? c.members * p.group : min(p.group - 16 * c.block_of_16, 16);
        // (the parts were written past the second-level caches and are read past this XCD's own, which may hold an earlier
        // call's: buffer loads with the bit for that.  A fence would empty the cache for everybody: 40 us instead of 32 where
        // 256 heads are joined at once)
        const auto parts_at = __builtin_amdgcn_make_buffer_rsrc((void *)p.parts, 0, -1, 0x00020000);
        auto read4 = [&](int at) {
            return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(parts_at, 4 * at, 0, kDeviceScope));
        };
        auto read1 = [&](int at) {
            return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(parts_at, 4 * at, 0, kDeviceScope));
        };
        // part 0 is what its span opened, the others what theirs went on with
        auto slot_of = [&](int i) { return (2 * (c.group + i) + (i == 0 ? 1 : 0)) * kSlot; };
        // Threads across the heads' elements, and across the parts where there are threads enough.  The loads of
        // a batch of parts are under way together, their maxima and sums with them (64 parts: 17 us with a loop
        // that waits for each).
        constexpr int kBatch = 16;
        const int quads = q_heads * (DIM / 4), sets = max(kThreads / quads, 1);
        float *folded = &joined[0][0][0];             // [sets][quads]: four elements, the maximum, the sum
        for (int base = 0; base < quads; base += kThreads) {
            const int at = sets > 1 ? tid % quads : base + tid, set = sets > 1 ? tid / quads : 0;
            const int h = at / (DIM / 4);
            floatx4 v = {0.f, 0.f, 0.f, 0.f};
            float most = kNone, l = 0.f;
            if (at < quads && set < sets) {
                for (int i = set; i < parts; i += kBatch * sets) {
                    floatx4 part[kBatch];
                    float part_most[kBatch], part_sum[kBatch];
#pragma unroll
                    for (int j = 0; j < kBatch; j++) {
                        const int from = slot_of(min(i + j * sets, parts - 1));
                        part_most[j] = read1(from + 16 * DIM + h), part_sum[j] = read1(from + 16 * DIM + 16 + h);
                        part[j] = read4(from + 4 * at);
                    }
                    float next_most = most;
#pragma unroll
                    for (int j = 0; j < kBatch; j++) next_most = fmaxf(next_most, part_most[j]);
                    const float keep = __builtin_amdgcn_exp2f(most - next_most);
                    most = next_most, v *= keep, l *= keep;
#pragma unroll
                    for (int j = 0; j < kBatch; j++) {
                        if (i + j * sets < parts) {
                            const float share = __builtin_amdgcn_exp2f(part_most[j] - most);
                            v += share * part[j], l += share * part_sum[j];
                        }
                    }
                }
                if (sets > 1) {
                    float *to = folded + 8 * (set * quads + at);
                    *(floatx4 *)to = v, to[4] = most, to[5] = l;
                }
            }
            if (sets > 1) __syncthreads();
            if (at < quads && set == 0) {
                for (int i = 1; i < sets; i++) {
                    const float *from = folded + 8 * (i * quads + at);
                    const float next_most = fmaxf(most, from[4]);
                    const float keep = __builtin_amdgcn_exp2f(most - next_most), share = __builtin_amdgcn_exp2f(from[4] - next_most);
                    v = keep * v + share * *(const floatx4 *)from, l = keep * l + share * from[5], most = next_most;
                }
                const int64_t to = SHARED ? (c.row + h / p.group) * p.ldo + (int64_t)(q_head + h % p.group) * DIM + 4 * at - h * DIM
                                          : c.row * p.ldo + (int64_t)q_head * DIM + 4 * at;
                store_out(p, to, l == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : v / l);
            }
        }
        __syncthreads();
    }
}

template <bool Q8, int DIM>
hipError_t launch(const AttentionArgs &a, int compute_units, hipStream_t stream) {
    const int groups = std::min(Shape<Q8, DIM>::kPerUnit * compute_units, kMostGroups);
    if (a.rows_each > 1) hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, DIM, true>), dim3((unsigned)groups), dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, DIM, false>), dim3((unsigned)groups), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}
template <bool Q8>
hipError_t launch_dim(const AttentionArgs &a, int head_dim, int compute_units, hipStream_t stream) {
    switch (head_dim) {
        case 64: return launch<Q8, 64>(a, compute_units, stream);
        case 96: return launch<Q8, 96>(a, compute_units, stream);
        case 128: return launch<Q8, 128>(a, compute_units, stream);
        case 192: return launch<Q8, 192>(a, compute_units, stream);
        default: return launch<Q8, 256>(a, compute_units, stream);
    }
}

constexpr size_t kArrivedBytes = kMostGroups * sizeof(uint32_t);

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

extern "C" {

size_t jl_kv_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
    return kArrivedBytes + (size_t)2 * kMostGroups * 16 * ((size_t)head_dim + 2) * sizeof(float);
}

int jl_kv_attention_workspace_init(jl_context *ctx, void *workspace, size_t workspace_bytes) {
    JL_REQUIRE(ctx && workspace, "jl_kv_attention_workspace_init: null argument");
    JL_REQUIRE(aligned(workspace, 16), "jl_kv_attention_workspace_init: the workspace must be 16-byte aligned");
    if (workspace_bytes < kArrivedBytes)
        return jl_fail(JL_ERR_WORKSPACE, "jl_kv_attention_workspace_init: workspace of %zu bytes", workspace_bytes);
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    return jl_launch_fill(ctx, (float *)workspace, 0.f, kArrivedBytes / sizeof(float));
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
    // (a row's list of tiles of 32 tokens, times its heads, all rows together: a 32-bit number)
    const int64_t table_tokens = std::min(table_stride * cache->page_tokens, (int64_t)INT_MAX - 64);
    const int64_t lists = rows * cache->kv_heads * ((heads / cache->kv_heads + 15) / 16);
    JL_REQUIRE(lists <= 0 || table_tokens / 32 + 2 + kStart <= (int64_t)(UINT32_MAX - 2 * kMostGroups) / lists,
               "jl_kv_attention: %lld rows of %d heads over %lld tokens in one call", (long long)rows, heads, (long long)table_tokens);
    const float scale_of_powers = scale * 1.44269504088896340736f;   // weights are powers of two
    JL_REQUIRE(std::isfinite(scale_of_powers), "jl_kv_attention: scale %g", (double)scale);
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
    JL_REQUIRE(out != q, "jl_kv_attention: out in place of q");
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    AttentionArgs a;
    a.cache = jl_kv_view(cache);
    a.q = q, a.ldq = ldq, a.ldo = ldo;
    a.positions = positions, a.row_requests = row_requests, a.table = block_table;
    a.requests = (int)requests, a.table_stride = table_stride, a.table_tokens = (int)table_tokens;
    a.scale = scale_of_powers;
    a.window = window > INT32_MAX ? 0 : (int)window;   // one that reaches behind every position
    a.group = heads / cache->kv_heads;
    a.blocks_of_16 = (a.group + 15) / 16;
    // Twice as many rows as requests, or more: some are of one, unless they are padding.  (32 heads over 8 of 128, one request,
    // each row alone and together: a prompt of 2048 tokens 753 and 187 us, of 512 64 and 27; 4 rows after 30 000 tokens 79 and
    // 44, after 1000 11.8 and 14.0.  32 heads over 32, 512 tokens: 224 and 32.  64 rows of 64 requests of up to 8192 tokens
    // padded to 512 rows: 118 and 124; to 72, which are too few: 105 and 118.)
    a.rows_each = 1;
    if (row_requests && rows >= 2 * requests)
        while (2 * a.rows_each * a.group <= 16) a.rows_each *= 2;
    a.rows = (int)rows;
    a.out = out, a.out_f16 = out_f16 != 0;
    a.arrived = (uint32_t *)workspace;
    a.parts = (float *)((uint8_t *)workspace + kArrivedBytes);
    JL_HIP(cache->type == JL_KV_Q8_0 ? launch_dim<true>(a, dim, ctx->compute_units, ctx->stream)
                                     : launch_dim<false>(a, dim, ctx->compute_units, ctx->stream));
    return JL_OK;
}

}  // extern "C"
