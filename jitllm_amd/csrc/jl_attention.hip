// jl_kv_attention: attention of one new token a row over its request's pages.
//
// Mathematics.  For a row and a head of k and v, S = K Q^T over tiles of 32 tokens and up to 16 query heads (the heads
// that share k and v), P = 2^(S - m) with a running maximum m, O = O 2^(m_old - m) + V^T P^T, l the sum of P; the result
// is O / l, and two parts (m, l, O) of a row join by the same rule.  scale * log2(e) is folded into q.
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
// join in LDS.  A row's head that a cut goes through leaves its parts in the workspace, and a second launch joins them
// in their order.
#include <algorithm>
#include <climits>
#include <cmath>

#include "jl_kv.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / JL_WAVE;
constexpr int kTile = 32;                 // tokens
constexpr int kLeastSpan = kWaves;        // tiles: one a wave
constexpr int kMostGroups = 1024;         // workgroups of a launch, and spans
constexpr float kNone = -3.0e38f;         // the running maximum of nothing: finite, so that differences are numbers

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

struct Part {             // a row's head that is cut: its parts are spans `group` ... group + count - 1
    int row, head, group, count;
};

struct AttentionArgs {
    JlKvView cache;
    const float *q;
    int64_t ldq, ldo;
    const int32_t *positions, *row_requests, *table;
    int64_t requests, table_stride;
    float scale;          // times log2(e): weights are powers of two
    int window;           // 0: none
    int group;            // query heads to a head of k and v
    int blocks_of_16;     // ... in sixteens
    int rows;
    void *out;
    bool out_f16;
    bool by_head;         // `cut` has an entry per row and head instead of one per span
    Part *cut;
    float *parts;         // [2 * spans][16 * (DIM + 2)]
};

// The tokens [first, end) that a row sees.
struct Range {
    int first, end;
    __device__ int tiles() const { return end > first ? (end + kTile - 1) / kTile - first / kTile : 0; }
};
__device__ __forceinline__ Range range_of(const AttentionArgs &p, int row) {
    const int position = p.positions[row];
    const int request = p.row_requests ? p.row_requests[row] : row;
    const int64_t held = min((int64_t)p.table_stride << p.cache.page_shift, (int64_t)INT_MAX);
    Range r;
    r.end = position >= 0 && request >= 0 && request < p.requests ? (int)min((int64_t)position + 1, held) : 0;
    r.first = p.window > 0 ? max(position - p.window + 1, 0) : 0;
    return r;
}

// k and v pass once: loads that do not stay in the caches (512 MB in 16 KB pieces, nothing else done: 90 us with ordinary
// loads, 80 with these).
template <typename T>
__device__ __forceinline__ T load_at(const uint8_t *base, uint32_t offset) {
    return __builtin_nontemporal_load((const T *)(base + offset));
}
__device__ __forceinline__ jl_half2v as_half2(uint32_t x) { return __builtin_bit_cast(jl_half2v, x); }
__device__ __forceinline__ uint32_t as_u32(jl_half2v x) { return __builtin_bit_cast(uint32_t, x); }

// A tile's k and v as they lie in memory.  Lane (g, m) = (lane / 16, lane % 16) has, of k, token m of each 16-token half,
// and of v the tokens 4 g + i of each half at a few consecutive elements: head_dim is cut into pieces of 128, 64 and 32,
// and m has 8, 4 or 2 values of a piece.
template <bool Q8, int DIM>
struct Raw;

template <int DIM>
struct Raw<false, DIM> {
    static constexpr int kSteps = DIM / 32;
    static constexpr int kWide = DIM / 128, kMid = DIM % 128 / 64, kThin = DIM % 64 / 32;
    uintx4 k[2][kSteps];
    uintx4 v4[2][4][kWide ? kWide : 1];
    uintx2 v2[2][4];
    uint32_t v1[2][4];
    __device__ static int element(int step, int g) { return 32 * step + 8 * g; }   // first of the eight of k step `step`
    __device__ void load_k(int half, const uint8_t *part, int in_page, int, int g, int m) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) k[half][s] = load_at<uintx4>(part, (in_page + m) * (2 * DIM) + 64 * s + 16 * g);
    }
    __device__ void load_v(int half, const uint8_t *part, int in_page, int, int g, int m) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t row = (in_page + 4 * g + i) * (2 * DIM);
#pragma unroll
            for (int w = 0; w < kWide; w++) v4[half][i][w] = load_at<uintx4>(part, row + 256 * w + 16 * m);
            if constexpr (kMid) v2[half][i] = load_at<uintx2>(part, row + 256 * kWide + 8 * m);
            if constexpr (kThin) v1[half][i] = load_at<uint32_t>(part, row + 256 * kWide + 128 * kMid + 4 * m);
        }
    }
    __device__ jl_half8 k_operand(int half, int step) const { return __builtin_bit_cast(jl_half8, k[half][step]); }
    // masked tokens' values are nothing, whatever lies there
    __device__ void mask_v(const bool (&seen)[2][4]) {
#pragma unroll
        for (int h = 0; h < 2; h++)
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
    // eight tokens of the column that output block `block` takes of this lane
    __device__ jl_half8 v_operand(int block) const {
        uintx4 r;
        const int word = block / 2;
        const uint32_t pick = block % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int pair = 0; pair < 4; pair++) {
            const int h = pair / 2, i = pair % 2 * 2;
            uint32_t a, b;
            if (word < 4 * kWide) a = v4[h][i][word / 4][word % 4], b = v4[h][i + 1][word / 4][word % 4];
            else if (word < 4 * kWide + 2 * kMid) a = v2[h][i][word % 2], b = v2[h][i + 1][word % 2];
            else a = v1[h][i], b = v1[h][i + 1];
            r[pair] = __builtin_amdgcn_perm(b, a, pick);
        }
        return __builtin_bit_cast(jl_half8, r);
    }
};

template <int DIM>
struct Raw<true, DIM> {
    static constexpr int kSteps = DIM / 32, kPairs = DIM / 64, kTail = DIM % 64 / 32;
    static constexpr int kWide = DIM / 128, kMid = DIM % 128 / 64, kThin = DIM % 64 / 32;
    static constexpr int kPieces = kWide + kMid + kThin;
    uintx4 k[2][kPairs];
    uintx2 k_tail[2];
    uint16_t k_scale[2][kPairs + kTail];
    uintx2 v2[2][4][kWide ? kWide : 1];
    uint32_t v1[2][4];
    uint16_t v0[2][4];
    uintx2 v_scale[2][kPieces];
    // (16 consecutive bytes serve two steps: a lane's loads stay 16 bytes wide)
    __device__ static int element(int step, int g) {
        return step < 2 * kPairs ? 64 * (step / 2) + 16 * g + 8 * (step % 2) : 64 * kPairs + 8 * g;
    }
    __device__ void load_k(int half, const uint8_t *part, int in_page, int page_shift, int g, int m) {
        const uint32_t row = (in_page + m) * DIM, scales = ((uint32_t)DIM << page_shift) + 2 * (in_page + m);
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            k[half][i] = load_at<uintx4>(part, row + 64 * i + 16 * g);
            k_scale[half][i] = load_at<uint16_t>(part, scales + ((2 * (2 * i + g / 2)) << page_shift));
        }
        if constexpr (kTail) {
            k_tail[half] = load_at<uintx2>(part, row + 64 * kPairs + 8 * g);
            k_scale[half][kPairs] = load_at<uint16_t>(part, scales + ((2 * 2 * kPairs) << page_shift));
        }
    }
    __device__ void load_v(int half, const uint8_t *part, int in_page, int page_shift, int g, int m) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t row = (in_page + 4 * g + i) * DIM;
#pragma unroll
            for (int w = 0; w < kWide; w++) v2[half][i][w] = load_at<uintx2>(part, row + 128 * w + 8 * m);
            if constexpr (kMid) v1[half][i] = load_at<uint32_t>(part, row + 128 * kWide + 4 * m);
            if constexpr (kThin) v0[half][i] = load_at<uint16_t>(part, row + 128 * kWide + 64 * kMid + 2 * m);
        }
        const uint32_t scales = ((uint32_t)DIM << page_shift) + 2 * (in_page + 4 * g);
#pragma unroll
        for (int w = 0; w < kWide; w++) v_scale[half][w] = load_at<uintx2>(part, scales + ((2 * (4 * w + m / 4)) << page_shift));
        if constexpr (kMid) v_scale[half][kWide] = load_at<uintx2>(part, scales + ((2 * (4 * kWide + m / 8)) << page_shift));
        if constexpr (kThin) v_scale[half][kWide + kMid] = load_at<uintx2>(part, scales + ((2 * (4 * kWide + 2 * kMid)) << page_shift));
    }
    __device__ jl_half8 k_operand(int half, int step) const {
        uint32_t lo, hi;
        uint32_t d;
        if (step < 2 * kPairs) lo = k[half][step / 2][step % 2 * 2], hi = k[half][step / 2][step % 2 * 2 + 1], d = k_scale[half][step / 2];
        else lo = k_tail[half].x, hi = k_tail[half].y, d = k_scale[half][kPairs + kTail - 1];
        const jl_half2v dd = as_half2(d | d << 16);
        jl_half2v a, b, c, e;
        jl_bytes_to_half(lo, a, b);
        jl_bytes_to_half(hi, c, e);
        a *= dd, b *= dd, c *= dd, e *= dd;
        return jl_half8{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
    }
    // (a byte times a scale of 0; the scale alone can be an infinity or NaN)
    __device__ void mask_v(const bool (&seen)[2][4]) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int w = 0; w < kPieces; w++)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    v_scale[h][w][c] &= (seen[h][2 * c] ? 0xffffu : 0u) | (seen[h][2 * c + 1] ? 0xffff0000u : 0u);
    }
    __device__ jl_half8 v_operand(int block) const {
        uintx4 r;
        const int piece = block < 8 * kWide ? block / 8 : block < 8 * kWide + 4 * kMid ? kWide : kWide + kMid;
#pragma unroll
        for (int pair = 0; pair < 4; pair++) {
            const int h = pair / 2, i = pair % 2 * 2;
            uint32_t a, b;
            int byte;
            if (block < 8 * kWide) a = v2[h][i][block / 8][block % 8 / 4], b = v2[h][i + 1][block / 8][block % 8 / 4], byte = block % 4;
            else if (block < 8 * kWide + 4 * kMid) a = v1[h][i], b = v1[h][i + 1], byte = block % 4;
            else a = v0[h][i], b = v0[h][i + 1], byte = block % 2;
            // byte `byte` of both tokens under 0x64, as in jl_bytes_to_half
            const uint32_t both = __builtin_amdgcn_perm(b, a, 0x0c040c00u + byte * 0x00010001u) ^ 0x64806480u;
            const jl_half2v bias = {(_Float16)1152.f, (_Float16)1152.f};
            r[pair] = as_u32((as_half2(both) - bias) * as_half2(v_scale[h][piece][i / 2]));
        }
        return __builtin_bit_cast(jl_half8, r);
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

template <bool Q8, int DIM>
__global__ void __launch_bounds__(kThreads, DIM == 256 ? 1 : 2) jl_kv_attention_kernel(AttentionArgs p) {
    constexpr int kSteps = DIM / 32, kBlocks = DIM / 16;
    constexpr int kRound = DIM == 256 ? 128 : DIM;            // elements that are joined at a time: 64 KB of LDS at most
    constexpr int kStride = kRound + 4;                       // (four floats on: rows start on other banks)
    __shared__ float joined[kWaves][16][kStride];
    __shared__ float joined_max[kWaves][16], joined_sum[kWaves][16];
    __shared__ int64_t scan[kWaves];
    __shared__ int64_t start_tiles;
    __shared__ int start_row;
    const int tid = threadIdx.x, lane = tid % JL_WAVE, wave = __builtin_amdgcn_readfirstlane(tid / JL_WAVE);
    const int g = lane / 16, m = lane % 16;
    const int heads = p.cache.kv_heads * p.blocks_of_16;      // of a row's list
    const int width = p.cache.kv_heads * p.group * DIM;

    // ---- this workgroup's span of the list of tiles
    const int per = (p.rows + kThreads - 1) / kThreads;
    int64_t mine = 0;
    for (int i = 0; i < per; i++) {
        const int r = tid * per + i;
        if (r < p.rows) mine += range_of(p, r).tiles();
    }
    int64_t through = mine;
#pragma unroll
    for (int off = 1; off < JL_WAVE; off <<= 1) {
        const int64_t other = __shfl_up(through, off, JL_WAVE);
        if (lane >= off) through += other;
    }
    if (lane == JL_WAVE - 1) scan[wave] = through;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kWaves; w++) {
        if (w < wave) through += scan[w];
        all += scan[w];
    }
    const int64_t total = all * heads;
    int64_t span = (total + gridDim.x - 1) / gridDim.x;
    if (span < kLeastSpan) span = kLeastSpan;
    const int64_t begin = span * blockIdx.x;
    // rows with nothing to read
    for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
        if (range_of(p, r).tiles() > 0) continue;
        for (int c = 4 * tid; c < width; c += 4 * kThreads) store_out(p, r * p.ldo + c, floatx4{0.f, 0.f, 0.f, 0.f});
        if (p.by_head)
            for (int h = tid; h < heads; h += kThreads) p.cut[r * heads + h].count = 0;
    }
    if (!p.by_head && tid == 0) p.cut[blockIdx.x].count = 0;
    if (begin >= total) return;
    {
        const int64_t from = begin / heads;
        if (from >= through - mine && from < through) {
            int64_t before = through - mine;
            int r = tid * per;
            for (int n; before + (n = range_of(p, r).tiles()) <= from; r++) before += n;
            start_row = r;
            start_tiles = before;
        }
    }
    __syncthreads();
    int row = __builtin_amdgcn_readfirstlane(start_row);
    Range range = range_of(p, row);
    int tiles = range.tiles();
    const int64_t into = begin - start_tiles * heads;
    int head = (int)(into / tiles), tile = (int)(into % tiles);
    int64_t left = min(span, total - begin);

    while (left > 0) {
        row = __builtin_amdgcn_readfirstlane(row), head = __builtin_amdgcn_readfirstlane(head), tile = __builtin_amdgcn_readfirstlane(tile);
        const int count = __builtin_amdgcn_readfirstlane((int)min((int64_t)(tiles - tile), left));
        const int first = __builtin_amdgcn_readfirstlane(range.first), end = __builtin_amdgcn_readfirstlane(range.end);
        const int kv_head = head / p.blocks_of_16, block_of_16 = head % p.blocks_of_16;
        const int q_head = kv_head * p.group + 16 * block_of_16, q_heads = min(p.group - 16 * block_of_16, 16);
        const int request = p.row_requests ? p.row_requests[row] : row;
        const int32_t *table = p.table + request * p.table_stride;

        // ---- q, times a power of two that brings its largest value to 2^10 ... 2^11: both parts are then binary16
        // numbers of full precision however large or small the row is
        jl_half8 q_hi[kSteps], q_lo[kSteps];
        float undo;
        {
            floatx4 x[kSteps][2];
            const float *from = p.q + row * p.ldq + (q_head + (m < q_heads ? m : 0)) * DIM;
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
                    const float y = x[s][i / 4][i % 4] * to;
                    q_hi[s][i] = (_Float16)y;
                    q_lo[s][i] = (_Float16)(y - (float)q_hi[s][i]);
                }
        }

        floatx4 o[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) o[b] = floatx4{0.f, 0.f, 0.f, 0.f};
        float top = kNone, sum = 0.f;

        // the pages of a tile's two halves; a half behind the last token, and a page outside the cache, is -1
        auto pages_of = [&](int t, int (&page)[2]) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int token = t * kTile + 16 * h;
                page[h] = token < end ? table[token >> p.cache.page_shift] : -1;
                if ((unsigned)page[h] >= (unsigned)p.cache.pages) page[h] = -1;
            }
        };
        auto part_of = [&](int page) {
            return p.cache.k + ((int64_t)(page < 0 ? 0 : page) * p.cache.kv_heads + kv_head) * p.cache.part_bytes;
        };
        const int in_page_mask = (1 << p.cache.page_shift) - 1;
        Raw<Q8, DIM> raw;
        const int last = first / kTile + tile + count;        // (the list's tiles of a row begin with the one of its first token)
        int t = first / kTile + tile + wave;
        if (t < last) {
            int page[2], next[2] = {-1, -1};
            pages_of(t, page);
#pragma unroll
            for (int h = 0; h < 2; h++) raw.load_k(h, part_of(page[h]), (t * kTile + 16 * h) & in_page_mask, p.cache.page_shift, g, m);
#pragma unroll
            for (int h = 0; h < 2; h++)
                raw.load_v(h, part_of(page[h]) + p.cache.v_offset, (t * kTile + 16 * h) & in_page_mask, p.cache.page_shift, g, m);
            if (t + kWaves < last) pages_of(t + kWaves, next);
            for (; t < last; t += kWaves) {
                const bool more = t + kWaves < last;
                // S
                floatx4 s[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    s[h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < kSteps; i++) {
                        const jl_half8 k = raw.k_operand(h, i);
                        s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q_lo[i], s[h], 0, 0, 0);
                        s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q_hi[i], s[h], 0, 0, 0);
                    }
                }
                // k of the next tile goes out as soon as this one's is used
                if (more) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        raw.load_k(h, part_of(next[h]), ((t + kWaves) * kTile + 16 * h) & in_page_mask, p.cache.page_shift, g, m);
                }
                const bool whole = t * kTile >= first && t * kTile + kTile <= end && page[0] >= 0 && page[1] >= 0;
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = s[i / 4][i % 4] * undo;
                if (!whole) {
                    bool seen[2][4];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int token = t * kTile + 16 * (i / 4) + 4 * g + i % 4;
                        seen[i / 4][i % 4] = token >= first && token < end && page[i / 4] >= 0;
                        x[i] = seen[i / 4][i % 4] ? x[i] : -INFINITY;
                    }
                    raw.mask_v(seen);
                }
                float most = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                most = over_groups_max(most);
                // The maximum may fall behind by a factor of 2^8 before everything is brought to the new one: weights
                // stay far inside binary16, and after a row's first tiles this is rare.
                if (__any(most > top + 8.f)) {
                    const float next_top = fmaxf(top, most);
                    const float keep = __builtin_amdgcn_exp2f(top - next_top);
                    top = next_top;
                    sum *= keep;
#pragma unroll
                    for (int b = 0; b < kBlocks; b++) o[b] *= keep;
                }
                uintx4 hi, lo;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float a = __builtin_amdgcn_exp2f(x[i] - top), b = __builtin_amdgcn_exp2f(x[i + 1] - top);
                    sum += a + b;
                    const auto two = __builtin_amdgcn_cvt_pkrtz(a, b);
                    hi[i / 2] = __builtin_bit_cast(uint32_t, two);
                    lo[i / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a - (float)two[0], b - (float)two[1]));
                }
                const jl_half8 p_hi = __builtin_bit_cast(jl_half8, hi), p_lo = __builtin_bit_cast(jl_half8, lo);
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    const jl_half8 v = raw.v_operand(b);
                    o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p_lo, o[b], 0, 0, 0);
                    o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p_hi, o[b], 0, 0, 0);
                }
                if (more) {
                    page[0] = next[0], page[1] = next[1];
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        raw.load_v(h, part_of(page[h]) + p.cache.v_offset, ((t + kWaves) * kTile + 16 * h) & in_page_mask, p.cache.page_shift, g, m);
                    if (t + 2 * kWaves < last) pages_of(t + 2 * kWaves, next);
                }
            }
        }

        // ---- the four waves' parts into one
        sum = over_groups_sum(sum);
        if (g == 0) joined_max[wave][m] = top, joined_sum[wave][m] = sum;
        __syncthreads();
        const float together = fmaxf(fmaxf(joined_max[0][m], joined_max[1][m]), fmaxf(joined_max[2][m], joined_max[3][m]));
        const float share = __builtin_amdgcn_exp2f(top - together);
        const bool opens = tile == 0, closes = tile + count == tiles;
        float *slot = p.parts + (int64_t)(2 * blockIdx.x + (opens ? 1 : 0)) * (16 * (DIM + 2));
#pragma unroll
        for (int from = 0; from < DIM; from += kRound) {
            if (from > 0) __syncthreads();
            if (m < q_heads) {
#pragma unroll
                for (int b = from / 16; b < (from + kRound) / 16; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) joined[wave][m][out_element<DIM>(b, 4 * g + i) - from] = o[b][i] * share;
            }
            __syncthreads();
            for (int c = 4 * tid; c < q_heads * kRound; c += 4 * kThreads) {
                const int h = c / kRound, d = c % kRound;
                floatx4 v = *(const floatx4 *)&joined[0][h][d] + *(const floatx4 *)&joined[1][h][d] +
                            *(const floatx4 *)&joined[2][h][d] + *(const floatx4 *)&joined[3][h][d];
                if (opens && closes) {
                    const float most = fmaxf(fmaxf(joined_max[0][h], joined_max[1][h]), fmaxf(joined_max[2][h], joined_max[3][h]));
                    float l = 0.f;
#pragma unroll
                    for (int w = 0; w < kWaves; w++) l += joined_sum[w][h] * __builtin_amdgcn_exp2f(joined_max[w][h] - most);
                    v = l == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : v / l;
                    store_out(p, row * p.ldo + (int64_t)(q_head + h) * DIM + from + d, v);
                } else {
                    *(floatx4 *)(slot + h * DIM + from + d) = v;
                }
            }
        }
        if (!(opens && closes) && tid < q_heads) {
            const float most = fmaxf(fmaxf(joined_max[0][tid], joined_max[1][tid]), fmaxf(joined_max[2][tid], joined_max[3][tid]));
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; w++) l += joined_sum[w][tid] * __builtin_amdgcn_exp2f(joined_max[w][tid] - most);
            slot[16 * DIM + tid] = most;
            slot[16 * DIM + 16 + tid] = l;
        }
        if (opens && tid == 0 && (p.by_head || !closes)) {
            Part *cut = p.cut + (p.by_head ? row * heads + head : blockIdx.x);
            const int64_t here = begin + (min(span, total - begin) - left);   // the head's first tile in the list
            *cut = Part{row, head, (int)blockIdx.x, closes ? 0 : (int)((here + tiles - 1) / span) - (int)blockIdx.x + 1};
        }
        __syncthreads();
        left -= count;
        tile = 0;
        if (closes && ++head == heads) {
            head = 0;
            do {
                row++;
                if (row >= p.rows) break;
                range = range_of(p, row);
                tiles = range.tiles();
            } while (tiles == 0);
        }
    }
}

// Joins the parts of the row's head in cut[blockIdx.x], query head blockIdx.y of the sixteen.
template <int DIM>
__global__ void __launch_bounds__(256) jl_kv_attention_join_kernel(AttentionArgs p) {
    constexpr int kLanes = DIM / 4, kSets = 256 / kLanes;      // threads across a row; parts summed side by side
    __shared__ float most[kMostGroups], sums[kMostGroups];
    __shared__ floatx4 folded[kSets][kLanes];
    __shared__ float fold[8];
    const Part cut = p.cut[blockIdx.x];
    if (cut.count <= 0) return;
    const int kv_head = cut.head / p.blocks_of_16, block_of_16 = cut.head % p.blocks_of_16, h = blockIdx.y;
    if (16 * block_of_16 + h >= p.group) return;
    const int tid = threadIdx.x;
    // part 0 is what its span opened, the others what theirs went on with
    auto slot = [&](int part) { return p.parts + (int64_t)(2 * (cut.group + part) + (part == 0 ? 1 : 0)) * (16 * (DIM + 2)); };
    float top = kNone;
    for (int i = tid; i < cut.count; i += 256) {
        most[i] = slot(i)[16 * DIM + h];
        sums[i] = slot(i)[16 * DIM + 16 + h];
        top = fmaxf(top, most[i]);
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, JL_WAVE));
    if (tid % JL_WAVE == 0) fold[tid / JL_WAVE] = top;
    __syncthreads();
    top = fmaxf(fmaxf(fold[0], fold[1]), fmaxf(fold[2], fold[3]));
    const int at = tid % kLanes, set = tid / kLanes;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (set < kSets) {
        for (int i = set; i < cut.count; i += kSets) {
            const float share = __builtin_amdgcn_exp2f(most[i] - top);
            v += share * *(const floatx4 *)(slot(i) + h * DIM + 4 * at);
        }
        folded[set][at] = v;
    }
    for (int i = 0; i < cut.count; i++) l += sums[i] * __builtin_amdgcn_exp2f(most[i] - top);
    __syncthreads();
    if (tid < kLanes) {
        v = folded[0][tid];
        for (int i = 1; i < kSets; i++) v += folded[i][tid];
        v = l == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : v / l;
        store_out(p, cut.row * p.ldo + (int64_t)(kv_head * p.group + 16 * block_of_16 + h) * DIM + 4 * tid, v);
    }
}

template <bool Q8, int DIM>
hipError_t launch(const AttentionArgs &a, int groups, int cuts, hipStream_t stream) {
    hipLaunchKernelGGL((jl_kv_attention_kernel<Q8, DIM>), dim3((unsigned)groups), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((jl_kv_attention_join_kernel<DIM>), dim3((unsigned)cuts, (unsigned)(a.group < 16 ? a.group : 16)), dim3(256), 0,
                       stream, a);
    return hipGetLastError();
}
template <bool Q8>
hipError_t launch_dim(const AttentionArgs &a, int head_dim, int groups, int cuts, hipStream_t stream) {
    switch (head_dim) {
        case 64: return launch<Q8, 64>(a, groups, cuts, stream);
        case 96: return launch<Q8, 96>(a, groups, cuts, stream);
        case 128: return launch<Q8, 128>(a, groups, cuts, stream);
        case 192: return launch<Q8, 192>(a, groups, cuts, stream);
        default: return launch<Q8, 256>(a, groups, cuts, stream);
    }
}

constexpr size_t kCutBytes = kMostGroups * sizeof(Part);

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

extern "C" {

size_t jl_kv_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
    return kCutBytes + (size_t)2 * kMostGroups * 16 * (head_dim + 2) * sizeof(float);
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
    JL_REQUIRE(std::isfinite(scale), "jl_kv_attention: scale %g", (double)scale);
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
    const JlOnDevice on(ctx);
    JL_HIP(on.status);
    AttentionArgs a;
    a.cache = jl_kv_view(cache);
    a.q = q, a.ldq = ldq, a.ldo = ldo;
    a.positions = positions, a.row_requests = row_requests, a.table = block_table;
    a.requests = requests, a.table_stride = table_stride;
    a.scale = scale * 1.44269504088896340736f;
    a.window = window > INT32_MAX ? 0 : (int)window;   // one that reaches behind every position
    a.group = heads / cache->kv_heads;
    a.blocks_of_16 = (a.group + 15) / 16;
    a.rows = (int)rows;
    a.out = out, a.out_f16 = out_f16 != 0;
    a.cut = (Part *)workspace;
    a.parts = (float *)((uint8_t *)workspace + kCutBytes);
    const int groups = std::min(2 * ctx->compute_units, kMostGroups);
    const int64_t row_heads = rows * cache->kv_heads * a.blocks_of_16;
    a.by_head = row_heads <= groups;
    const int cuts = a.by_head ? (int)row_heads : groups;
    JL_HIP(cache->type == JL_KV_Q8_0 ? launch_dim<true>(a, dim, groups, cuts, ctx->stream) : launch_dim<false>(a, dim, groups, cuts, ctx->stream));
    return JL_OK;
}

}  // extern "C"
