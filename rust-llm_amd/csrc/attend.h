// Attention of new tokens over the paged cache (include/rl_mixers.h).
//
// A workgroup takes one key-value head of one sequence, up to 16 RT of its query
// rows (a row of a verify times a query head of the group), and one part of the
// sequence's length; where a length has several parts a second kernel joins them.
// Its four waves take tiles of 32 tokens in turn, each with a running maximum and
// sum of its own:
//   S^T = K Q^T   16x16x32 products, tokens by rows: a lane holds eight scores of
//                 one query row
//   w = 2^(S - m) rounded to 16 bits where it stands: the eight tokens of a lane
//                 are the eight that the next product wants of it
//   O^T += V^T w  values are loaded by token as they lie in the cache and turned
//                 in registers (v_perm), so no LDS and no transposed cache
// K and V of the next tile are loaded as soon as this one's registers are free.
// Per tile and wave the bytes of K and V bound it (HBM); the products of up to 32
// rows hide behind them. One sequence of 131071 tokens, 32 / 8 heads of 128 bf16: 96
// us, 5.5 TB/s (a large copy reaches 4.9, half of it writes). 64 int8 sequences of
// 2048: 58 us, 4.7 TB/s; of 128 to 8192: 70 us, 3.8 TB/s, since their parts differ in
// size. 611 tokens of 4 heads of 256: 10 us, the chain of lengths, pages, keys,
// values and joins.
#pragma once
#include "kv_cache.h"

namespace rl {

struct AttendArgs {
    CacheArgs cache;
    const void *q;
    void *out;
    float *lse;
    uint64_t q_row, q_head, out_row, out_head;
    const int32_t *starts, *lens, *pages;
    uint32_t rows, seqs, q_heads, table_width, window, most_rows, max_len;
    float scale;
    uint32_t group;       // query heads of a key-value head
    uint32_t blocks;      // row blocks a sequence, or with `packed` of all
    uint32_t packed;      // whether a workgroup's sequence is found from its row block
    uint32_t part_tiles;  // tiles of 32 tokens a part
    uint32_t wide;        // whether q and out are aligned for 16-byte accesses
    float *part_out;      // [row * q_heads + head][part][HD]: sums of the weighted values
    float2 *part_sum;     // [row * q_heads + head][part]: maximum and sum
    uint32_t *part_count; // [row * q_heads + head]: parts to join, and ATTEND_NONE if the row sees nothing or has no prefix; zero between calls
    uint32_t parts;       // parts a row has room for
    uint32_t *arrived;    // [row * q_heads + head], of a block's first: its parts that are done; zero between calls
    uint32_t group_inv, blocks_inv, columns_inv, heads_inv, tiles_inv; // inverse_of group, blocks, seqs * kv heads, kv heads, part_tiles
    uint32_t joins;       // whether the last part's workgroup joins them (ATTEND_JOINED: the only one, with the prefix's), else k_attend_join does
    // Shared prefixes. The rows of a group's sequences group_starts[g] .. group_starts[g + 1] see all of its prefix: part p
    // of it is partial result `shared` + p of their `stride`, with a maximum of -inf where it has no tokens.
    const int32_t *group_starts;
    uint32_t shared, shared_parts, stride, group_end; // group_end: the call's sequences (ATTEND_PREFIX), its groups (ATTEND_JOINED)
};

// What a launch does: sequences by themselves; the prefixes of groups of sequences, in which `seqs`, `lens`, `pages` and
// `max_len` are the groups' and their prefixes'; sequences whose rows have a prefix's partial results beside their own.
enum AttendMode { ATTEND_ALONE, ATTEND_PREFIX, ATTEND_JOINED };

constexpr uint32_t ATTEND_THREADS = 256, ATTEND_WAVES = 4, ATTEND_TILE = 32;
// Row blocks side by side, where those of a batch are counted through: eight of a run are on one XCD, whose L2 then has the
// keys and values for all but the first.
constexpr uint32_t ATTEND_RUN = 8;
constexpr uint32_t ATTEND_MAX_PARTS = 256, ATTEND_NONE = 1u << 31;
// Parts that the last of their workgroups joins, which saves a launch (one sequence of 611 tokens, 5 parts: 11.2 us with
// it, 10.1 without); more are too much for one CU (21 parts of 16 rows of 256: 31.4 us with the launch, 40.5 without).
constexpr uint32_t ATTEND_FEW = 16;
constexpr int ATTEND_STORED = 0x0F70; // s_waitcnt vmcnt(0)

constexpr int attend_dim(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Whether a workgroup takes two row tiles of `count` that a sequence has: keys and values are read once for both, but
// fewer workgroups share a CU. bf16 queries, us, two / one, sequences x tokens, query / key-value heads x dim:
//   64:  1 x 20011 tokens, 16/8, 18 rows 15.7 / 17.5, 36 rows 19.0 / 20.0; 32 x 3001 37.8 / 42.7, 53.2 / 59.7
//   128: a tile left over costs a block's time (32 x 3001, 32/8, 36 rows: bf16 137 / 118, int8 84.6 / 80.9); else int8
//        20 rows 45.6 / 57.3, 64 rows 86.4 / 104, bf16 83.2 / 89.9, 134 / 144, with columns for half the CUs or fewer
//        (4 x 8001) bf16 30.2 / 29.1, 58.9 / 48.6
//   256: the sums take the registers (32 x 3001, 16/4, 32 rows of int8 61.5 / 53.9)
inline bool attend_two(uint32_t format, uint32_t dim, uint64_t count, uint64_t columns) {
    if (count < 2 || attend_dim(dim) == 256) return false;
    if (attend_dim(dim) == 64) return true;
    return count % 2 == 0 && (format == RL_I8 || format == RL_F8 || columns >= 256);
}

// Workgroups of k_attend that share a CU: as many as its registers allow without spills.
constexpr int attend_resident(uint32_t query_bytes, uint32_t format, uint32_t dim, int row_tiles) {
    const bool eight = format == RL_I8 || format == RL_F8;
    switch (attend_dim(dim)) {
    case 64: return row_tiles == 1 ? 3 : 2;
    case 128: return row_tiles == 1 ? (eight && query_bytes == 2 ? 3 : 2) : eight ? 2 : 1;
    default: return eight ? 2 : 1;
    }
}

typedef vec<uint32_t, 4> u32x4;

__device__ inline f32x4 mfma(vec<half_t, 8> a, vec<half_t, 8> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma(vec<bhalf_t, 8> a, vec<bhalf_t, 8> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The sequence's rows, and what a row sees: [begin, end). len is 0 or more and n at most 2^23, so no sum here leaves 32
// bits; tokens past a tile's or a block's end are counted unsigned, since len may be the largest.
template <AttendMode MODE>
struct AttendSpan {
    int32_t len, n, window;
    __device__ int32_t end(int32_t i) const { return MODE == ATTEND_PREFIX ? len : max(len - n + i + 1, 0); }
    __device__ int32_t begin(int32_t i) const { return MODE == ATTEND_ALONE && window ? max(end(i) - window, 0) : 0; }
};

// Two 8-bit codes, the low or high half of u, as two 16-bit values. Keys: int8 codes lie in the cache with their sign
// bit flipped, and 0x6400 | b is 1024 + b in f16, so each reads as the code and 1152, exactly. The 1152 comes off each key
// before its product, again exactly: taken off the finished score as 1152 sum q it costs a score what f32 sums of numbers
// a hundred times the codes lose, 2e-4 for queries of mean 0 and 1e-2 for a mean of 8 (256 dims).
constexpr float KEY_BIAS = 1152.0f;
template <int FMT, bool HIGH>
__device__ inline uint32_t pair_f16(uint32_t u) {
    if constexpr (FMT == RL_F8) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, HIGH));
    else return __builtin_amdgcn_perm(0x64646464u, u, HIGH ? 0x04030402u : 0x04010400u);
}
template <int FMT, bool HIGH>
__device__ inline uint32_t pair_bf16(uint32_t u) {
    if constexpr (FMT == RL_F8) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, HIGH));
    } else {
        const vec<bhalf_t, 2> w = {(bhalf_t)(float)(int8_t)(u >> (HIGH ? 16 : 0)),
                                   (bhalf_t)(float)(int8_t)(u >> (HIGH ? 24 : 8))};
        return __builtin_bit_cast(uint32_t, w);
    }
}

// Two values that workgroups on other XCDs read, or have written, in this launch.
__device__ inline void shared_store(float *p, float2 x) {
    __hip_atomic_store((uint64_t *)p, __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float2 shared_load(const float *p) {
    return __builtin_bit_cast(float2, __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Four columns of a finished row: its weighted values over its sum, which holds the
// weights at 2^LIFT times their size.
constexpr float ATTEND_LIFT = 8.0f;
template <typename T>
__device__ inline void attend_write(const AttendArgs &a, uint64_t row, uint64_t head, uint32_t d, bool none, float2 ms,
                                    f32x4 x, float lift) {
    if (d >= a.cache.dim) return;
    none = none && !(ms.y != ms.y);
    float y[4];
#pragma unroll
    for (int c = 0; c < 4; c++) y[c] = none ? 0.0f : x[c] / ms.y;
    store_f32((T *)a.out + row * a.out_row + head * a.out_head + d, a.wide, y);
    if (d == 0 && a.lse)
        a.lse[row * a.q_heads + head] = none ? -INFINITY : ((ms.x - lift) + log2f(ms.y)) * 0.693147180559945309f;
}

// One partial result more of four columns of a row, at its maximum and sum.
__device__ inline void attend_add(float2 &ms, f32x4 &x, float2 more, f32x4 y) {
    if (more.x == -INFINITY && more.y == 0.0f) return; // no tokens: its columns may be anything
    const float most = fmaxf(ms.x, more.x), f = ms.x == -INFINITY ? 1.0f : exp2_fast(ms.x - most), g = exp2_fast(more.x - most);
    ms = make_float2(most, ms.y * f + more.y * g);
    x = x * f + y * g;
}

// The maximum of a part whose tokens all have scores of -inf: it has tokens, but no weight beside any other.
constexpr float ATTEND_LOWEST = -3.402823466e38f;

// What workgroup `number` of a launch does is in attend_body.h, which k_attend and attend_block have each as their own text:
// with the function inlined, k_attend took 2 % longer (one row over 611 tokens of 256 dims 9.95 -> 10.25 us).
template <typename T, int FMT, int HD, int RT, bool P16, AttendMode MODE>
__global__ void __launch_bounds__(ATTEND_THREADS, attend_resident(sizeof(T), FMT, HD, RT)) k_attend(AttendArgs a) {
    const uint32_t number = blockIdx.x;
#include "attend_body.h"
}

template <typename T, int FMT, int HD, int RT, bool P16, AttendMode MODE>
__device__ __forceinline__ void attend_block(AttendArgs a, uint32_t number) {
#include "attend_body.h"
}

// Prefixes and the sequences' own tokens side by side, for calls too small to fill the device with either: k_attend_join
// then joins both. `groups`: workgroups of the prefixes.
template <typename T, int FMT, int HD, bool P16>
__global__ void __launch_bounds__(ATTEND_THREADS, HD == 256 ? 1 : attend_resident(sizeof(T), FMT, HD, 1)) k_attend_both(AttendArgs prefix, AttendArgs own, uint32_t groups) {
    if (blockIdx.x < groups) attend_block<T, FMT, HD, 1, P16, ATTEND_PREFIX>(prefix, blockIdx.x);
    else attend_block<T, FMT, HD, 1, P16, ATTEND_JOINED>(own, blockIdx.x - groups);
}

// Joins the parts of a row and head where they are more than ATTEND_FEW: one
// workgroup each, a thread four columns of every PER-th part, all loaded before the
// first is needed. Latency only: 4.2 us for 64 parts of 32 rows of 128.
template <typename T, int FMT, int HD, AttendMode MODE>
__global__ void __launch_bounds__(ATTEND_THREADS) k_attend_join(AttendArgs a) {
    constexpr uint32_t COLS = HD / 4, PER = ATTEND_THREADS / COLS, AHEAD = 8;
    __shared__ float factor[ATTEND_MAX_PARTS], reduce[2][ATTEND_WAVES];
    __shared__ f32x4 partial[PER][COLS];
    const uint64_t at = blockIdx.x;
    constexpr bool JOINED = MODE == ATTEND_JOINED;
    const uint32_t tid = threadIdx.x, count = a.part_count[at], own = min(count & ~ATTEND_NONE, a.parts);
    if (!own) return; // written already, or no sequence's
    const uint32_t n = own + (JOINED && !(count & ATTEND_NONE) ? a.shared_parts : 0), stride = JOINED ? a.stride : a.parts;
    const uint32_t c = tid % COLS, p0 = tid / COLS;
    const f32x4 *x = (const f32x4 *)(a.part_out + at * stride * HD) + c;
    const auto slot = [&](uint32_t p) { return JOINED && p >= own ? a.shared + (p - own) : p; };
    f32x4 ahead[AHEAD];
#pragma unroll
    for (uint32_t j = 0; j < AHEAD; j++) {
        const uint32_t p = p0 + j * PER;
        ahead[j] = x[(uint64_t)slot(p < n ? p : 0) * COLS];
    }
    const float2 ms = tid < n ? a.part_sum[at * stride + slot(tid)] : make_float2(-INFINITY, 0.0f);
    float most = group_max<64>(ms.x);
    if (tid % 64 == 0) reduce[0][tid / 64] = most;
    __syncthreads();
    if (tid == 0) a.part_count[at] = 0;
    most = fmaxf(fmaxf(reduce[0][0], reduce[0][1]), fmaxf(reduce[0][2], reduce[0][3]));
    const float f = ms.x == -INFINITY ? 0.0f : exp2_fast(ms.x - most);
    factor[tid] = f;
    float sum = group_sum<64>(ms.x == -INFINITY ? ms.y : ms.y * f); // a part without tokens has 0, or NaN
    if (tid % 64 == 0) reduce[1][tid / 64] = sum;
    __syncthreads();
    sum = reduce[1][0] + reduce[1][1] + reduce[1][2] + reduce[1][3];
    f32x4 total = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t j = 0; j < AHEAD; j++)
        if (p0 + j * PER < n && (!JOINED || factor[p0 + j * PER] != 0.0f)) total += ahead[j] * factor[p0 + j * PER];
    for (uint32_t p = p0 + AHEAD * PER; p < n; p += PER)
        if (!JOINED || factor[p] != 0.0f) total += x[(uint64_t)slot(p) * COLS] * factor[p]; // of no tokens: may be anything
    partial[p0][c] = total;
    __syncthreads();
    if (p0) return;
#pragma unroll
    for (uint32_t j = 1; j < PER; j++) total += partial[j][c];
    attend_write<T>(a, at / a.q_heads, at % a.q_heads, c * 4, JOINED ? most == -INFINITY : (count & ATTEND_NONE) != 0, make_float2(most, sum), total,
                    FMT == RL_F16 ? ATTEND_LIFT : 0.0f);
}

// Launches the kernel for queries of type T (attend_*.hip, one unit a type).
template <typename T>
void launch_attend(const AttendArgs &a, AttendMode mode, uint32_t format, uint32_t row_tiles, uint32_t groups, hipStream_t s);
template <typename T>
void launch_attend_both(const AttendArgs &prefix, const AttendArgs &own, uint32_t format, uint32_t prefix_groups, uint32_t own_groups,
                        hipStream_t s);

}  // namespace rl
