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
    uint32_t joins;       // whether the last part's workgroup joins them, else k_attend_join does
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

template <typename T, int FMT, int HD, int RT, bool P16, AttendMode MODE>
__global__ void __launch_bounds__(ATTEND_THREADS, attend_resident(sizeof(T), FMT, HD, RT)) k_attend(AttendArgs a) {
    constexpr bool EIGHT = FMT == RL_I8 || FMT == RL_F8, F32Q = sizeof(T) == 4;
    // Element types of the two products. 8-bit codes are exact in either; queries fit f16 scaled by a power of two
    // (below), weights times a value's step need bf16's range.
    using MK = std::conditional_t<FMT == RL_BF16, bhalf_t, half_t>;
    using MV = std::conditional_t<FMT == RL_F16, half_t, bhalf_t>;
    // f32 queries are split into parts that add up to them (24 bits in three bf16 parts, 22 in two of f16), and so are
    // the weights of f32 outputs. Those of 16-bit outputs are two parts too (16 or 22 bits): one alone, of 8 bits, cost as
    // much as the output's own rounding (0.0025 off f64 against 0.0017 over 64 int8 sequences), and a second product
    // hides behind the loads.
    constexpr int QP = !F32Q ? 1 : std::is_same_v<MK, bhalf_t> ? 3 : 2, PP = F32Q && std::is_same_v<MV, bhalf_t> ? 3 : 2;
    constexpr int ROWS = 16 * RT, VD = HD / 16, SIZE = EIGHT ? 1 : 2;
    constexpr int KC = HD * SIZE / 64;        // 64-byte chunks of a key
    constexpr int VW = VD * SIZE / 4;         // dwords of a value that a lane holds
    constexpr int STEPS = HD / 32;            // products a score tile
    constexpr float LIFT = FMT == RL_F16 ? ATTEND_LIFT : 0.0f; // weights up to 2^8: their second f16 parts stay normal
    constexpr bool Q_REGS = RT * QP * STEPS <= 4;
    constexpr int QS = HD + 8;
    constexpr size_t Q_BYTES = (size_t)QP * ROWS * QS * 2, O_BYTES = (size_t)ATTEND_WAVES * 16 * (HD + 4) * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
    __shared__ float mults[ROWS], maxima[ATTEND_WAVES][ROWS], sums[ATTEND_WAVES][ROWS];
    __shared__ bool last;

    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const uint32_t G = a.group;
    // Not written while the kernel runs: read through the scalar cache where the index is the wave's.
    typedef const __attribute__((address_space(4))) int32_t constant_i32;
    const constant_i32 *starts = (constant_i32 *)(uintptr_t)a.starts, *lens = (constant_i32 *)(uintptr_t)a.lens;
    // The first row of sequence or group i.
    const auto first_of = [&](uint32_t i) {
        if constexpr (MODE == ATTEND_PREFIX) {
            const int32_t at = min(max(((constant_i32 *)(uintptr_t)a.group_starts)[i], 0), (int32_t)a.group_end);
            return starts ? starts[at] : at;
        } else
            return starts ? starts[i] : (int32_t)i;
    };
    uint32_t s, head, part, block;
    if (a.packed) {
        const uint32_t y = blockIdx.x / 8, at = (y / ATTEND_RUN * 8 + blockIdx.x % 8) * ATTEND_RUN + y % ATTEND_RUN;
        const uint2 column = split_by(at, a.blocks, a.blocks_inv), of = split_by(column.x, a.cache.heads, a.heads_inv);
        const uint32_t b = column.y;
        part = of.x, head = of.y;
        if (part >= a.parts) return;
        // The last sequence whose row blocks begin at or before this one; no two begin at the same.
        const auto first_block = [&](uint32_t i) { return (uint32_t)min(max(first_of(i), 0), (int32_t)a.rows) * G / ROWS + i; };
        s = 0;
        for (uint32_t hi = a.seqs; hi - s > 1;) {
            const uint32_t mid = s + (hi - s) / 2;
            if (first_block(mid) <= b) s = mid;
            else hi = mid;
        }
        if (first_block(s) > b) return;
        block = b - first_block(s);
    } else {
        // The row blocks of one sequence, head and part are eight workgroups apart: on one XCD.
        const uint2 eight = split_by(blockIdx.x / 8, a.blocks, a.blocks_inv);
        const uint2 job = split_by(eight.x * 8 + blockIdx.x % 8, a.seqs * a.cache.heads, a.columns_inv);
        const uint2 of = split_by(job.y, a.cache.heads, a.heads_inv);
        block = eight.y, part = job.x, s = of.x, head = of.y;
        if (part >= a.parts) return;
    }
    const int32_t first = first_of(s);
    uint32_t shared_parts = 0; // of the sequence's prefix
    if constexpr (MODE == ATTEND_JOINED) {
        const constant_i32 *group_starts = (constant_i32 *)(uintptr_t)a.group_starts;
        if ((int32_t)s >= group_starts[0] && (int32_t)s < group_starts[a.group_end]) shared_parts = a.shared_parts;
    }
    const int64_t rows = MODE == ATTEND_PREFIX ? (int64_t)first_of(s + 1) - first : starts ? (int64_t)starts[s + 1] - first : 1;
    if (rows <= 0 || first < 0 || first + rows > a.rows) return; // no rows, or `starts` is not what it should be
    AttendSpan<MODE> span{max(lens[s], 0), (int32_t)rows, (int32_t)a.window}; // a negative length is none
    const uint32_t expanded = (uint32_t)span.n * G;
    const int32_t longest = span.end(span.n - 1);
    const uint32_t page = a.cache.page;
    // What the call's bounds or the page table do not cover is NaN, written once.
    if ((uint32_t)span.n > a.most_rows || span.len > (int64_t)a.max_len ||
        (longest > 0 && split_by(longest - 1, page, a.cache.page_inv).x >= a.table_width)) {
        if (part || block) return;
        const uint32_t dim = a.cache.dim;
        for (uint64_t i = tid; i < (uint64_t)expanded * dim; i += ATTEND_THREADS) {
            const uint32_t e = (uint32_t)(i / dim), d = (uint32_t)(i - (uint64_t)e * dim);
            const uint64_t row = first + e / G, qh = head * G + e % G;
            if constexpr (MODE == ATTEND_PREFIX) { // one part that is NaN, and no others
                if (d < a.shared_parts)
                    a.part_sum[(row * a.q_heads + qh) * a.stride + a.shared + d] = d ? make_float2(-INFINITY, 0.0f) : make_float2(0.0f, NAN);
                continue;
            }
            ((T *)a.out)[row * a.out_row + qh * a.out_head + d] = (T)NAN;
            if (d == 0 && a.lse) a.lse[row * a.q_heads + qh] = NAN;
        }
        return;
    }
    if (block >= (expanded + ROWS - 1) / ROWS) return;
    const uint32_t r0 = block * ROWS;
    const uint32_t count = min(expanded - r0, (uint32_t)ROWS);
    const auto by_group = [&](uint32_t e) { return split_by(e, G, a.group_inv); }; // (query row, query head of the group)
    const int32_t i0 = by_group(r0).x, i1 = by_group(r0 + count - 1).x; // query rows of the block
    const int32_t begin_min = span.begin(i0), begin_max = span.begin(i1), end_min = span.end(i0), end_max = span.end(i1);
    const bool mixed = begin_min != begin_max || end_min != end_max;
    const int32_t tile0 = begin_min / (int)ATTEND_TILE, tiles = (int32_t)((end_max + ATTEND_TILE - 1) / ATTEND_TILE) - tile0;
    const uint32_t parts = tiles > 0 ? split_by(tiles + a.part_tiles - 1, a.part_tiles, a.tiles_inv).x : 1; // of this block
    if (part >= parts) {
        if constexpr (MODE == ATTEND_PREFIX) // nothing here
            for (uint32_t i = tid; i < count; i += ATTEND_THREADS) {
                const uint2 e = by_group(r0 + i);
                a.part_sum[((uint64_t)(first + e.x) * a.q_heads + head * G + e.y) * a.stride + a.shared + part] = make_float2(-INFINITY, 0.0f);
            }
        return;
    }

    // The block's queries, a few values a thread; they go to LDS while the first tile is on its way.
    constexpr uint32_t TPR = ATTEND_THREADS / ROWS, EPT = HD / TPR;
    const uint32_t q_row = tid / TPR, q_at = tid % TPR * EPT;
    float x[EPT] = {};
    if (q_row < count) {
        const uint2 e = by_group(r0 + q_row);
        const T *q = (const T *)a.q + (uint64_t)(first + e.x) * a.q_row + (uint64_t)(head * G + e.y) * a.q_head;
#pragma unroll
        for (uint32_t j = 0; j < EPT; j += 4)
            if (q_at + j < a.cache.dim) { // dim is a multiple of 16
                float y[4];
                load_f32(q + q_at + j, a.wide, y);
#pragma unroll
                for (int c = 0; c < 4; c++) x[j + c] = y[c];
            }
    }

    const uint32_t col = lane % 16, quad = lane / 16;
    f32x4 O[RT][VD];
    float top[RT], total[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        top[rt] = -INFINITY, total[rt] = 0.0f;
#pragma unroll
        for (int m = 0; m < VD; m++) O[rt][m] = f32x4{0, 0, 0, 0};
    }

    const uint32_t dim_bytes = a.cache.dim * SIZE;
    const uint8_t *keys = (const uint8_t *)a.cache.keys, *values = (const uint8_t *)a.cache.values;
    const auto *table = (constant_i32 *)(uintptr_t)(a.pages + (uint64_t)s * a.table_width);
    const uint32_t pool = (uint32_t)(a.cache.slots / page);
    bool poison = false; // a page number that is none

    u32x4 kr[2][KC];
    uint32_t vr[8][VW];
    f32x4 ks[2], vs[2];

    // Where a tile's tokens lie. P16 (pages of a multiple of 16 tokens): each half of a tile lies in one page, at[u] is
    // its first vector. Else lane l has the vector of token l % 32. Tokens that no row sees, whose pages are not looked
    // up, are the nearest that some row does: what is loaded for them is masked, and no load is conditional.
    // Page numbers are fetched two tiles ahead, before the keys of the next: waiting for them waits for nothing newer.
    struct Place {
        uint64_t at[2];
    };
    struct Pages {
        uint32_t id[2];
    };
    auto in_sight = [&](int32_t t) {
        return (uint32_t)(P16 ? min(max(t, begin_min & ~15), (end_max - 1) & ~15) : min(max(t, begin_min), end_max - 1));
    };
    auto fetch = [&](int32_t t0) {
        Pages p{{0, 0}};
#pragma unroll
        for (int u = 0; u < (P16 ? 2 : 1); u++)
            p.id[u] = (uint32_t)table[split_by(in_sight(t0 + (P16 ? 16 * u : (int)(lane % 32))), page, a.cache.page_inv).x];
        return p;
    };
    auto place = [&](int32_t t0, const Pages &p) {
        Place w{{0, 0}};
#pragma unroll
        for (int u = 0; u < (P16 ? 2 : 1); u++) {
            const uint32_t t = in_sight(t0 + (P16 ? 16 * u : (int)(lane % 32)));
            poison |= p.id[u] >= pool;
            w.at[u] = ((uint64_t)(p.id[u] < pool ? p.id[u] : 0) * a.cache.heads + head) * page + split_by(t, page, a.cache.page_inv).y;
        }
        return w;
    };
    auto vector_at = [&](const Place &w, uint32_t token) -> uint64_t { // token of the tile
        if constexpr (P16) return w.at[token / 16] + token % 16;
        else return __shfl(w.at[0], token);
    };
    // Lanes past the head's end load its start: as keys they are zeroed before use, as values they are columns that are
    // not written.
    auto load_keys = [&](const Place &w) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint8_t *p = keys + (P16 ? w.at[u] * dim_bytes + col * dim_bytes : vector_at(w, 16 * u + col) * dim_bytes);
#pragma unroll
            for (uint32_t c = 0; c < KC; c++) {
                const uint32_t at = c * 64 + quad * 16;
                kr[u][c] = *(const u32x4 *)(p + (at < dim_bytes ? at : 0));
            }
            if constexpr (EIGHT) {
                if constexpr (P16) ks[u] = *(const f32x4 *)(a.cache.key_steps + w.at[u] + quad * 4);
                else
#pragma unroll
                    for (int i = 0; i < 4; i++) ks[u][i] = a.cache.key_steps[vector_at(w, 16 * u + quad * 4 + i)];
            }
        }
    };
    auto load_values = [&](const Place &w) {
        constexpr int PER = VW < 4 ? VW : 4;
        const uint32_t at = col * VW * 4 < dim_bytes ? col * VW * 4 : 0; // dim is a multiple of 16: a lane has all or none
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint64_t v = P16 ? w.at[j / 4] : vector_at(w, j / 4 * 16 + quad * 4 + j % 4);
            const uint8_t *p = values + (P16 ? v * dim_bytes + (quad * 4 + j % 4) * dim_bytes : v * dim_bytes) + at;
#pragma unroll
            for (int c = 0; c < VW; c += PER) {
                const vec<uint32_t, PER> x = *(const vec<uint32_t, PER> *)(p + c * 4);
#pragma unroll
                for (int e = 0; e < PER; e++) vr[j][c + e] = x[e];
            }
            if constexpr (EIGHT && !P16) vs[j / 4][j % 4] = a.cache.value_steps[v];
        }
        if constexpr (EIGHT && P16) {
#pragma unroll
            for (int u = 0; u < 2; u++) vs[u] = *(const f32x4 *)(a.cache.value_steps + w.at[u] + quad * 4);
        }
    };

    // The product with the values: for each of a lane's VD columns the eight tokens' values, column by column.
    auto multiply = [&](const u32x4 &v, const vec<MV, 8> (&w)[RT][PP], int column) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int p = 0; p < PP; p++)
                O[rt][column] = mfma(__builtin_bit_cast(vec<MV, 8>, v), w[rt][p], O[rt][column]);
    };
    // f(values of eight tokens, column) for each of a lane's columns.
    auto each_column = [&](auto f) {
        if constexpr (!EIGHT) {
#pragma unroll
            for (int c = 0; c < VW; c++) {
                u32x4 lo, hi;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    lo[j] = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x05040100u);
                    hi[j] = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x07060302u);
                }
                f(lo, 2 * c);
                f(hi, 2 * c + 1);
            }
        } else {
#pragma unroll
            for (int c = 0; c < VW; c++) {
                u32x4 x[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t lo = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x05010400u);
                    const uint32_t hi = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x07030602u);
                    x[0][j] = pair_bf16<FMT, false>(lo);
                    x[1][j] = pair_bf16<FMT, true>(lo);
                    x[2][j] = pair_bf16<FMT, false>(hi);
                    x[3][j] = pair_bf16<FMT, true>(hi);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) f(x[e], 4 * c + e);
            }
        }
    };

    const int32_t part_begin = tile0 + (int32_t)(part * a.part_tiles);
    const int32_t part_end = min(part_begin + (int32_t)a.part_tiles, tile0 + tiles);
    int32_t tile = part_begin + (int32_t)wave;
    Pages ahead{{0, 0}}; // of this wave's next tile
    if (tile < part_end) {
        // In the order of the loop's own loads: a wait in the loop has to hold for the first tile too.
        const int32_t t0 = tile * (int)ATTEND_TILE;
        const Pages now = fetch(t0);
        ahead = fetch((int32_t)(t0 + ATTEND_WAVES * ATTEND_TILE)); // may be past the last token, and past 2^31: any in sight
        const Place at = place(t0, now);
        __builtin_amdgcn_sched_barrier(0);
        load_keys(at);
        __builtin_amdgcn_sched_barrier(0);
        load_values(at);
        __builtin_amdgcn_sched_barrier(0);
    }
    // Queries into LDS in the type of the product. In f16 a row is scaled by the power of two that brings its largest
    // value to [1, 2), which costs nothing of its values down to 2^-24 of the largest.
    {
        MK *qs = (MK *)lds;
        float unit = 1.0f;
        if constexpr (std::is_same_v<MK, half_t>) {
            float m = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < EPT; j++) m = fmaxf(m, fabsf(x[j]));
            m = group_max<TPR>(m);
            // 2^-e for m in [2^e, 2^(e+1)); the bounds keep it and its inverse normal.
            const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 100);
            const float down = __uint_as_float((uint32_t)(127 - e) << 23);
            unit = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (uint32_t j = 0; j < EPT; j++) x[j] *= down;
        }
#pragma unroll
        for (int p = 0; p < QP; p++)
#pragma unroll
            for (uint32_t j = 0; j < EPT; j++) {
                const MK y = (MK)x[j];
                qs[(p * ROWS + q_row) * QS + q_at + j] = y;
                x[j] -= (float)y;
            }
        if (tid % TPR == 0) mults[q_row] = a.scale * 1.44269504088896341f * unit;
    }
    __syncthreads();
    const MK *qs = (const MK *)lds;
    // Contraction order of a product: 16-bit keys 32 dims in order, 8-bit ones the first or second half of each lane's
    // 16 bytes. Queries follow it.
    auto q_fragment = [&](int rt, int p, int st) {
        const uint32_t d = EIGHT ? st / 2 * 64 + quad * 16 + st % 2 * 8 : st * 32 + quad * 8;
        return *(const vec<MK, 8> *)(qs + (p * ROWS + rt * 16 + col) * QS + d);
    };
    vec<MK, 8> qf[Q_REGS ? RT : 1][Q_REGS ? QP : 1][Q_REGS ? STEPS : 1];
    if constexpr (Q_REGS) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int p = 0; p < QP; p++)
#pragma unroll
                for (int st = 0; st < STEPS; st++) qf[rt][p][st] = q_fragment(rt, p, st);
    }
    float mult[RT];
    int32_t row_begin[RT], row_end[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t r = rt * 16 + col;
        mult[rt] = mults[r];
        const int32_t i = r < count ? by_group(r0 + r).x : 0;
        row_begin[rt] = r < count ? span.begin(i) : begin_min; // rows past the block's see what any of it sees
        row_end[rt] = r < count ? span.end(i) : end_max;
    }
    // A tile; with `more` the next one's loads go out as their registers become free. That is known to the compiler, so
    // that a wait for this tile's values leaves the next one's keys on their way.
    auto step = [&](auto more) {
        constexpr bool MORE = decltype(more)::value;
        const int32_t t0 = tile * (int)ATTEND_TILE;
        f32x4 S[RT][2];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int rt = 0; rt < RT; rt++) S[rt][u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            vec<MK, 8> k[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if constexpr (EIGHT) {
                    const uint32_t x = kr[u][st / 2][st % 2 * 2], y = kr[u][st / 2][st % 2 * 2 + 1];
                    const u32x4 w = {pair_f16<FMT, false>(x), pair_f16<FMT, true>(x), pair_f16<FMT, false>(y), pair_f16<FMT, true>(y)};
                    k[u] = __builtin_bit_cast(vec<MK, 8>, w);
                    if constexpr (FMT == RL_I8) k[u] -= (MK)KEY_BIAS;
                } else {
                    k[u] = __builtin_bit_cast(vec<MK, 8>, kr[u][st]);
                    // Queries are zeros past the head's end; 16-bit keys may hold what a zero does not cancel.
                    if (a.cache.dim != HD && st * 64 + quad * 16 >= dim_bytes) k[u] = vec<MK, 8>{};
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int p = 0; p < QP; p++) {
                    vec<MK, 8> q;
                    if constexpr (Q_REGS) q = qf[rt][p][st];
                    else q = q_fragment(rt, p, st);
#pragma unroll
                    for (int u = 0; u < 2; u++) S[rt][u] = mfma(k[u], q, S[rt][u]);
                }
        }
        const f32x4 step[2] = {ks[0], ks[1]};
        Place next{{0, 0}};
        if constexpr (MORE) {
            const int32_t t1 = t0 + (int)(ATTEND_WAVES * ATTEND_TILE);
            next = place(t1, ahead);
            ahead = fetch((int32_t)(t1 + ATTEND_WAVES * ATTEND_TILE));
            __builtin_amdgcn_sched_barrier(0);
            load_keys(next);
            __builtin_amdgcn_sched_barrier(0);
        }
        // A tile that some row of the block does not see all of.
        const bool edge = t0 < begin_max || end_min - t0 < (int)ATTEND_TILE;
        vec<MV, 8> w[RT][PP];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float x[8], most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (EIGHT) x[j] = S[rt][j / 4][j % 4] * (step[j / 4][j % 4] * mult[rt]);
                else x[j] = S[rt][j / 4][j % 4] * mult[rt];
                if (edge) {
                    const int32_t t = t0 + j / 4 * 16 + (int)quad * 4 + j % 4;
                    if (t < row_begin[rt] || t >= row_end[rt]) x[j] = -INFINITY;
                }
                most = fmaxf(most, x[j]);
            }
            most = fmaxf(rows_max(most), top[rt]);
            if (__any(most > top[rt])) {
                const float keep = most == -INFINITY ? 1.0f : exp2_fast(top[rt] - most);
                total[rt] *= keep;
#pragma unroll
                for (int m = 0; m < VD; m++) O[rt][m] *= keep;
                top[rt] = most;
            }
            const float base = (most == -INFINITY ? 0.0f : most) - LIFT;
            float rest[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float p = exp2_fast(x[j] - base);
                total[rt] += p;
                if constexpr (EIGHT) {
                    p *= vs[j / 4][j % 4];
                    if (edge && x[j] == -INFINITY) p = 0.0f; // whatever the step of an unseen token is
                }
                rest[j] = p;
            }
            if constexpr (std::is_same_v<MV, bhalf_t>) { // the first part cut off, not rounded: a mask, and one v_perm for two
                u32x4 cut;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const uint32_t u0 = __float_as_uint(rest[j]), u1 = __float_as_uint(rest[j + 1]);
                    cut[j / 2] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
                    rest[j] -= __uint_as_float(u0 & 0xFFFF0000u);
                    rest[j + 1] -= __uint_as_float(u1 & 0xFFFF0000u);
                }
                w[rt][0] = __builtin_bit_cast(vec<MV, 8>, cut);
            } else
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    w[rt][0][j] = (MV)rest[j];
                    rest[j] -= (float)w[rt][0][j];
                }
#pragma unroll
            for (int i = 1; i < PP; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    w[rt][i][j] = (MV)rest[j];
                    rest[j] -= (float)w[rt][i][j];
                }
        }
        bool stray = false;
        constexpr uint32_t E = std::is_same_v<MV, half_t> ? 0x7C00u : 0x7F80u; // the exponent of what is not finite
        if constexpr (!EIGHT) {
            if (edge) { // values that no row sees may be anything: zeros; one that is not finite may only reach the rows that see it
                uint32_t odd = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int32_t t = t0 + j / 4 * 16 + (int)quad * 4 + j % 4;
                    const bool out = t < begin_min || t >= end_max;
#pragma unroll
                    for (int c = 0; c < VW; c++) {
                        if (out) vr[j][c] = 0;
                        odd |= (vr[j][c] & E) == E || (vr[j][c] >> 16 & E) == E;
                    }
                }
                stray = mixed && __any(odd);
            }
        }
        if (__builtin_expect(stray, 0)) {
            // Such values take part as zeros, and a second product counts those that a row sees: NaN where it sees any.
            vec<MV, 8> sees[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int32_t t = t0 + j / 4 * 16 + (int)quad * 4 + j % 4;
                    sees[rt][j] = (MV)(t >= row_begin[rt] && t < row_end[rt] ? 1.0f : 0.0f);
                }
            each_column([&](const u32x4 &v, int column) {
                constexpr uint32_t ONE = std::is_same_v<MV, half_t> ? 0x3C00u : 0x3F80u;
                u32x4 fine, odd;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t m = ((v[j] & E) == E ? 0xFFFFu : 0u) | ((v[j] >> 16 & E) == E ? 0xFFFF0000u : 0u);
                    fine[j] = v[j] & ~m, odd[j] = m & (ONE | ONE << 16);
                }
                multiply(fine, w, column);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    const f32x4 seen = mfma(__builtin_bit_cast(vec<MV, 8>, odd), sees[rt], f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int i = 0; i < 4; i++) O[rt][column][i] = seen[i] > 0.0f ? NAN : O[rt][column][i];
                }
            });
        } else
            each_column([&](const u32x4 &v, int column) { multiply(v, w, column); });
        if constexpr (MORE) {
            __builtin_amdgcn_sched_barrier(0);
            load_values(next);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (; tile + (int)ATTEND_WAVES < part_end; tile += ATTEND_WAVES) step(std::true_type{});
    if (tile < part_end) step(std::false_type{});

#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        total[rt] = rows_sum(total[rt]);
        if (__any(poison)) total[rt] = NAN;
        if (quad == 0) maxima[wave][rt * 16 + col] = top[rt], sums[wave][rt * 16 + col] = total[rt];
    }
    // Every wave's 16 rows side by side in LDS, then each thread adds four columns of a row.
    float *ob = (float *)lds; // [wave][16][HD + 4]
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int m = 0; m < VD; m += 4)
                *(f32x4 *)(ob + (wave * 16 + col) * (HD + 4) + (quad * 4 + i) * VD + m) =
                    f32x4{O[rt][m][i], O[rt][m + 1][i], O[rt][m + 2][i], O[rt][m + 3][i]};
        __syncthreads();
        for (uint32_t i = tid; i < 16 * (HD / 4); i += ATTEND_THREADS) {
            const uint32_t r = rt * 16 + i / (HD / 4), d = i % (HD / 4) * 4;
            if (r >= count) break;
            const uint2 e = by_group(r0 + r);
            float2 ms = make_float2(maxima[0][r], 0.0f);
#pragma unroll
            for (uint32_t v = 1; v < ATTEND_WAVES; v++) ms.x = fmaxf(ms.x, maxima[v][r]);
            f32x4 x = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t v = 0; v < ATTEND_WAVES; v++) { // a wave without tokens adds zeros (or NaN)
                const float f = maxima[v][r] == -INFINITY ? 1.0f : exp2_fast(maxima[v][r] - ms.x);
                ms.y += sums[v][r] * f;
                x += *(const f32x4 *)(ob + (v * 16 + i / (HD / 4)) * (HD + 4) + d) * f;
            }
            const uint64_t row = first + e.x, qh = head * G + e.y, at = row * a.q_heads + qh;
            bool none = span.end(e.x) <= span.begin(e.x);
            if constexpr (MODE != ATTEND_ALONE)
                if (!none && ms.x == -INFINITY) ms.x = ATTEND_LOWEST;
            if constexpr (MODE == ATTEND_PREFIX) {
                const uint64_t slot = at * a.stride + a.shared + part;
                *(f32x4 *)(a.part_out + slot * HD + d) = x;
                if (d == 0) a.part_sum[slot] = ms;
                continue;
            } else if constexpr (MODE == ATTEND_JOINED) {
                if (a.parts == 1) {
                    const uint64_t slot = at * a.stride + a.shared;
                    constexpr uint32_t AHEAD = 8; // parts loaded at a time
                    for (uint32_t p0 = 0; p0 < shared_parts; p0 += AHEAD) {
                        float2 more[AHEAD];
                        f32x4 y[AHEAD];
#pragma unroll
                        for (uint32_t p = 0; p < AHEAD; p++) {
                            const uint64_t from = slot + min(p0 + p, shared_parts - 1);
                            more[p] = a.part_sum[from], y[p] = *(const f32x4 *)(a.part_out + from * HD + d);
                        }
#pragma unroll
                        for (uint32_t p = 0; p < AHEAD; p++)
                            if (p0 + p < shared_parts) attend_add(ms, x, more[p], y[p]);
                    }
                    attend_write<T>(a, row, qh, d, ms.x == -INFINITY, ms, x, LIFT);
                } else {
                    *(f32x4 *)(a.part_out + (at * a.stride + part) * HD + d) = x;
                    if (d == 0) a.part_sum[at * a.stride + part] = ms;
                    if (d == 0 && part == 0) a.part_count[at] = parts | (shared_parts ? 0 : ATTEND_NONE);
                }
                continue;
            }
            if (parts == 1) attend_write<T>(a, row, qh, d, none, ms, x, LIFT);
            else if (a.joins) {
                shared_store(a.part_out + (at * a.parts + part) * HD + d, float2{x[0], x[1]});
                shared_store(a.part_out + (at * a.parts + part) * HD + d + 2, float2{x[2], x[3]});
                if (d == 0) shared_store((float *)(a.part_sum + at * a.parts + part), ms);
            } else {
                *(f32x4 *)(a.part_out + (at * a.parts + part) * HD + d) = x;
                if (d == 0) a.part_sum[at * a.parts + part] = ms;
                if (d == 0 && part == 0) a.part_count[at] = parts | (none ? ATTEND_NONE : 0);
            }
        }
    }
    if (MODE != ATTEND_ALONE || parts == 1 || !a.joins) return;
    // The last of the block's parts to arrive joins them. Every wave's results are written before the arrival, and both
    // sides go past the caches that XCDs do not share.
    __builtin_amdgcn_s_waitcnt(ATTEND_STORED);
    __syncthreads();
    const auto of = [&](uint32_t r) {
        const uint2 e = by_group(r0 + r);
        return (uint64_t)(first + e.x) * a.q_heads + head * G + e.y;
    };
    if (tid == 0) {
        uint32_t *arrived = a.arrived + of(0);
        last = atomicAdd(arrived, 1u) == parts - 1;
        if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // ready for the next call
    }
    __syncthreads();
    if (!last) return;
    float *factor = (float *)lds; // [ROWS][ATTEND_FEW]
    {
        constexpr uint32_t EACH = ATTEND_FEW / TPR;
        const uint32_t j = tid % TPR;
        const float2 *sum_of = a.part_sum + of(q_row < count ? q_row : 0) * a.parts;
        float2 ms[EACH];
        float most = -INFINITY, sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < EACH; i++) {
            const uint32_t p = j + i * TPR;
            ms[i] = shared_load((const float *)(sum_of + (p < parts ? p : 0)));
            if (p >= parts) ms[i] = make_float2(-INFINITY, 0.0f);
            most = fmaxf(most, ms[i].x);
        }
        most = group_max<TPR>(most);
#pragma unroll
        for (uint32_t i = 0; i < EACH; i++) {
            const float f = ms[i].x == -INFINITY ? 0.0f : exp2_fast(ms[i].x - most);
            factor[q_row * ATTEND_FEW + j + i * TPR] = f;
            sum += ms[i].x == -INFINITY ? ms[i].y : ms[i].y * f; // a part without tokens has 0, or NaN
        }
        sum = group_sum<TPR>(sum);
        if (j == 0) maxima[0][q_row] = most, sums[0][q_row] = sum;
    }
    __syncthreads();
    for (uint32_t i = tid; i < count * (HD / 4); i += ATTEND_THREADS) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
        const uint2 e = by_group(r0 + r);
        const float *x = a.part_out + of(r) * a.parts * HD + d;
        f32x4 all = {0, 0, 0, 0};
        for (uint32_t p0 = 0; p0 < parts; p0 += 8) {
            float2 y[8][2];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const float *z = x + (p0 + j < parts ? p0 + j : p0) * HD;
                y[j][0] = shared_load(z), y[j][1] = shared_load(z + 2);
            }
#pragma unroll
            for (uint32_t j = 0; j < 8; j++)
                if (p0 + j < parts) all += f32x4{y[j][0].x, y[j][0].y, y[j][1].x, y[j][1].y} * factor[r * ATTEND_FEW + p0 + j];
        }
        attend_write<T>(a, first + e.x, head * G + e.y, d, span.end(e.x) <= span.begin(e.x),
                        make_float2(maxima[0][r], sums[0][r]), all, LIFT);
    }
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

}  // namespace rl
