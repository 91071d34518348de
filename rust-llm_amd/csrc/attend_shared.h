// Attention over a prefix that many rows share (include/rl_mixers.h).
//
// k_attend gives each wave other tokens of the same rows, which suits few rows. Here
// the waves of a workgroup have rows of their own, 16 RT each, and the same tokens: a
// tile of keys and values is loaded once for all, converted to the 16 bits of the
// products, turned, and laid into LDS as the fragments that the products take, so a
// wave's own work is its products and its softmax:
//   S^T = K Q^T, w = 2^(S - m), O^T += V^T w   as in attend.h, 32 tokens at a time
// A workgroup has two halves of four waves, with the same rows and every other tile.
// Waves 0 and 1 of a half bring the keys, 2 and 3 the values: in registers while the
// tile before is computed, into the other of two buffers behind it. The halves are half
// a tile apart, so that one's products pass beside the other's softmax (5 % faster than
// in step). Their sums are added at the end. Every row sees the whole prefix, so only
// the last tile has a mask.
//
// Bound in the tiles by instructions, which two waves on a SIMD pass with some overlap
// only (8 products and 32 sums take 257 cycles, alone 164 and 190): a tile of 64 tokens
// and 32 rows of 128 bf16 is 96 products of 16 cycles and 480 vector instructions a
// wave. Beside the tiles by the start and the end of a workgroup, the one a CU holds:
// the chain of pages, queries and the first tile, and the sums by way of LDS.
// 256 rows a key-value head, 8 heads of 128, 16384 tokens bf16: 48 us, 358 TFLOP/s
// (k_attend 106 us). Its 256 workgroups have 16 tiles of 1.41 us each (in 8, 4, 2 and 1
// parts 69, 114, 204 and 385 us), which leaves 25 for start and end. Over the whole, waves
// issue 35 % of their time, 20 % they wait for a unit and 46 % for loads, LDS and each
// other; matrix units are busy 28 %, vector units 42 %. 640 rows, 8001 tokens int8 in
// pages of 24, and two prefixes of a half and a third: 115 us, 335 TFLOP/s, two rounds of
// workgroups of 21 tiles, 1.6 us each, and 25 for start and end. f32 queries, in two or
// three parts: the first call 78 us, over f16 62, the second 203.
#pragma once
#include "attend.h"

namespace rl {

// Tiles of 16 rows that a wave may have: two share each fragment that is read; f32 queries and heads of 256 take the
// registers for one.
template <typename T>
constexpr int shared_row_tiles(int hd) {
    return sizeof(T) == 4 || hd == 256 ? 1 : 2;
}

// Tokens of a tile: as many as give each thread eight 16-byte units to bring.
constexpr int shared_tile(int hd) { return 8192 / hd; }

constexpr uint32_t SHARED_THREADS = 512;
template <int I>
using Int = std::integral_constant<int, I>;
// Powers of two by which a weight may pass 1. Those of f16 products are 2^8 times their size already, and stay below 2^13.
constexpr float SHARED_SLACK = 4.0f;

template <typename T, int FMT, int HD, int RT, bool P16>
__global__ void __launch_bounds__(SHARED_THREADS, 2) k_attend_shared(AttendArgs a) {
    constexpr bool EIGHT = FMT == RL_I8 || FMT == RL_F8, F32Q = sizeof(T) == 4;
    using MK = std::conditional_t<FMT == RL_BF16, bhalf_t, half_t>;
    using MV = std::conditional_t<FMT == RL_F16, half_t, bhalf_t>;
    // Parts of queries and weights, as in k_attend.
    constexpr int QP = !F32Q ? 1 : std::is_same_v<MK, bhalf_t> ? 3 : 2, PP = F32Q && std::is_same_v<MV, bhalf_t> ? 3 : 2;
    constexpr float LIFT = FMT == RL_F16 ? ATTEND_LIFT : 0.0f;
    constexpr int TILE = shared_tile(HD), KS = TILE / 32, UT = TILE / 16, STEPS = HD / 32, VD = HD / 16, ROWS = 64 * RT;
    constexpr int UNITS = HD / 8; // of eight dims, 16 bytes as 16-bit values
    static_assert(TILE * UNITS == 8 * 128, "eight units a thread");
    constexpr int SIZE = EIGHT ? 1 : 2;
    using Raw = std::conditional_t<EIGHT, uint2, u32x4>;
    // Of each half of the workgroup, two buffers. At the end the sums take the fragments' place.
    constexpr int FRAGMENTS = TILE * UNITS, OS = HD + 4;
    constexpr size_t FRAGMENT_BYTES = (size_t)2 * 2 * 2 * FRAGMENTS * 16, SUM_BYTES = (size_t)2 * ROWS * OS * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[FRAGMENT_BYTES > SUM_BYTES ? FRAGMENT_BYTES : SUM_BYTES];
    __shared__ uint64_t places[2][2][P16 ? 1 : TILE]; // vectors of a tile's tokens
    __shared__ __attribute__((aligned(16))) float key_steps[2][2][EIGHT ? TILE : 4], value_steps[2][2][EIGHT ? TILE : 4];
    __shared__ __attribute__((aligned(16))) float masks[2][2][TILE]; // 0, or -inf past the prefix: the scores' first value
    __shared__ float2 half_sums[2][ROWS];
    __shared__ uint32_t bad;

    const uint32_t half = __builtin_amdgcn_readfirstlane(threadIdx.x / 256), tid = threadIdx.x % 256, lane = tid % 64;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
    u32x4(*kbuf)[FRAGMENTS] = (u32x4(*)[FRAGMENTS])lds + 4 * half, (*vbuf)[FRAGMENTS] = kbuf + 2;
    auto &where = places[half];
    auto &ksteps = key_steps[half];
    auto &vsteps = value_steps[half];
    auto &mask = masks[half];
    const uint32_t G = a.group, col = lane % 16, quad = lane / 16;
    // The row blocks of one head and part are eight workgroups apart: on one XCD, whose L2 has the tokens for all but the
    // first.
    const uint2 eight = split_by(blockIdx.x / 8, a.blocks, a.blocks_inv);
    const uint2 job = split_by(eight.x * 8 + blockIdx.x % 8, a.cache.heads, a.heads_inv);
    const uint32_t part = job.x, head = job.y;
    if (part >= a.parts) return;
    // Which of them are without rows may follow a pattern, and workgroups go to shader engines in turn: each eight begins with
    // another (3 groups of 32 rows, every other block empty: a call of 78.9 us in one order for all, 51.2 so).
    const uint32_t block = split_by(eight.x + eight.y, a.blocks, a.blocks_inv).y;
    typedef const __attribute__((address_space(4))) int32_t constant_i32;
    const constant_i32 *starts = (constant_i32 *)(uintptr_t)a.starts, *group_starts = (constant_i32 *)(uintptr_t)a.group_starts;
    const auto first_of = [&](uint32_t g) {
        const int32_t at = min(max(group_starts[g], 0), (int32_t)a.group_end);
        return starts ? min(max(starts[at], 0), (int32_t)a.rows) : min(at, (int32_t)a.rows);
    };
    const auto first_block = [&](uint32_t g) { return (uint32_t)first_of(g) * G / ROWS + g; };
    uint32_t g = 0;
    for (uint32_t hi = a.seqs; hi - g > 1;) {
        const uint32_t mid = g + (hi - g) / 2;
        if (first_block(mid) <= block) g = mid;
        else hi = mid;
    }
    if (first_block(g) > block) return;
    const int32_t first = first_of(g), rows = first_of(g + 1) - first;
    const uint32_t r0 = (block - first_block(g)) * ROWS;
    if (rows <= 0 || r0 >= (uint32_t)rows * G) return;
    const uint32_t count = min((uint32_t)rows * G - r0, (uint32_t)ROWS);
    const int32_t len = max(((constant_i32 *)(uintptr_t)a.lens)[g], 0);
    const uint32_t page = a.cache.page, tiles = ((uint32_t)len + TILE - 1) / TILE;
    const bool nan = len > (int64_t)a.max_len || (len > 0 && split_by(len - 1, page, a.cache.page_inv).x >= a.table_width);
    const uint32_t begin = part * a.part_tiles, end = min(begin + a.part_tiles, tiles);
    const auto slot_of = [&](uint32_t r) { // of a row's partial result
        const uint2 e = split_by(r0 + r, G, a.group_inv);
        return ((uint64_t)(first + e.x) * a.q_heads + head * G + e.y) * a.stride + a.shared + part;
    };
    if (nan || begin >= end) { // no tokens; what the call's bounds or the table do not cover is one part that is NaN
        if (threadIdx.x < count) a.part_sum[slot_of(threadIdx.x)] = nan && part == 0 ? make_float2(0.0f, NAN) : make_float2(-INFINITY, 0.0f);
        return;
    }
    if (threadIdx.x == 0) bad = 0;

    // Where tokens lie. P16 (pages of a multiple of 16 tokens): a tile's blocks of 16 each lie in one page, whose numbers are
    // fetched through the scalar cache a tile ahead of the loads. Else a thread looks the page of one token up, two tiles
    // ahead, and leaves its vector in LDS.
    const int32_t *table = a.pages + (uint64_t)g * a.table_width;
    const uint32_t pool = (uint32_t)(a.cache.slots / page), dim_bytes = a.cache.dim * SIZE;
    const auto split_at = [&](uint32_t t) { return split_by(t, page, a.cache.page_inv); };
    bool poison = false; // a page number that is none
    const auto place_of = [&](uint32_t tile) { return split_at(min(tile * TILE + tid % TILE, (uint32_t)len - 1)); };
    const auto put_place = [&](uint32_t tile, uint32_t id, uint32_t in_page) {
        if (P16 || tid >= TILE) return;
        if (id >= pool) poison = true, id = 0;
        where[tile / 2 & 1][tid] = ((uint64_t)id * a.cache.heads + head) * page + in_page;
    };
    // A thread's share of a tile: keys unit by unit, or eight tokens of one unit of values.
    const bool keys = wave < 2;
    const uint32_t sub = tid % 128;
    const uint32_t group = sub / UNITS; // of eight tokens of values, in the order of a lane's scores
    const uint32_t token0 = keys ? group : group / 4 * 32 + group % 4 * 4;
    const auto token_of = [&](int j) { return token0 + (uint32_t)(keys ? j * (128 / UNITS) : j / 4 * 16 + j % 4); };
    const uint32_t unit = sub % UNITS; // 128 is a multiple of UNITS
    const bool in_dim = unit * 8 < a.cache.dim;
    const uint32_t in_vector = in_dim ? unit * 8 * SIZE : 0;
    const uint8_t *source = (const uint8_t *)(keys ? a.cache.keys : a.cache.values);
    Raw raw[8];
    float key_step = 0.0f, value_step = 0.0f; // of token sub % TILE, brought by the waves of the keys
    // P16: the blocks that a wave's units are of, in order (with values of 64 dims, four that its lanes choose of), the numbers
    // of their pages and where in the cache their first vectors are.
    constexpr int OWN = HD == 256 ? 2 : HD == 128 ? 4 : 8;
    const bool upper = wave & 1, late = lane >= 32;
    const auto block_at = [&](uint32_t tile, int i) {
        const int block = HD == 256 || keys ? i : HD == 128 ? 2 * upper + i / 2 : 4 * upper + i % 4;
        return split_at(min(tile * TILE + 16 * block, ((uint32_t)len - 1) & ~15u));
    };
    uint32_t ids[P16 ? OWN : 1];
    uint64_t v0 = 0, v1 = 0, v2 = 0, v3 = 0, v4 = 0, v5 = 0, v6 = 0, v7 = 0; // not an array: it would go to memory
    const auto fetch = [&](uint32_t tile) {
        if constexpr (P16)
#pragma unroll
            for (int i = 0; i < OWN; i++) ids[i] = (uint32_t)((constant_i32 *)(uintptr_t)table)[block_at(tile, i).x];
    };
    const auto locate = [&](uint32_t tile) {
        if constexpr (P16) {
            const auto one = [&](int i) {
                poison |= ids[i] >= pool;
                return ((uint64_t)(ids[i] < pool ? ids[i] : 0) * a.cache.heads + head) * page + block_at(tile, i).y;
            };
            v0 = one(0), v1 = one(1);
            if constexpr (OWN > 2) v2 = one(2), v3 = one(3);
            if constexpr (OWN > 4) v4 = one(4), v5 = one(5), v6 = one(6), v7 = one(7);
        }
    };
    const auto own = [&](auto i) { // the wave's i-th
        constexpr int I = decltype(i)::value;
        if constexpr (I == 0) return v0;
        else if constexpr (I == 1) return v1;
        else if constexpr (I == 2) return v2;
        else if constexpr (I == 3) return v3;
        else if constexpr (I == 4) return v4;
        else if constexpr (I == 5) return v5;
        else if constexpr (I == 6) return v6;
        else return v7;
    };
    // The thread's j-th unit of a tile that has been located (P16).
    const auto load_unit = [&](uint32_t tile, auto unit_j) {
        constexpr int J = decltype(unit_j)::value;
        const uint32_t in_block = token_of(J) % 16 * dim_bytes + in_vector;
        if constexpr (!P16) raw[J] = *(const Raw *)(source + where[tile / 2 & 1][token_of(J)] * dim_bytes + in_vector);
        else if constexpr (HD >= 128) raw[J] = *(const Raw *)(source + own(Int<J * OWN / 8>{}) * dim_bytes + in_block);
        else {
            const uint64_t early = own(Int<J / 4>{}), behind = own(Int<2 + J / 4>{}), key = own(Int<J>{});
            raw[J] = *(const Raw *)(source + (keys ? key : late ? behind : early) * dim_bytes + in_block);
        }
    };
    const auto load_steps = [&](uint32_t tile) {
        if (!EIGHT || !keys) return;
        uint64_t at;
        if constexpr (!P16) at = where[tile / 2 & 1][sub % TILE];
        else {
            const uint64_t b0 = OWN == 8 && upper ? v4 : v0, b1 = OWN == 8 && upper ? v5 : v1, b2 = OWN == 8 && upper ? v6 : v2,
                           b3 = OWN == 8 && upper ? v7 : v3;
            at = (OWN > 2 && late ? (lane & 16 ? b3 : b2) : lane & 16 ? b1 : b0) + lane % 16;
        }
        key_step = a.cache.key_steps[at], value_step = a.cache.value_steps[at];
    };
    const auto load = [&](uint32_t tile) {
        load_unit(tile, Int<0>{}), load_unit(tile, Int<1>{}), load_unit(tile, Int<2>{}), load_unit(tile, Int<3>{});
        load_unit(tile, Int<4>{}), load_unit(tile, Int<5>{}), load_unit(tile, Int<6>{}), load_unit(tile, Int<7>{});
        load_steps(tile);
    };
    // Tokens past the prefix and dims past the head are zeros.
    const auto put = [&](uint32_t tile) {
        const uint32_t b = tile / 2 & 1, left = (uint32_t)len - tile * TILE;
        if (left < TILE || a.cache.dim != HD)
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (!in_dim || token_of(j) >= left) raw[j] = Raw{};
        if (keys) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t t = token_of(j), c = t % 16;
                u32x4 x;
                if constexpr (EIGHT) {
                    const u32x4 w = {pair_f16<FMT, false>(raw[j].x), pair_f16<FMT, true>(raw[j].x), pair_f16<FMT, false>(raw[j].y),
                                     pair_f16<FMT, true>(raw[j].y)};
                    vec<half_t, 8> k = __builtin_bit_cast(decltype(k), w);
                    if constexpr (FMT == RL_I8) k -= (half_t)KEY_BIAS;
                    if (left < TILE || a.cache.dim != HD)
                        if (!in_dim || t >= left) k = vec<half_t, 8>{};
                    x = __builtin_bit_cast(u32x4, k);
                } else x = raw[j];
                // Unit 4 st + q of token 16 u + c is lane 16 q + c's of fragment (u, st), turned by the unit among 16 lanes:
                // units of one token would else all be in the same banks.
                kbuf[b][(t / 16 * STEPS + unit / 4) * 64 + unit % 4 * 16 + (c + unit) % 16] = x;
            }
        } else {
            u32x4 out[8];
            if constexpr (!EIGHT) {
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        out[2 * c][j] = __builtin_amdgcn_perm(raw[2 * j + 1][c], raw[2 * j][c], 0x05040100u);
                        out[2 * c + 1][j] = __builtin_amdgcn_perm(raw[2 * j + 1][c], raw[2 * j][c], 0x07060302u);
                    }
            } else {
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t y = c ? raw[2 * j + 1].y : raw[2 * j + 1].x, x = c ? raw[2 * j].y : raw[2 * j].x;
                        const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05010400u), hi = __builtin_amdgcn_perm(y, x, 0x07030602u);
                        out[4 * c][j] = pair_bf16<FMT, false>(lo);
                        out[4 * c + 1][j] = pair_bf16<FMT, true>(lo);
                        out[4 * c + 2][j] = pair_bf16<FMT, false>(hi);
                        out[4 * c + 3][j] = pair_bf16<FMT, true>(hi);
                    }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) { // dim d is column d % VD of lane row d / VD
                const uint32_t d = unit * 8 + e;
                vbuf[b][(group / 4 * VD + d % VD) * 64 + group % 4 * 16 + d / VD] = out[e];
            }
        }
        if constexpr (EIGHT)
            if (keys && sub < TILE) ksteps[b][sub] = sub < left ? key_step : 1.0f, vsteps[b][sub] = sub < left ? value_step : 0.0f;
        if (tid < TILE) mask[b][tid] = tid < left ? 0.0f : -INFINITY;
    };

    // The halves take tiles in turn. The first tiles' pages, then the queries, then the first tile: each is on its way
    // while the one before is used.
    const uint32_t mine = begin + half;
    uint2 at0{}, at1{};
    uint32_t id0 = 0, id1 = 0;
    if constexpr (P16) fetch(mine);
    else {
        at0 = place_of(mine), at1 = place_of(mine + 2); // of tokens past the prefix: its last
        id0 = (uint32_t)table[at0.x], id1 = (uint32_t)table[at1.x];
    }
    // The wave's queries as the second operand: lane (row col, quad) has dims 32 st + 8 quad .. + 8.
    const uint32_t w0 = wave * 16 * RT;
    const bool idle = w0 >= count;
    float x[RT][STEPS][8] = {};
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t r = w0 + rt * 16 + col;
        if (r < count) {
            const uint2 e = split_by(r0 + r, G, a.group_inv);
            const T *p = (const T *)a.q + (uint64_t)(first + e.x) * a.q_row + (uint64_t)(head * G + e.y) * a.q_head;
#pragma unroll
            for (int st = 0; st < STEPS; st++)
                if (st * 32 + quad * 8 < a.cache.dim) load_f32(p + st * 32 + quad * 8, a.wide, x[rt][st]); // dim is a multiple of 16
        }
    }
    __syncthreads(); // for `bad`
    put_place(mine, id0, at0.y);
    put_place(mine + 2, id1, at1.y);
    __syncthreads();
    locate(mine); // a tile past the part's end is one of the prefix's
    load(mine);
    fetch(mine + 2);
    vec<MK, 8> q[RT][QP][STEPS];
    float mult[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        float unit_of = 1.0f;
        if constexpr (std::is_same_v<MK, half_t>) { // as in k_attend
            float m = 0.0f;
#pragma unroll
            for (int st = 0; st < STEPS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(x[rt][st][j]));
            m = rows_max(m);
            const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 100);
            const float down = __uint_as_float((uint32_t)(127 - e) << 23);
            unit_of = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int st = 0; st < STEPS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[rt][st][j] *= down;
        }
        // The scale's sign goes to the queries: scores are then compared before they are scaled. So does NaN.
        const float sign = a.scale < 0.0f ? -1.0f : a.scale >= 0.0f ? 1.0f : a.scale;
#pragma unroll
        for (int p = 0; p < QP; p++)
#pragma unroll
            for (int st = 0; st < STEPS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    q[rt][p][st][j] = (MK)(x[rt][st][j] * sign);
                    x[rt][st][j] -= (float)q[rt][p][st][j] * sign;
                }
        // Not zero, which would make NaN of a masked score: times 2^-149 every other is below 2^-21.
        mult[rt] = fmaxf(fabsf(a.scale) * 1.44269504088896341f * unit_of, 0x1p-149f);
    }
    f32x4 O[RT][VD];
    float top[RT], total[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        top[rt] = -INFINITY, total[rt] = 0.0f;
#pragma unroll
        for (int m = 0; m < VD; m++) O[rt][m] = f32x4{0, 0, 0, 0};
    }

    // A tile's work in steps of 32 tokens: the scores of step k + 1, the weights of step k and the products with the values of
    // step k - 1 are independent of each other, so that matrix and vector instructions can pass side by side.
    f32x4 S[KS][RT][2];
    vec<MV, 8> w[KS][RT][PP];
    const auto scores = [&](uint32_t b, int ks) {
        constexpr int DEEP = 2; // steps of the contraction whose fragments are read at a time
        vec<MK, 8> kf[2][DEEP][2];
        const auto read = [&](int st0) {
#pragma unroll
            for (int i = 0; i < DEEP; i++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int st = st0 + i;
                    kf[st0 / DEEP & 1][i][u] = __builtin_bit_cast(
                        vec<MK, 8>, kbuf[b][((ks * 2 + u) * STEPS + st) * 64 + quad * 16 + (col + 4 * st + quad) % 16]);
                }
        };
#pragma unroll
        for (int u = 0; u < 2; u++) {
            S[ks][0][u] = *(const f32x4 *)&mask[b][ks * 32 + u * 16 + quad * 4];
#pragma unroll
            for (int rt = 1; rt < RT; rt++) S[ks][rt][u] = S[ks][0][u];
        }
        read(0);
#pragma unroll
        for (int st0 = 0; st0 < STEPS; st0 += DEEP) {
            if (st0 + DEEP < STEPS) read(st0 + DEEP);
#pragma unroll
            for (int i = 0; i < DEEP; i++)
#pragma unroll
                for (int p = 0; p < QP; p++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
                            S[ks][rt][u] = mfma(kf[st0 / DEEP & 1][i][u], q[rt][p][st0 + i], S[ks][rt][u]);
        }
    };
    typedef vec<bhalf_t, 2> bf16x2;
    uint32_t less_low = 0x0000BF80u, less_high = 0xBF800000u; // pairs of bf16
    // The second is what the f32 -1 is, and as an immediate it would not be read as a pair.
    asm("" : "+v"(less_low), "+v"(less_high));
    const auto weights = [&](uint32_t b, int ks) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float base = (top[rt] == -INFINITY ? 0.0f : top[rt]) - LIFT;
            float rest[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float p = exp2_fast(fmaf(S[ks][rt][j / 4][j % 4], mult[rt], -base));
                total[rt] += p;
                if constexpr (EIGHT) p *= vsteps[b][ks * 32 + j / 4 * 16 + quad * 4 + j % 4];
                rest[j] = p;
            }
            if constexpr (std::is_same_v<MV, bhalf_t>) { // the first part cut off, as in k_attend
                u32x4 cut;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const uint32_t both = __builtin_amdgcn_perm(__float_as_uint(rest[j + 1]), __float_as_uint(rest[j]), 0x07060302u);
                    // Less the first part, taken from the pair by a product with (-1, 0) or (0, -1): exact.
                    const bf16x2 pair = __builtin_bit_cast(bf16x2, both);
                    cut[j / 2] = both;
                    rest[j] = __builtin_amdgcn_fdot2_f32_bf16(pair, __builtin_bit_cast(bf16x2, less_low), rest[j], false);
                    rest[j + 1] = __builtin_amdgcn_fdot2_f32_bf16(pair, __builtin_bit_cast(bf16x2, less_high), rest[j + 1], false);
                }
                w[ks][rt][0] = __builtin_bit_cast(vec<MV, 8>, cut);
            } else
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    w[ks][rt][0][j] = (MV)rest[j];
                    rest[j] -= (float)w[ks][rt][0][j];
                }
#pragma unroll
            for (int i = 1; i < PP; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    w[ks][rt][i][j] = (MV)rest[j];
                    rest[j] -= (float)w[ks][rt][i][j];
                }
        }
    };
    const auto products = [&](uint32_t b, int ks) {
        constexpr int DEEP = 2;
        vec<MV, 8> vf[2][DEEP];
        const auto read = [&](int m0) {
#pragma unroll
            for (int i = 0; i < DEEP; i++) vf[m0 / DEEP & 1][i] = __builtin_bit_cast(vec<MV, 8>, vbuf[b][(ks * VD + m0 + i) * 64 + lane]);
        };
        read(0);
#pragma unroll
        for (int m0 = 0; m0 < VD; m0 += DEEP) {
            if (m0 + DEEP < VD) read(m0 + DEEP);
#pragma unroll
            for (int p = 0; p < PP; p++)
#pragma unroll
                for (int m = 0; m < DEEP; m++)
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) O[rt][m0 + m] = mfma(vf[m0 / DEEP & 1][m], w[ks][rt][p], O[rt][m0 + m]);
        }
    };
    // A row's base is no more than SHARED_SLACK below the largest of its scores: it follows only when it has to, for all rows
    // of the wave at once. Weights that are still to be multiplied have the base that they were formed with, so their products
    // come first, and zeros in their place.
    const auto rebase = [&](uint32_t b, int ks) {
        float most[RT];
        bool up = false;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            most[rt] = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if constexpr (EIGHT) S[ks][rt][u] *= *(const f32x4 *)&ksteps[b][ks * 32 + u * 16 + quad * 4];
#pragma unroll
                for (int i = 0; i < 4; i++) most[rt] = fmaxf(most[rt], S[ks][rt][u][i]);
            }
            most[rt] = rows_max(most[rt]) * mult[rt];
            up |= most[rt] > top[rt] + SHARED_SLACK;
        }
        if (!__any(up)) return;
        if (ks > 0) {
            products(b, ks - 1);
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int p = 0; p < PP; p++) w[ks - 1][rt][p] = vec<MV, 8>{};
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float now = fmaxf(most[rt], top[rt]), keep = now == -INFINITY ? 1.0f : exp2_fast(top[rt] - now);
            total[rt] *= keep;
#pragma unroll
            for (int m = 0; m < VD; m++) O[rt][m] *= keep;
            top[rt] = now;
        }
    };
    const auto advance = [&](uint32_t b, int k) {
        if (k + 1 < KS) scores(b, k + 1);
        if (k < KS) weights(b, k);
        if (k > 0) products(b, k - 1);
        if (k + 1 < KS) rebase(b, k + 1);
    };

    if (mine < end) put(mine);
    __syncthreads();
    // Both parts of a tile end at a barrier, which every wave comes to equally often: the second half once before its first
    // tile, and whoever is done with its tiles for the rest.
    uint32_t barriers = 2 * ((end - begin + 1) / 2) + 1;
    const auto meet = [&] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        barriers--;
    };
    if (half) meet();
    for (uint32_t tile = mine; tile < end; tile += 2) {
        const bool more = tile + 2 < end, further = tile + 4 < end;
        uint32_t id = 0, in_page = 0;
        if (more) {
            locate(tile + 2);
            load(tile + 2);
        }
        fetch(tile + 4);
        if (!P16 && further) {
            const uint2 place = place_of(tile + 4);
            id = (uint32_t)table[place.x], in_page = place.y;
        }
        const uint32_t b = tile / 2 & 1;
        if (!idle) {
            scores(b, 0);
            rebase(b, 0);
            advance(b, 0);
            if constexpr (KS == 4) advance(b, 1);
        }
        meet();
        if (!idle) {
            if constexpr (KS != 4) advance(b, 1);
            if constexpr (KS == 2) advance(b, 2);
            if constexpr (KS == 4) advance(b, 2), advance(b, 3), advance(b, 4);
        }
        if (more) put(tile + 2);
        if (further) put_place(tile + 4, id, in_page);
        meet();
    }
    while (barriers) meet();
    // Both halves' sums side by side in LDS, then each thread adds four columns of a row, lines at a time.
    float *sums = (float *)lds; // [half][row][OS]
    if (poison) bad = 1;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        total[rt] = rows_sum(total[rt]);
        const uint32_t r = w0 + rt * 16 + col;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int m = 0; m < VD; m += 4)
                *(f32x4 *)(sums + (half * ROWS + r) * OS + (quad * 4 + i) * VD + m) =
                    f32x4{O[rt][m][i], O[rt][m + 1][i], O[rt][m + 2][i], O[rt][m + 3][i]};
        if (quad == 0) half_sums[half][r] = make_float2(top[rt], total[rt]);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count * (HD / 4); i += SHARED_THREADS) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
        const float2 x = half_sums[0][r], y = half_sums[1][r]; // a half without tokens has sums of 0
        const float most = fmaxf(x.x, y.x);
        const float f = x.x == -INFINITY ? 1.0f : exp2_fast(x.x - most), g2 = y.x == -INFINITY ? 1.0f : exp2_fast(y.x - most);
        const uint64_t slot = slot_of(r);
        *(f32x4 *)(a.part_out + slot * HD + d) = *(const f32x4 *)(sums + r * OS + d) * f + *(const f32x4 *)(sums + (ROWS + r) * OS + d) * g2;
        if (d == 0) a.part_sum[slot] = make_float2(most == -INFINITY ? ATTEND_LOWEST : most, bad ? NAN : x.y * f + y.y * g2);
    }
}

// Launches the kernel for queries of type T (shared_*.hip, one unit a type).
template <typename T>
void launch_attend_shared(const AttendArgs &a, uint32_t format, bool two, uint32_t groups, hipStream_t s);

#ifdef RL_SHARED_UNIT
template <typename T, int FMT, int HD>
void launch_attend_shared_rows(const AttendArgs &a, bool two, uint32_t groups, hipStream_t s) {
    if constexpr (shared_row_tiles<T>(HD) == 2)
        if (two) {
            auto kern = a.cache.page % 16 ? k_attend_shared<T, FMT, HD, 2, false> : k_attend_shared<T, FMT, HD, 2, true>;
            hipLaunchKernelGGL(kern, dim3(groups), dim3(SHARED_THREADS), 0, s, a);
            return;
        }
    auto kern = a.cache.page % 16 ? k_attend_shared<T, FMT, HD, 1, false> : k_attend_shared<T, FMT, HD, 1, true>;
    hipLaunchKernelGGL(kern, dim3(groups), dim3(SHARED_THREADS), 0, s, a);
}

template <typename T, int FMT>
void launch_attend_shared_format(const AttendArgs &a, bool two, uint32_t groups, hipStream_t s) {
    switch (attend_dim(a.cache.dim)) {
    case 64: return launch_attend_shared_rows<T, FMT, 64>(a, two, groups, s);
    case 128: return launch_attend_shared_rows<T, FMT, 128>(a, two, groups, s);
    default: return launch_attend_shared_rows<T, FMT, 256>(a, two, groups, s);
    }
}

template <typename T>
void launch_attend_shared(const AttendArgs &a, uint32_t format, bool two, uint32_t groups, hipStream_t s) {
    if constexpr (!std::is_same_v<T, bhalf_t>)
        if (format == RL_F16) return launch_attend_shared_format<T, RL_F16>(a, two, groups, s);
    if constexpr (!std::is_same_v<T, half_t>)
        if (format == RL_BF16) return launch_attend_shared_format<T, RL_BF16>(a, two, groups, s);
    if (format == RL_I8) return launch_attend_shared_format<T, RL_I8>(a, two, groups, s);
    launch_attend_shared_format<T, RL_F8>(a, two, groups, s);
}
#endif

}  // namespace rl
