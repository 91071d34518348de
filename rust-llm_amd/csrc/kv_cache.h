// The paged key-value cache (include/rl_mixers.h): its layout, and the kernels
// that write rows into it (turned and quantised) and read them back.
#pragma once
#include "rotary.h"

namespace rl {

// Codes are [page][head][token of the page][dim], steps (8-bit formats) f32
// [page][head][token]: the tokens of one page and head lie together, as the
// attention reads them. int8 codes of keys have their sign bit flipped, which
// saves the attention an instruction a dword.
constexpr uint32_t KEY_SIGNS = 0x80808080u;
struct CacheArgs {
    void *keys, *values;
    float *key_steps, *value_steps;
    uint64_t slots; // at most 2^32
    uint32_t page, heads, dim;
    uint32_t page_inv, vectors_inv; // inverse_of the page and of the vectors of a row, 2 heads
};

// The vector of a slot and head, counted in vectors of dim values.
__device__ inline uint64_t cache_vector(const CacheArgs &c, uint32_t slot, uint32_t head) {
    const uint2 p = split_by(slot, c.page, c.page_inv);
    return ((uint64_t)p.x * c.heads + head) * c.page + p.y;
}

struct CacheRows {
    const void *keys, *values; // outputs of a read
    uint64_t key_row, key_head, value_row, value_head;
    uint32_t rows;
    uint32_t wide; // whether 16-byte accesses to them are aligned
};

constexpr uint32_t CACHE_THREADS = 256;
constexpr uint32_t CACHE_MAX_ROWS = 16; // rows a workgroup, LDS holds their angles
// Vectors that a group of lanes has on their way: 20000 rows of 4 heads of 256 take 31.0 us with 1, 29.1 with 2, 29.2
// with 3, 29.6 with 4; 5003 rows 10.5, 11.1, 11.6, 12.1.
constexpr int CACHE_AHEAD = 2;

// Turns the eight values x of a head's key, at on, if they are among the turned ones. raw: as they were read. Their
// partners in the half layout of a multiple of 8 pairs are another lane's eight, elsewhere read again.
template <typename T, int G>
__device__ inline void turn8(const RotaryArgs &r, const T *in, uint32_t at, const float2 *cs, const vec<T, 8> &raw, float (&x)[8]) {
    const uint32_t turned = 2 * r.pairs;
    if (at >= turned) return;
    if (!r.interleaved && r.pairs % 8 == 0) {
        const bool second = at >= r.pairs;
        const uint32_t i = second ? at - r.pairs : at;
        const vec<uint32_t, 2 * sizeof(T)> mine = __builtin_bit_cast(vec<uint32_t, 2 * sizeof(T)>, raw);
        vec<uint32_t, 2 * sizeof(T)> theirs;
#pragma unroll
        for (int j = 0; j < 2 * (int)sizeof(T); j++) theirs[j] = __shfl(mine[j], i / 8 + (second ? 0 : r.pairs / 8), G);
        const vec<T, 8> y = __builtin_bit_cast(vec<T, 8>, theirs);
#pragma unroll
        for (int j = 0; j < 8; j++) { // turn_a or turn_b
            const float2 w = cs[i + j];
            x[j] = x[j] * w.x + (float)y[j] * (second ? w.y : -w.y);
        }
    } else if (r.interleaved && at + 8 <= turned) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2 w = cs[(at + j) / 2];
            const float p = x[j], q = x[j + 1];
            x[j] = turn_a(p, q, w);
            x[j + 1] = turn_b(p, q, w);
        }
    } else {
        // One value after the other: unrolled, this takes twice the registers of everything else.
#pragma unroll 1
        for (uint32_t j = 0; j < 8 && at + j < turned; j++) {
            const uint32_t e = at + j;
            const bool second = r.interleaved ? e & 1 : e >= r.pairs;
            const uint32_t i = r.interleaved ? e / 2 : second ? e - r.pairs : e;
            const uint32_t other = r.interleaved ? e ^ 1 : second ? i : e + r.pairs;
            const float2 w = cs[i];
            const float z = (float)in[e] * w.x + (float)in[other] * (second ? w.y : -w.y);
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) x[k] = k == j ? z : x[k];
        }
    }
}

// G lanes hold a vector of up to 8 G values, eight a lane. Vectors of a workgroup's
// rows: keys of every head, then values of every head. One pass: the largest
// magnitude is reduced over the lanes while the values stay in registers. The
// first CACHE_AHEAD vectors of a group are loaded before the angles are formed and
// waited for. A workgroup is one chain (position, angles, barrier, codes), so what
// counts is how many share a CU: with partners and the rare layouts at 110
// registers four did, 5003 rows of 4 heads of 256 bf16 to f8 (31 MB) took 16.7 us;
// with 55 eight do, 11.8 us (2.6 TB/s). 64 int8 rows of 8 heads of 128: 3.4 us,
// all chain.
template <typename T, int FMT, int G>
__global__ void __launch_bounds__(CACHE_THREADS) k_cache_write(CacheArgs c, CacheRows in, const int64_t *slots,
                                                               uint32_t rows_a_group, RotaryArgs r,
                                                               const int64_t *positions) {
    __shared__ float2 cs[CACHE_MAX_ROWS * ROTARY_MAX_PAIRS / 2];
    constexpr uint32_t GROUPS = CACHE_THREADS / G;
    const uint32_t row0 = blockIdx.x * rows_a_group, n = min(rows_a_group, in.rows - row0);
    const uint32_t lane = threadIdx.x % G, at = lane * 8, all = n * 2 * c.heads;
    const bool here = at < c.dim, wide = in.wide;
    const uint32_t from = here ? at : 0; // lanes past the head's end load its start
    struct Item {
        const T *p;
        bool is_value;
        uint32_t rr, head;
        int64_t slot;
        vec<T, 8> x;
    };
    auto load = [&](uint32_t i, Item &t) { // past the end the last vector again
        i = min(i, all - 1);
        const uint2 row_vector = split_by(i, 2 * c.heads, c.vectors_inv);
        t.rr = row_vector.x;
        const uint32_t h2 = row_vector.y;
        t.is_value = h2 >= c.heads;
        t.head = t.is_value ? h2 - c.heads : h2;
        const uint64_t row = row0 + t.rr;
        t.slot = slots[row];
        t.p = t.is_value ? (const T *)in.values + row * in.value_row + t.head * in.value_head
                         : (const T *)in.keys + row * in.key_row + t.head * in.key_head;
        if (wide) {
            constexpr int PER = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 8; j += PER) {
                const vec<T, PER> x = *(const vec<T, PER> *)(t.p + from + j);
#pragma unroll
                for (int e = 0; e < PER; e++) t.x[j + e] = x[e];
            }
        } else
#pragma unroll
            for (int j = 0; j < 8; j++) t.x[j] = t.p[from + j];
    };
    auto store = [&](const Item &t) {
        if (t.slot < 0 || (uint64_t)t.slot >= c.slots) return;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = here ? (float)t.x[j] : 0.0f;
        if (here && !t.is_value) turn8<T, G>(r, t.p, at, cs + t.rr * r.pairs, t.x, x);
        const uint64_t v = cache_vector(c, (uint32_t)t.slot, t.head);
        if constexpr (FMT == RL_F16 || FMT == RL_BF16) {
            using S = std::conditional_t<FMT == RL_F16, half_t, bhalf_t>;
            if (here) store_f32((S *)(t.is_value ? c.values : c.keys) + v * c.dim + at, true, x);
        } else {
            constexpr float TOP = FMT == RL_I8 ? 127.0f : 448.0f;
            // The largest magnitude by its bits, in which infinities and NaNs are the largest.
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(x[j]) & 0x7FFFFFFFu);
            const float m = __uint_as_float(group_max_bits<G>(most));
            const float step = m < INFINITY ? m / TOP : NAN;
            float y[8];
            if (step > 0x1p-90f && step < 0x1p90f) {
                // The IEEE quotient by one reciprocal: x r and its remainder's correction are correctly rounded where r is
                // the rounded 1 / step and nothing leaves the normal numbers (Markstein); a quotient so small that its remainder
                // does is far below 2^-10, where the smallest code begins, and rounds to 0 either way.
                const float r = 1.0f / step;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float z = x[j] * r;
                    y[j] = __builtin_amdgcn_fmed3f(fmaf(fmaf(-z, step, x[j]), r, z), -TOP, TOP);
                }
            } else
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = step > 0.0f ? __builtin_amdgcn_fmed3f(x[j] / step, -TOP, TOP) : 0.0f;
            if (here) {
                uint2 u = encode8<FMT>(y);
                if (FMT == RL_I8 && !t.is_value) u.x ^= KEY_SIGNS, u.y ^= KEY_SIGNS;
                *reinterpret_cast<uint2 *>((uint8_t *)(t.is_value ? c.values : c.keys) + v * c.dim + at) = u;
                if (lane == 0) (t.is_value ? c.value_steps : c.key_steps)[v] = step;
            }
        }
    };
    Item item[CACHE_AHEAD];
    const uint32_t group = threadIdx.x / G;
#pragma unroll
    for (int j = 0; j < CACHE_AHEAD; j++) load(group + j * GROUPS, item[j]);
    for (uint32_t i = threadIdx.x; i < n * r.pairs; i += CACHE_THREADS)
        cs[i] = rotary_angle(r, positions[row0 + i / r.pairs], i % r.pairs);
    if (r.pairs) __syncthreads();
    for (uint32_t i = group;;) {
#pragma unroll
        for (int j = 0; j < CACHE_AHEAD; j++)
            if (i + j * GROUPS < all) store(item[j]);
        i += CACHE_AHEAD * GROUPS;
        if (i >= all) break;
#pragma unroll
        for (int j = 0; j < CACHE_AHEAD; j++) load(i + j * GROUPS, item[j]);
    }
}

// The same mapping the other way: no work but the bytes. The 5003 rows above 7.8 us, 6.8 at least (4.6 TB/s), 64 int8 rows 2.5.
template <typename T, int FMT, int G>
__global__ void __launch_bounds__(CACHE_THREADS) k_cache_read(CacheArgs c, CacheRows out, const int64_t *slots) {
    const uint32_t lane = threadIdx.x % G, at = lane * 8;
    // At most 2^23 workgroups of 32 vectors: below 2^28.
    const uint2 row_vector = split_by(blockIdx.x * (CACHE_THREADS / G) + threadIdx.x / G, 2 * c.heads, c.vectors_inv);
    const uint64_t row = row_vector.x;
    if (row >= out.rows || at >= c.dim) return;
    const uint32_t h2 = row_vector.y;
    const bool is_value = h2 >= c.heads;
    const uint32_t head = is_value ? h2 - c.heads : h2;
    const int64_t slot = slots[row];
    float x[8];
    if (slot < 0 || (uint64_t)slot >= c.slots) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = NAN;
    } else {
        const uint64_t v = cache_vector(c, (uint32_t)slot, head);
        const void *codes = is_value ? c.values : c.keys;
        if constexpr (FMT == RL_F16 || FMT == RL_BF16) {
            using S = std::conditional_t<FMT == RL_F16, half_t, bhalf_t>;
            load_f32((const S *)codes + v * c.dim + at, true, x);
        } else {
            uint2 u = *reinterpret_cast<const uint2 *>((const uint8_t *)codes + v * c.dim + at);
            if (FMT == RL_I8 && !is_value) u.x ^= KEY_SIGNS, u.y ^= KEY_SIGNS;
            decode8<FMT>(u, x);
            const float step = (is_value ? c.value_steps : c.key_steps)[v];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= step;
        }
    }
    T *to = is_value ? (T *)out.values + row * out.value_row + head * out.value_head
                     : (T *)out.keys + row * out.key_row + head * out.key_head;
    store_f32(to + at, out.wide, x);
}

}  // namespace rl
