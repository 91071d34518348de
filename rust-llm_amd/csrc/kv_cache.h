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
    uint64_t slots;
    uint32_t page, heads, dim;
};

// The vector of a slot and head, counted in vectors of dim values.
__device__ inline uint64_t cache_vector(const CacheArgs &c, uint64_t slot, uint32_t head) {
    const uint64_t p = slot / c.page;
    return (p * c.heads + head) * c.page + (slot - p * c.page);
}

struct CacheRows {
    const void *keys, *values; // outputs of a read
    uint64_t key_row, key_head, value_row, value_head;
    uint32_t rows;
    uint32_t wide; // whether 16-byte accesses to them are aligned
};

constexpr uint32_t CACHE_THREADS = 256;
constexpr uint32_t CACHE_MAX_ROWS = 16; // rows a workgroup, LDS holds their angles

// Eight values of a head's key, turned if they are among the turned ones. A
// partner that another lane holds is read again (it is in the cache).
template <typename T>
__device__ inline void turned8(const RotaryArgs &r, const T *in, bool wide, uint32_t at, const float2 *cs,
                               float (&x)[8]) {
    const uint32_t turned = 2 * r.pairs;
    load_f32(in + at, wide, x);
    if (at >= turned) return;
    if (!r.interleaved && r.pairs % 8 == 0) {
        const bool second = at >= r.pairs;
        const uint32_t i = second ? at - r.pairs : at;
        float y[8];
        load_f32(in + (second ? i : at + r.pairs), wide, y);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = second ? turn_b(y[j], x[j], cs[i + j]) : turn_a(x[j], y[j], cs[i + j]);
    } else {
        for (int j = 0; j < 8 && at + j < turned; j++) {
            const uint32_t e = at + j;
            if (r.interleaved) {
                const float2 w = cs[e / 2];
                x[j] = e & 1 ? turn_b((float)in[e - 1], (float)in[e], w) : turn_a((float)in[e], (float)in[e + 1], w);
            } else if (e < r.pairs)
                x[j] = turn_a((float)in[e], (float)in[e + r.pairs], cs[e]);
            else
                x[j] = turn_b((float)in[e - r.pairs], (float)in[e], cs[e - r.pairs]);
        }
    }
}

// G lanes hold a vector of up to 8 G values, eight a lane. Vectors of a workgroup's
// rows: keys of every head, then values of every head. One pass: the largest
// magnitude is reduced over the lanes while the values stay in registers.
template <typename T, int FMT, int G>
__global__ void __launch_bounds__(CACHE_THREADS) k_cache_write(CacheArgs c, CacheRows in, const int64_t *slots,
                                                               uint32_t rows_a_group, RotaryArgs r,
                                                               const int64_t *positions) {
    __shared__ float2 cs[CACHE_MAX_ROWS * ROTARY_MAX_PAIRS / 2];
    const uint32_t row0 = blockIdx.x * rows_a_group, n = min(rows_a_group, in.rows - row0);
    for (uint32_t i = threadIdx.x; i < n * r.pairs; i += CACHE_THREADS)
        cs[i] = rotary_angle(r, positions[row0 + i / r.pairs], i % r.pairs);
    if (r.pairs) __syncthreads();
    const uint32_t lane = threadIdx.x % G, at = lane * 8;
    const bool here = at < c.dim, wide = in.wide;
    for (uint32_t i = threadIdx.x / G; i < n * 2 * c.heads; i += CACHE_THREADS / G) {
        const uint32_t rr = i / (2 * c.heads), h2 = i - rr * 2 * c.heads;
        const bool is_value = h2 >= c.heads;
        const uint32_t head = is_value ? h2 - c.heads : h2;
        const uint64_t row = row0 + rr;
        const int64_t slot = slots[row];
        if (slot < 0 || (uint64_t)slot >= c.slots) continue;
        float x[8] = {};
        if (here) {
            if (is_value)
                load_f32((const T *)in.values + row * in.value_row + head * in.value_head + at, wide, x);
            else
                turned8(r, (const T *)in.keys + row * in.key_row + head * in.key_head, wide, at, cs + rr * r.pairs, x);
        }
        const uint64_t v = cache_vector(c, (uint64_t)slot, head);
        if constexpr (FMT == RL_F16 || FMT == RL_BF16) {
            using S = std::conditional_t<FMT == RL_F16, half_t, bhalf_t>;
            if (here) store_f32((S *)(is_value ? c.values : c.keys) + v * c.dim + at, true, x);
        } else {
            constexpr float TOP = FMT == RL_I8 ? 127.0f : 448.0f;
            float m = 0.0f;
            bool bad = false; // an infinity or a NaN
#pragma unroll
            for (int j = 0; j < 8; j++) {
                m = fmaxf(m, fabsf(x[j]));
                bad |= !(fabsf(x[j]) < INFINITY);
            }
            m = group_max<G>(bad ? INFINITY : m);
            const float step = m < INFINITY ? m / TOP : NAN;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = step > 0.0f ? fminf(fmaxf(x[j] / step, -TOP), TOP) : 0.0f;
            if (here) {
                uint2 u = encode8<FMT>(y);
                if (FMT == RL_I8 && !is_value) u.x ^= KEY_SIGNS, u.y ^= KEY_SIGNS;
                *reinterpret_cast<uint2 *>((uint8_t *)(is_value ? c.values : c.keys) + v * c.dim + at) = u;
                if (lane == 0) (is_value ? c.value_steps : c.key_steps)[v] = step;
            }
        }
    }
}

// The same mapping the other way.
template <typename T, int FMT, int G>
__global__ void __launch_bounds__(CACHE_THREADS) k_cache_read(CacheArgs c, CacheRows out, const int64_t *slots) {
    const uint32_t lane = threadIdx.x % G, at = lane * 8;
    const uint64_t i = (uint64_t)blockIdx.x * (CACHE_THREADS / G) + threadIdx.x / G;
    const uint32_t per = 2 * c.heads;
    const uint64_t row = i / per;
    if (row >= out.rows || at >= c.dim) return;
    const uint32_t h2 = (uint32_t)(i - row * per);
    const bool is_value = h2 >= c.heads;
    const uint32_t head = is_value ? h2 - c.heads : h2;
    const int64_t slot = slots[row];
    float x[8];
    if (slot < 0 || (uint64_t)slot >= c.slots) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = NAN;
    } else {
        const uint64_t v = cache_vector(c, (uint64_t)slot, head);
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
