// Rotary positions (include/rl_mixers.h): the angles, and the kernel that turns
// the heads of one or two tensors. The cache write (kv_cache.h) turns keys with
// the same angles.
#pragma once
#include "mix_types.h"

namespace rl {

constexpr uint32_t ROTARY_MAX_PAIRS = 256;

// What a kernel needs of a rotary handle. turns: revolutions a position of each pair.
struct RotaryArgs {
    const double *turns;
    uint32_t pairs;
    uint32_t interleaved;
    float magnitude;
    float sign; // -1: the negative angles
};

// (m cos, m sin) of pair i at a position. The revolutions are formed and reduced
// in f64: position * f_i is exact to 2^-53 of itself, and only the fraction of a
// revolution left over is rounded to f32 (an angle error below 2e-7).
__device__ inline float2 rotary_angle(const RotaryArgs &r, int64_t position, uint32_t i) {
    const double t = (double)position * r.turns[i];
    const float x = 2.0f * (float)(t - rint(t));
    float s, c;
    sincospif(x, &s, &c);
    return make_float2(r.magnitude * c, r.sign * (r.magnitude * s));
}

__device__ inline float turn_a(float a, float b, float2 cs) { return a * cs.x - b * cs.y; }
__device__ inline float turn_b(float a, float b, float2 cs) { return a * cs.y + b * cs.x; }

struct RotaryTensor {
    const void *in;
    void *out;
    uint64_t in_row, in_head, out_row, out_head;
    uint32_t heads, dim;
    uint32_t units; // of V values (half layout: V pairs) in a head
    uint32_t wide;  // whether the 16-byte accesses are aligned
};

constexpr uint32_t ROTARY_THREADS = 256;

// A unit of V values (V pairs of the half layout) of a head.
template <typename TI, typename TO, int V, bool INTERLEAVED>
__device__ inline void rotary_unit(const RotaryTensor &t, uint32_t u, uint64_t row, uint32_t pairs,
                                   const float2 *cs) {
    const uint32_t head = u / t.units, at = u - head * t.units;
    const TI *in = (const TI *)t.in + row * t.in_row + head * t.in_head;
    TO *out = (TO *)t.out + row * t.out_row + head * t.out_head;
    const bool wide = t.wide;
    const uint32_t turned = (INTERLEAVED ? 2 * pairs : pairs) / V; // units that are turned
    if (at < turned) {
        if constexpr (INTERLEAVED) {
            float x[V], y[V];
            load_f32(in + at * V, wide, x);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 w = cs[(at * V + j) / 2];
                y[j] = turn_a(x[j], x[j + 1], w);
                y[j + 1] = turn_b(x[j], x[j + 1], w);
            }
            store_f32(out + at * V, wide, y);
        } else {
            float a[V], b[V], y[V], z[V];
            load_f32(in + at * V, wide, a);
            load_f32(in + pairs + at * V, wide, b);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float2 w = cs[at * V + j];
                y[j] = turn_a(a[j], b[j], w);
                z[j] = turn_b(a[j], b[j], w);
            }
            store_f32(out + at * V, wide, y);
            store_f32(out + pairs + at * V, wide, z);
        }
    } else if ((const void *)in != (const void *)out) { // past the turned values: copied
        float x[V];
        const uint32_t e = 2 * pairs + (at - turned) * V;
        if (e + V <= t.dim) {
            load_f32(in + e, wide, x);
            store_f32(out + e, wide, x);
        } else
            for (uint32_t j = e; j < t.dim; j++) out[j] = (TO)(float)in[j];
    }
}

// One workgroup a row: the row's angles go to LDS once (an f64 product and a sincos
// a pair, shared by all heads), then every thread takes units of any head, 16 bytes
// where alignment allows. Bound by HBM, each value is read and written once: 4096
// f32 rows of 40 heads of 128 take 33.9 us, 4.95 TB/s, as a large copy does. One
// row is the chain of position, angle, barrier and turn: 3.8 us.
template <typename TI, typename TO, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(ROTARY_THREADS) k_rotary(RotaryArgs r, const int64_t *positions, RotaryTensor a,
                                                           RotaryTensor b) {
    __shared__ float2 cs[ROTARY_MAX_PAIRS];
    const uint64_t row = blockIdx.x;
    const int64_t position = positions[row];
    for (uint32_t i = threadIdx.x; i < r.pairs; i += ROTARY_THREADS) cs[i] = rotary_angle(r, position, i);
    __syncthreads();
    const uint32_t ua = a.heads * a.units, all = ua + b.heads * b.units;
    for (uint32_t u = threadIdx.x; u < all; u += ROTARY_THREADS) {
        if (u < ua)
            rotary_unit<TI, TO, V, INTERLEAVED>(a, u, row, r.pairs, cs);
        else
            rotary_unit<TI, TO, V, INTERLEAVED>(b, u - ua, row, r.pairs, cs);
    }
}

}  // namespace rl
