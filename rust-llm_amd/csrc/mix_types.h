// Element types of the token mixers: loads, stores and conversions of vectors of
// f32, f16 and bf16, and the 8-bit cache formats. Conversions from f32 round to
// nearest, ties to even.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "rl_mixers.h"

namespace rl {

typedef _Float16 half_t;
typedef __bf16 bhalf_t;

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));
typedef vec<float, 4> f32x4;

// (t / d, t % d) with inverse_of(d).
inline uint32_t inverse_of(uint32_t d) { return d > 1 ? (uint32_t)((1ull << 32) / d) : 0xFFFFFFFFu; }
__device__ inline uint2 split_by(uint32_t t, uint32_t d, uint32_t inv) { // (t / d, t % d)
    uint32_t q = __umulhi(t, inv), r = t - q * d; // the quotient, or one less
    if (r >= d) q++, r -= d;
    return make_uint2(q, r);
}

// N values at p as f32. `wide`: p is a multiple of 16 bytes (of the vector's size, if that is less).
template <int N, typename T>
__device__ inline void load_f32(const T *p, bool wide, float (&x)[N]) {
    constexpr int PER = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
    if (wide) {
#pragma unroll
        for (int i = 0; i < N; i += PER) {
            const vec<T, PER> v = *reinterpret_cast<const vec<T, PER> *>(p + i);
#pragma unroll
            for (int j = 0; j < PER; j++) x[i + j] = (float)v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = (float)p[i];
    }
}

template <int N, typename T>
__device__ inline void store_f32(T *p, bool wide, const float (&x)[N]) {
    constexpr int PER = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
    if (wide) {
#pragma unroll
        for (int i = 0; i < N; i += PER) {
            vec<T, PER> v;
#pragma unroll
            for (int j = 0; j < PER; j++) v[j] = (T)x[i + j];
            *reinterpret_cast<vec<T, PER> *>(p + i) = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = (T)x[i];
    }
}

// Eight bytes of a cache format as f32 (unscaled codes), and back.
template <int FMT>
__device__ inline void decode8(uint2 w, float (&x)[8]) {
    const uint32_t u[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if constexpr (FMT == RL_I8) {
#pragma unroll
            for (int j = 0; j < 4; j++) x[4 * i + j] = (float)(int8_t)(u[i] >> (8 * j));
        } else {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], false);
            const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], true);
            x[4 * i] = lo[0], x[4 * i + 1] = lo[1], x[4 * i + 2] = hi[0], x[4 * i + 3] = hi[1];
        }
    }
}

// x within the format's range.
template <int FMT>
__device__ inline uint2 encode8(const float (&x)[8]) {
    uint32_t u[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if constexpr (FMT == RL_I8) { // x + 1.5 2^23 has rint(x) in its last byte
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) b[j] = __float_as_uint(x[4 * i + j] + 12582912.0f);
            u[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u),
                                         __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), 0x05040100u);
        } else {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
            u[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
        }
    }
    return make_uint2(u[0], u[1]);
}

// The other half of a swap: lanes 16 apart (of 32) and 32 apart, without LDS.
__device__ inline float2 swap16(float x) { // each lane's own row of 16 and its neighbour's, in some order
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float2 swap32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Over the four lanes 16 apart.
__device__ inline float rows_max(float x) {
    float2 y = swap16(x);
    y = swap32(fmaxf(y.x, y.y));
    return fmaxf(y.x, y.y);
}
__device__ inline float rows_sum(float x) {
    float2 y = swap16(x);
    y = swap32(y.x + y.y);
    return y.x + y.y;
}

// Of the lane N further on in its row of 16, cyclically.
template <int N>
__device__ inline float rotate16(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + N, 0xf, 0xf, false));
}

// f over the aligned group of N lanes that holds the caller, N a power of two up to 64, the result in every lane. Without
// LDS: by quads, halves of a row of 16, rows, and rows swapped.
template <int CTRL>
__device__ inline float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false));
}
template <int N, typename F>
__device__ inline float group_reduce(float x, F f) {
    if constexpr (N > 1) x = f(x, dpp<0xB1>(x));  // lanes 1 0 3 2
    if constexpr (N > 2) x = f(x, dpp<0x4E>(x));  // lanes 2 3 0 1
    if constexpr (N > 4) x = f(x, dpp<0x141>(x)); // mirrored in eights
    if constexpr (N > 8) x = f(x, dpp<0x140>(x)); // mirrored in sixteens
    if constexpr (N > 16) {
        const float2 y = swap16(x);
        x = f(y.x, y.y);
    }
    if constexpr (N > 32) {
        const float2 y = swap32(x);
        x = f(y.x, y.y);
    }
    return x;
}
template <int N>
__device__ inline float group_sum(float x) {
    return group_reduce<N>(x, [](float a, float b) { return a + b; });
}
template <int N>
__device__ inline float group_max(float x) {
    return group_reduce<N>(x, [](float a, float b) { return fmaxf(a, b); });
}

// The largest of numbers that order as unsigned integers.
template <int N>
__device__ inline uint32_t group_max_bits(uint32_t x) {
    return __float_as_uint(group_reduce<N>(__uint_as_float(x), [](float a, float b) {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }));
}

}  // namespace rl
