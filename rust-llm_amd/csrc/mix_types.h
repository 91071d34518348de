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

template <int FMT>
__device__ inline uint2 encode8(const float (&x)[8]) {
    uint32_t u[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if constexpr (FMT == RL_I8) {
            u[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) u[i] |= ((uint32_t)(int32_t)rintf(x[4 * i + j]) & 255u) << (8 * j);
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

// Sum and maximum over the aligned group of N lanes that holds the caller, N a power of two.
template <int N>
__device__ inline float group_sum(float x) {
#pragma unroll
    for (int d = 1; d < N; d *= 2) x += __shfl_xor(x, d);
    return x;
}
template <int N>
__device__ inline float group_max(float x) {
#pragma unroll
    for (int d = 1; d < N; d *= 2) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}

}  // namespace rl
