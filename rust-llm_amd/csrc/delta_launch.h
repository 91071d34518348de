// Launches of the delta rule's kernels for one element type (delta_*.hip, one unit
// a type).
#pragma once
#include "delta_chunks.h"

namespace rl {

template <typename T>
void launch_delta_steps(const DeltaArgs &a, hipStream_t s);
template <typename T>
void launch_delta_chunks(const DeltaArgs &a, const DeltaWork &w, hipStream_t s);

// Waves of 16 columns up to which waves of 8 take their place. 9 rows of 32 heads of 128 x 128, us, 16 / 8 columns: one
// bf16 sequence (256 waves) 13.7 / 12.5, f32 12.4 / 11.0. With every SIMD busy the reductions cost, and 16 columns need fewer.
constexpr uint32_t DELTA_FEW = 512;

// Workgroups of k_delta_chunks: a sequence's heads in eights, 16 columns each.
inline uint64_t delta_groups(const DeltaArgs &a) {
    return ((uint64_t)a.seqs * a.value_heads + 7) / 8 * 8 * (a.value_dim / 16);
}

#ifdef RL_DELTA_UNIT
template <typename T, int Q>
void launch_delta_steps_of(const DeltaArgs &a, hipStream_t s) {
    constexpr uint32_t PER = 4 * Q * DELTA_WAVES;
    auto kern = a.key_dim <= 64 ? k_delta_steps<T, Q, Q> : a.key_dim <= 128 ? k_delta_steps<T, 2 * Q, Q> : k_delta_steps<T, 4 * Q, Q>;
    hipLaunchKernelGGL(kern, dim3(a.seqs * a.value_heads, (a.value_dim + PER - 1) / PER), dim3(64 * DELTA_WAVES), 0, s, a);
}

template <typename T>
void launch_delta_steps(const DeltaArgs &a, hipStream_t s) {
    if ((uint64_t)a.seqs * a.value_heads * (a.value_dim / 16) <= DELTA_FEW) launch_delta_steps_of<T, 2>(a, s);
    else launch_delta_steps_of<T, 4>(a, s);
}

template <typename T, int DK>
void launch_delta_chunks_dim(const DeltaArgs &a, const DeltaWork &w, hipStream_t s) {
    hipLaunchKernelGGL((k_delta_prepare<T, DK>), dim3((a.rows / CHUNK + a.seqs) * a.value_heads), dim3(256), 0, s, a, w);
    hipLaunchKernelGGL((k_delta_chunks<T, DK>), dim3((uint32_t)delta_groups(a)), dim3(DELTA_CHUNK_THREADS), 0, s, a, w);
}

template <typename T>
void launch_delta_chunks(const DeltaArgs &a, const DeltaWork &w, hipStream_t s) {
    switch (delta_dim(a.key_dim)) {
    case 64: return launch_delta_chunks_dim<T, 64>(a, w, s);
    case 128: return launch_delta_chunks_dim<T, 128>(a, w, s);
    default: return launch_delta_chunks_dim<T, 256>(a, w, s);
    }
}
#endif

}  // namespace rl
