// The instantiations of k_attend for one query type.
#pragma once
#include "attend.h"

namespace rl {

template <typename T, int FMT, int HD, int RT>
void launch_attend_rows(const AttendArgs &a, uint32_t groups, hipStream_t s) {
    if (a.cache.page % 16 == 0)
        hipLaunchKernelGGL((k_attend<T, FMT, HD, RT, true>), dim3(groups), dim3(ATTEND_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_attend<T, FMT, HD, RT, false>), dim3(groups), dim3(ATTEND_THREADS), 0, s, a);
    if (a.parts > 1 && !a.joins) hipLaunchKernelGGL((k_attend_join<T, FMT, HD>), dim3(a.rows * a.q_heads), dim3(ATTEND_THREADS), 0, s, a);
}

template <typename T, int FMT>
void launch_attend_format(const AttendArgs &a, bool two, uint32_t groups, hipStream_t s) {
    switch (attend_dim(a.cache.dim)) {
    case 64: return two ? launch_attend_rows<T, FMT, 64, 2>(a, groups, s) : launch_attend_rows<T, FMT, 64, 1>(a, groups, s);
    case 128: return two ? launch_attend_rows<T, FMT, 128, 2>(a, groups, s) : launch_attend_rows<T, FMT, 128, 1>(a, groups, s);
    default: return launch_attend_rows<T, FMT, 256, 1>(a, groups, s);
    }
}

template <typename T>
void launch_attend(const AttendArgs &a, uint32_t format, bool two, uint32_t groups, hipStream_t s) {
    // The ABI has refused the 16-bit format that is not the queries' own.
    if constexpr (!std::is_same_v<T, bhalf_t>)
        if (format == RL_F16) return launch_attend_format<T, RL_F16>(a, two, groups, s);
    if constexpr (!std::is_same_v<T, half_t>)
        if (format == RL_BF16) return launch_attend_format<T, RL_BF16>(a, two, groups, s);
    if (format == RL_I8) return launch_attend_format<T, RL_I8>(a, two, groups, s);
    launch_attend_format<T, RL_F8>(a, two, groups, s);
}

}  // namespace rl
