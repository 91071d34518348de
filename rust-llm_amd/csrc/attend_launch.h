// The instantiations of k_attend for one query type.
#pragma once
#include "attend.h"

namespace rl {

template <typename T, int FMT, int HD, int RT, AttendMode MODE>
void launch_attend_mode(const AttendArgs &a, uint32_t groups, hipStream_t s) {
    if (a.cache.page % 16 == 0)
        hipLaunchKernelGGL((k_attend<T, FMT, HD, RT, true, MODE>), dim3(groups), dim3(ATTEND_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_attend<T, FMT, HD, RT, false, MODE>), dim3(groups), dim3(ATTEND_THREADS), 0, s, a);
    if (MODE != ATTEND_PREFIX && !a.joins)
        hipLaunchKernelGGL((k_attend_join<T, FMT, HD, MODE>), dim3(a.rows * a.q_heads), dim3(ATTEND_THREADS), 0, s, a);
}

template <typename T, int FMT, int HD, int RT>
void launch_attend_rows(const AttendArgs &a, AttendMode mode, uint32_t groups, hipStream_t s) {
    if (mode == ATTEND_ALONE) launch_attend_mode<T, FMT, HD, RT, ATTEND_ALONE>(a, groups, s);
    else if (mode == ATTEND_PREFIX) launch_attend_mode<T, FMT, HD, RT, ATTEND_PREFIX>(a, groups, s);
    else launch_attend_mode<T, FMT, HD, RT, ATTEND_JOINED>(a, groups, s);
}

template <typename T, int FMT, int HD>
void launch_attend_dim(const AttendArgs &a, AttendMode mode, uint32_t row_tiles, uint32_t groups, hipStream_t s) {
    if (row_tiles == 2) launch_attend_rows<T, FMT, HD, 2>(a, mode, groups, s);
    else launch_attend_rows<T, FMT, HD, 1>(a, mode, groups, s);
}

template <typename T, int FMT>
void launch_attend_format(const AttendArgs &a, AttendMode mode, uint32_t row_tiles, uint32_t groups, hipStream_t s) {
    switch (attend_dim(a.cache.dim)) {
    case 64: return launch_attend_dim<T, FMT, 64>(a, mode, row_tiles, groups, s);
    case 128: return launch_attend_dim<T, FMT, 128>(a, mode, row_tiles, groups, s);
    default: return launch_attend_rows<T, FMT, 256, 1>(a, mode, groups, s);
    }
}

template <typename T, int FMT, int HD>
void launch_attend_both_dim(const AttendArgs &prefix, const AttendArgs &own, uint32_t prefix_groups, uint32_t own_groups, hipStream_t s) {
    const dim3 grid(prefix_groups + own_groups);
    if (own.cache.page % 16 == 0)
        hipLaunchKernelGGL((k_attend_both<T, FMT, HD, true>), grid, dim3(ATTEND_THREADS), 0, s, prefix, own, prefix_groups);
    else
        hipLaunchKernelGGL((k_attend_both<T, FMT, HD, false>), grid, dim3(ATTEND_THREADS), 0, s, prefix, own, prefix_groups);
    hipLaunchKernelGGL((k_attend_join<T, FMT, HD, ATTEND_JOINED>), dim3(own.rows * own.q_heads), dim3(ATTEND_THREADS), 0, s, own);
}

// Calls f with the cache's format, as the ABI lets queries of type T have it.
template <typename T, typename F>
void with_attend_format(uint32_t format, F f) {
    if constexpr (!std::is_same_v<T, bhalf_t>)
        if (format == RL_F16) return f(std::integral_constant<int, RL_F16>{});
    if constexpr (!std::is_same_v<T, half_t>)
        if (format == RL_BF16) return f(std::integral_constant<int, RL_BF16>{});
    if (format == RL_I8) return f(std::integral_constant<int, RL_I8>{});
    f(std::integral_constant<int, RL_F8>{});
}

template <typename T>
void launch_attend_both(const AttendArgs &prefix, const AttendArgs &own, uint32_t format, uint32_t prefix_groups, uint32_t own_groups,
                        hipStream_t s) {
    with_attend_format<T>(format, [&](auto f) {
        constexpr int FMT = decltype(f)::value;
        switch (attend_dim(own.cache.dim)) {
        case 64: return launch_attend_both_dim<T, FMT, 64>(prefix, own, prefix_groups, own_groups, s);
        case 128: return launch_attend_both_dim<T, FMT, 128>(prefix, own, prefix_groups, own_groups, s);
        default: return launch_attend_both_dim<T, FMT, 256>(prefix, own, prefix_groups, own_groups, s);
        }
    });
}

template <typename T>
void launch_attend(const AttendArgs &a, AttendMode mode, uint32_t format, uint32_t row_tiles, uint32_t groups, hipStream_t s) {
    with_attend_format<T>(format, [&](auto f) { launch_attend_format<T, decltype(f)::value>(a, mode, row_tiles, groups, s); });
}

}  // namespace rl
