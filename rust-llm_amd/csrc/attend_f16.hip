// k_attend for f16 queries, a unit of its own so that the types compile side by side.
#include "attend_launch.h"

template void rl::launch_attend<rl::half_t>(const rl::AttendArgs &, rl::AttendMode, uint32_t, uint32_t, uint32_t, hipStream_t);
template void rl::launch_attend_both<rl::half_t>(const rl::AttendArgs &, const rl::AttendArgs &, uint32_t, uint32_t, uint32_t, hipStream_t);
