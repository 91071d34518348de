// k_attend for f32 queries, a unit of its own so that the types compile side by side.
#include "attend_launch.h"

template void rl::launch_attend<float>(const rl::AttendArgs &, rl::AttendMode, uint32_t, uint32_t, uint32_t, hipStream_t);
template void rl::launch_attend_both<float>(const rl::AttendArgs &, const rl::AttendArgs &, uint32_t, uint32_t, uint32_t, hipStream_t);
