// k_attend for bf16 queries, a unit of its own so that the types compile side by side.
#include "attend_launch.h"

template void rl::launch_attend<rl::bhalf_t>(const rl::AttendArgs &, uint32_t, bool, uint32_t, hipStream_t);
