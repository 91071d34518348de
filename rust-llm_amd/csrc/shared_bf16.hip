// k_attend_shared for bf16 queries, a unit of its own so that the types compile side by side.
#define RL_SHARED_UNIT
#include "attend_shared.h"

template void rl::launch_attend_shared<rl::bhalf_t>(const rl::AttendArgs &, uint32_t, bool, uint32_t, hipStream_t);
