// k_attend_shared for f32 queries, a unit of its own so that the types compile side by side.
#define RL_SHARED_UNIT
#include "attend_shared.h"

template void rl::launch_attend_shared<float>(const rl::AttendArgs &, uint32_t, bool, uint32_t, hipStream_t);
