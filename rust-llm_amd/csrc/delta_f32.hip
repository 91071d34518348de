// The delta rule's kernels for f32 tensors, a unit of its own so that the types
// compile side by side.
#define RL_DELTA_UNIT
#include "delta_launch.h"

template void rl::launch_delta_steps<float>(const rl::DeltaArgs &, hipStream_t);
template void rl::launch_delta_chunks<float>(const rl::DeltaArgs &, const rl::DeltaWork &, hipStream_t);
