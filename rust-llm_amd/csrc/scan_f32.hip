// The scan's kernels for f32, a unit of its own so that the types compile side by side.
#define RL_SCAN_UNIT
#include "scan.h"

template void rl::launch_scan_steps<float>(const rl::ScanArgs &, hipStream_t);
template void rl::launch_scan<float>(const rl::ScanArgs &, hipStream_t);
