// The scan's kernels for f16, a unit of its own so that the types compile side by side.
#define RL_SCAN_UNIT
#include "scan.h"

template void rl::launch_scan_steps<rl::half_t>(const rl::ScanArgs &, hipStream_t);
template void rl::launch_scan<rl::half_t>(const rl::ScanArgs &, hipStream_t);
