// Leaky attention on float32 tensors: the kernels of attention_pass.h.
#include "attention_pass.h"

namespace slayer {

template <>
int launch_leaky<float>(const LeakyPass& p, int mode, bool whole, hipStream_t stream) {
    const bool main = mode != LEAKY_STATE && mode != LEAKY_STATE_SLOPE;
    const int64_t blocks = (int64_t)p.units * (main ? p.segments : p.segments - 1) * p.slices;
    if (blocks == 0) return 0;
    if (blocks > (1 << 24) - 1) return SLAYER_ERANGE;                        // fewer than 2^32 threads in a launch
    const dim3 grid((unsigned)blocks);
    switch (mode) {
        case LEAKY_STATE: return launch_leaky_mode<float, LEAKY_STATE>(p, grid, whole, stream);
        case LEAKY_MAIN: return launch_leaky_mode<float, LEAKY_MAIN>(p, grid, whole, stream);
        case LEAKY_BOTH: return launch_leaky_both<float>(p, grid, stream);
        case LEAKY_STATE_SLOPE: return launch_leaky_mode<float, LEAKY_STATE_SLOPE>(p, grid, whole, stream);
        default: return launch_leaky_mode<float, LEAKY_SLOPE>(p, grid, whole, stream);
    }
}

}  // namespace slayer
