// Instantiations of the gated bf16 product that also leaves its fp32 sums for the gradient.
#include "gmm_tile256.h"

namespace dmoe {

// Preconditions and tile_rows as launch_direct_bf16's.
int launch_direct_keep(const GmmArgs &args, int tile_rows, bool trans_b, hipStream_t stream) {
    if (tile_rows == 64)
        return trans_b ? launch_direct_one<64, 4, 1, true, true, false, 2, true>(args, stream) : launch_direct_one<64, 4, 1, false, true, false, 2, true>(args, stream);
    if (tile_rows == 128)
        return trans_b ? launch_direct_one<128, 4, 2, true, true, false, 0, true>(args, stream) : launch_direct_one<128, 4, 2, false, true, false, 0, true>(args, stream);
    return trans_b ? launch_tile256_one<true, true, false, true>(args, stream) : launch_tile256_one<false, true, false, true>(args, stream);
}

}  // namespace dmoe
