// Instantiations of the gated bf16 product that also leaves its fp32 sums for the gradient.  The sums are 8 bytes for every 2
// of the result: 8192 rows on 8 experts of 4096 x 28672: 1637 - 1734 us (0.94 GB of sums on top of 3.5 GB of other traffic; the
// form without them 1540), 64 experts of 768 rows, 2048 x 2816: 637 - 676 us.
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
