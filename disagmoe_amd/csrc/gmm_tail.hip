// Instantiations of the tile kernels for contractions that are no multiple of 32 long: the gated product that keeps its sums,
// and the product that takes its gradient back.
#include "gmm_tile256.h"

namespace dmoe {

template <bool TRANS_B, bool KEEP>
static int launch_tail_one(const GmmArgs &args, int tile_rows, hipStream_t stream) {
    if (tile_rows == 64) return launch_direct_one<64, 4, 1, TRANS_B, KEEP, false, 2, KEEP, true>(args, stream);
    if (tile_rows == 128) return launch_direct_one<128, 4, 2, TRANS_B, KEEP, false, 0, KEEP, true>(args, stream);
    return launch_tile256_one<TRANS_B, KEEP, false, KEEP, false, true>(args, stream);
}

int launch_tail(const GmmArgs &args, int tile_rows, bool trans_b, bool keep, hipStream_t stream) {
    if (keep) return trans_b ? launch_tail_one<true, true>(args, tile_rows, stream) : launch_tail_one<false, true>(args, tile_rows, stream);
    return trans_b ? launch_tail_one<true, false>(args, tile_rows, stream) : launch_tail_one<false, false>(args, tile_rows, stream);
}

}  // namespace dmoe
