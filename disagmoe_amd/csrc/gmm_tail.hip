// Instantiations of the 256 x 256 tile kernel for contractions that are no multiple of 32 long: the gated product that keeps
// its sums, and the product that takes its gradient back.
#include "gmm_tile256.h"

namespace dmoe {

int launch_tile256_tail(const GmmArgs &args, bool trans_b, bool keep, hipStream_t stream) {
    if (keep)
        return trans_b ? launch_tile256_one<true, true, false, true, false, true>(args, stream) : launch_tile256_one<false, true, false, true, false, true>(args, stream);
    return trans_b ? launch_tile256_one<true, false, false, false, false, true>(args, stream) : launch_tile256_one<false, false, false, false, false, true>(args, stream);
}

}  // namespace dmoe
