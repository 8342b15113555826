// Instantiations of the 4-bit product (w4.h) for row tiles of 32.
#include "w4.h"

namespace dmoe {

// As launch_w4_16.  Measured, 32 rows an expert, groups of 128, in us, as (64 columns, 4 wavefronts along k) / (128, 2): 512
// units, K 14336: 69.4 / 81.6; 704 units, K 1024: 12.1 / 13.5; 2048 units, K 1408: 43.6 / 37.5; 2816 units, K 2048: 83.6 / 63.1.
int launch_w4_32(const W4Args &args, int group, bool swiglu, hipStream_t stream) {
    const long long units = (long long)((args.N + 63) / 64) * args.m_tiles;
    if (units < 1024) return launch_w4_rows<2, 2, 1, 4>(args, group, swiglu, stream);
    return launch_w4_rows<2, 2, 2, 2>(args, group, swiglu, stream);
}

}  // namespace dmoe
