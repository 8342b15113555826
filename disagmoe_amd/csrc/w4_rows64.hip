// Instantiations of the 4-bit product (w4.h) for row tiles of 64.
#include "w4.h"

namespace dmoe {

// As launch_w4_16.  Measured, 64 rows an expert, groups of 128, in us, as (128 columns, 4 wavefronts along k) / (256, 2): 512
// units, K 14336: 94.5 / 122.3; the same with 256 rows (2048 units): 395.6 / 289.5; 704 units, K 1024: 26.6 / 15.9.
int launch_w4_64(const W4Args &args, int group, bool swiglu, hipStream_t stream) {
    const long long units = (long long)((args.N + 63) / 64) * args.m_tiles;
    if (units < 640) return launch_w4_rows<4, 2, 2, 4>(args, group, swiglu, stream);
    return launch_w4_rows<4, 2, 4, 2>(args, group, swiglu, stream);
}

}  // namespace dmoe
