// Instantiations of the 4-bit product (w4.h) for row tiles of 16.
#include "w4.h"

namespace dmoe {

// Columns of a workgroup and wavefronts along k by the work there is to fill the chip with (units of 64 columns of the
// weights x row tiles; 256 compute units, 16 wavefronts each).  Measured, one row an expert, groups of 128, in us, as
// (32 columns, 8 along k) / (64, 8) / (64, 4) / (128, 4): 128 units, K 14336: 16.2 / 20.6 / 33.1 / 34.6; 512 units, K 14336:
// 42.2 / 40.6 / 43.9 / 43.2; 704 units, K 1024: 11.2 / 8.7 / 7.2 / 8.0; 2816 units, K 2048: 51.7 / 42.2 / 35.5 / 36.6, and with 16
// rows an expert 79.9 / 59.1 / 56.7 / 46.2 (two wavefronts read the rows from the L1 cache that one has brought).
int launch_w4_16(const W4Args &args, int group, bool swiglu, hipStream_t stream) {
    const long long units = (long long)((args.N + 63) / 64) * args.m_tiles;
    if (units < 256) return launch_w4_rows<1, 1, 1, 8>(args, group, swiglu, stream);
    if (units < 640) return launch_w4_rows<1, 2, 1, 8>(args, group, swiglu, stream);
    if (units < 2048) return launch_w4_rows<1, 2, 1, 4>(args, group, swiglu, stream);
    return launch_w4_rows<1, 2, 2, 4>(args, group, swiglu, stream);
}

}  // namespace dmoe
