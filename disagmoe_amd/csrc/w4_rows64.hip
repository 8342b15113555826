// Instantiations of the 4-bit product (w4.h) for row tiles of 64.
#include "w4.h"

namespace dmoe {

// As launch_w4_16.  Measured, 64 rows an expert, groups of 128, in us, as (128 columns, 4 wavefronts along k) / (256, 2): 512
// units, K 14336: 94.5 / 122.3; the same with 256 rows (2048 units): 395.6 / 289.5; 704 units, K 1024: 26.6 / 15.9.
int launch_w4_64(const W4Args &args, int group, bool swiglu, hipStream_t stream) {
    const long long units = (long long)((args.N + 63) / 64) * args.m_tiles;
    // Two forms of four wavefronts along k spill in their loops (groups of 64 without and of 128 with zero points); a fragment
    // less and twice the wavefronts along the columns do not, nor do they need as many registers for the rows.  512 units, K
    // 14336: 141 / 107 and 180 / 101 us, where the others lose: 95 / 99 (groups of 128), 100 / 121 (of 64 with zero points), 107 /
    // 127 (of 32).  (Up columns that begin inside a tile leave one fragment in either form: 9.7 / 11.4 on 130 units, K 1024.)
    const bool spills = group != 32 && (group == 64) == (args.zeros == nullptr) && !(swiglu && args.n_out % 16 != 0);
    if (units < 640 && spills) return launch_w4_rows<4, 1, 4, 2>(args, group, swiglu, stream);
    if (units < 640) return launch_w4_rows<4, 2, 2, 4>(args, group, swiglu, stream);
    return launch_w4_rows<4, 2, 4, 2>(args, group, swiglu, stream);
}

}  // namespace dmoe
