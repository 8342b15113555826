// Instantiations of the 4-bit product (w4.h) for row tiles of 64.
#include "w4.h"

namespace dmoe {

// Workgroups of 128 columns, 4 wavefronts along k, as long as one round of them holds the work; of 256 columns, 2 along k, from
// there on.  (A workgroup fills a compute unit, and the row tiles of a column tile run on one XCD: the XCD with most of the column
// tiles decides.)  Measured, 64 rows an expert, in us, as (128, 4) / (256, 2):
//                                               groups of 128   64, zero points   32           32, zero points
//   K 14336,  4 experts x 4096 (16 to an XCD)      91 / 119        95 / 161       100 / 164     126 / 209
//             8 experts x 4096 (32, one round)    105 / 128       115 / 177       121 / 182     153 / 230
//             9 experts x 3584 (36)               186 / 125       193 / 173       204 / 178     265 / 229
//            13 experts x 4096 (52)               212 / 141       204 / 183       217 / 195     274 / 240
//   K 4096,   4, 8                       31 / 38, 37 / 41  33 / 51, 38 / 53  34 / 52, 40 / 54  44 / 65, 49 / 68
//             9, 13                      60 / 40, 65 / 43  63 / 51, 66 / 54  65 / 52, 69 / 57  84 / 65, 88 / 68
//   K 1024,   4, 8                       12 / 14, 15 / 16  13 / 17, 16 / 19  14 / 18, 16 / 19  16 / 21, 20 / 23
//             9, 13                      25 / 15, 28 / 17  26 / 19, 30 / 21  27 / 19, 29 / 20  34 / 22, 37 / 24
int launch_w4_64(const W4Args &args, int group, bool swiglu, hipStream_t stream) {
    const long long columns = (args.N + 127) / 128;
    const bool one_round = (columns + kXcds - 1) / kXcds * args.m_tiles * kXcds <= device_cus();
    // Two forms of four wavefronts along k spill in their loops (groups of 64 without and of 128 with zero points); a fragment
    // less and twice the wavefronts along the columns do not, nor do they need as many registers for the rows.  (128, 4) / this,
    // 8 experts x 4096: K 14336: 124 / 113 and 217 / 105, K 4096: 43 / 36 and 63 / 33, K 1024: 18 / 14 and 24 / 13; 1 expert x 512:
    // 83 / 83 and 130 / 81, 29 / 27 and 43 / 26, 13 / 10 and 17 / 10; where the others lose: 95 / 99 (groups of 128), 100 / 121 (of 64
    // with zero points), 107 / 127 (of 32).  (Up columns that begin inside a tile leave one fragment in either form: 9.7 / 11.4 on
    // 130 row tiles of 64 columns, K 1024.)
    const bool spills = group != 32 && (group == 64) == (args.zeros == nullptr) && !(swiglu && args.n_out % 16 != 0);
    if (one_round && spills) return launch_w4_rows<4, 1, 4, 2>(args, group, swiglu, stream);
    if (one_round) return launch_w4_rows<4, 2, 2, 4>(args, group, swiglu, stream);
    return launch_w4_rows<4, 2, 4, 2>(args, group, swiglu, stream);
}

}  // namespace dmoe
