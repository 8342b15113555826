// Instantiations of the 256 x 256 tile kernel for fp16 operands with scales (the 4-bit weights' form for many rows, w4.hip).
// 8192 rows on 8 experts of 4096 x 28672, gated: 1645 - 1765 us, 1090 - 1170 TFLOP/s, the rate of the bf16 build.
#include "gmm_tile256.h"

namespace dmoe {

int launch_tile256_half(const GmmArgs &args, bool swiglu, hipStream_t stream) {
    return swiglu ? launch_tile256_one<true, true, false, false, true>(args, stream) : launch_tile256_one<true, false, false, false, true>(args, stream);
}

}  // namespace dmoe
