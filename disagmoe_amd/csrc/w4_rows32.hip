// Instantiations of the 4-bit product (w4.h) for row tiles of 32.
#include "w4.h"

namespace dmoe {

int launch_w4_32(const W4Args &args, int group, bool swiglu, hipStream_t stream) { return launch_w4_rows<2, 2, 1, 8>(args, group, swiglu, stream); }

}  // namespace dmoe
