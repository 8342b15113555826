// Instantiations of the 4-bit product (w4.h) for row tiles of 64.
#include "w4.h"

namespace dmoe {

int launch_w4_64(const W4Args &args, int group, bool swiglu, hipStream_t stream) { return launch_w4_rows<4, 2, 4, 2>(args, group, swiglu, stream); }

}  // namespace dmoe
