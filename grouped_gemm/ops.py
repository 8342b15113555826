"""grouped_gemm.ops by the upstream package's name: gmm under autograd, and gmm_swiglu (same module object as disagmoe_amd.grouped_gemm.ops)."""
import sys

import disagmoe_amd.grouped_gemm.ops as _impl

sys.modules[__name__] = _impl
