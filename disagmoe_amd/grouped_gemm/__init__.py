"""``grouped_gemm`` as the reference imports it: the ``backend`` module (``gmm``, ``get_arguments``,
``gmm_with_arguments``) on the HIP grouped GEMM, and ``ops``, the same products under autograd (the upstream package's
name for them; the expert-worker path itself trains nothing)."""
from . import backend, ops  # noqa: F401
