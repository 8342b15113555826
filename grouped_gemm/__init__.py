"""``grouped_gemm`` as the reference imports it: the ``backend`` module (``gmm``, ``get_arguments``,
``gmm_with_arguments``) on the HIP grouped GEMM, and the upstream package's name ``ops`` for the products under autograd."""
from . import backend, ops  # noqa: F401
