"""Sizes on the host in any integer type and stride are the same launch, bit for bit."""
import pytest
import torch

from disagmoe_amd.grouped_gemm import backend as gg
from helpers import announce, dev

pytestmark = pytest.mark.gpu


def _rand(shape, seed):
    g = torch.Generator(device=dev()).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=dev()).to(torch.bfloat16)


@pytest.mark.parametrize("where", ["batch_sizes", "host_batch_sizes"])
def test_types_and_strides(where):
    sizes = [130, 0, 3, 67]
    a, b, dh = _rand((200, 256), 1), _rand((4, 256, 512), 2), _rand((200, 256), 3)
    w4 = gg.quantize_weight_w4(b)
    kinds = {"int64": torch.tensor(sizes), "int32": torch.tensor(sizes, dtype=torch.int32),
             "strided": torch.tensor(sizes).repeat_interleave(2)[::2], "strided int32": torch.tensor(sizes, dtype=torch.int32).repeat_interleave(3)[::3]}
    results = {}
    for kind, host in kinds.items():
        announce(where=where, kind=kind)
        n, more = (host, {}) if where == "batch_sizes" else (torch.tensor(sizes, device=dev()), dict(host_batch_sizes=host))
        h, u = gg.gmm_swiglu_keep(a, b, n, **more)
        da, db = gg.gmm_swiglu_backward(dh, u, a, b, n, **more)
        results[kind] = (gg.gmm(a, b, n, **more), gg.gmm_swiglu(a, b, n, **more), h, u, da, db, gg.gmm_wgrad(a, dh, n, **more),
                         gg.gmm_w4(a, w4, n, **more), gg.gmm_w4_swiglu(a, w4, n, **more))
    for kind, got in results.items():
        for i, (x, want) in enumerate(zip(got, results["int64"])):
            assert torch.equal(x, want), (kind, i)
