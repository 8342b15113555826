"""Refusals of the gradient entry points that answer without a device, and their names."""
import pytest
import torch

from disagmoe_amd import _lib
from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.grouped_gemm import ops


def test_host_side_argument_errors():
    lib = _lib.load()
    p = 0x100000   # never touched: every call is refused before a launch

    def wgrad(a=p, dc=p + 0x1000, db=p + 0x2000, bs=p, rows=16, E=4, K=64, N=64, dtype=_lib.BF16):
        return lib.dmoe_gmm_wgrad(a, dc, db, bs, rows, E, K, N, dtype, None, None, 0, None, None)

    assert wgrad(dtype=_lib.FP16) == _lib.ERR_DTYPE and wgrad(dtype=_lib.FP8_E4M3) == _lib.ERR_DTYPE
    for bad in (dict(K=60), dict(N=12), dict(K=0), dict(E=0), dict(E=1025), dict(rows=-1), dict(rows=1 << 31)):
        assert wgrad(**bad) == _lib.ERR_SHAPE, bad
    for bad in (dict(a=None), dict(dc=None), dict(db=None), dict(bs=None), dict(db=p), dict(db=p + 0x1000), dict(a=p + 8), dict(dc=p + 0x1002),
                dict(db=p + 0x2004)):
        assert wgrad(**bad) == _lib.ERR_ARG, bad

    def keep(a=p, b=p, h=p + 0x1000, u=p + 0x2000, bs=p, rows=16, K=64, I=64, dtype=_lib.BF16):
        return lib.dmoe_gmm_swiglu_keep(a, b, h, u, bs, rows, 4, K, I, 0, dtype, None, None, 0, None, None)

    assert keep(dtype=_lib.FP16) == _lib.ERR_DTYPE
    assert keep(K=60) == _lib.ERR_SHAPE and keep(I=12) == _lib.ERR_SHAPE
    for bad in (dict(a=None), dict(b=None), dict(h=None), dict(u=None), dict(bs=None), dict(a=p + 2), dict(u=p + 0x2008)):
        assert keep(**bad) == _lib.ERR_ARG, bad
    assert keep(rows=0) == 0

    def back(dh=p, u=p + 0x1000, a=p + 0x2000, b=p + 0x3000, du=p + 0x4000, da=p + 0x5000, db=p + 0x6000, bs=p, rows=16, K=64, I=64,
             dtype=_lib.BF16):
        return lib.dmoe_gmm_swiglu_backward(dh, u, a, b, du, da, db, bs, rows, 4, K, I, 0, dtype, None, None, 0, None, None)

    assert back(dtype=_lib.FP16) == _lib.ERR_DTYPE
    assert back(K=60) == _lib.ERR_SHAPE and back(I=12) == _lib.ERR_SHAPE and back(I=1 << 21) == _lib.ERR_SHAPE
    for bad in (dict(dh=None), dict(u=None), dict(a=None), dict(b=None), dict(du=None), dict(bs=None), dict(du=p), dict(du=p + 0x1000),
                dict(da=p), dict(da=p + 0x2000), dict(dh=p + 8), dict(db=p + 0x6002)):
        assert back(**bad) == _lib.ERR_ARG, bad
    assert back(da=None, db=None, rows=0) == 0

    assert lib.dmoe_zero_rows_behind(None, p, 4, 4, 64, _lib.BF16, None) == _lib.ERR_ARG
    assert lib.dmoe_zero_rows_behind(p, p, 4, 4, 60, _lib.BF16, None) == _lib.ERR_SHAPE
    assert lib.dmoe_zero_rows_behind(p, p, 4, 4, 64, _lib.FP32, None) == _lib.ERR_DTYPE
    assert lib.dmoe_zero_rows_behind(p, p, 0, 4, 64, _lib.BF16, None) == 0


def test_upstream_name():
    import grouped_gemm.ops
    assert grouped_gemm.ops is ops


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device behaviour")
def test_no_cpu_fallback():
    a, b = torch.zeros(4, 8, dtype=torch.bfloat16, requires_grad=True), torch.zeros(1, 8, 16, dtype=torch.bfloat16)
    n = torch.tensor([4])
    for call in (lambda: ops.gmm(a, b, n), lambda: ops.gmm_swiglu(a, b, n), lambda: gg.gmm_swiglu_keep(a, b, n),
                 lambda: gg.gmm_wgrad(a, a, n)):
        with pytest.raises(RuntimeError):
            call()
