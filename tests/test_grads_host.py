"""Refusals of the gradient norm and clipping that answer without a device."""
import ctypes
import math

import numpy as np
import pytest
import torch

from disagmoe_amd import _lib
from disagmoe_amd.ops import grads


def _call(name, entries, *limit, workspace=0x1000, ws_bytes=_lib.GRAD_WORKSPACE_BYTES, norm=0x2000):
    """An entry point on made-up addresses: every case here is refused before anything is launched."""
    table = np.zeros(max(len(entries), 1), dtype=grads._GRAD)
    for i, e in enumerate(entries):
        table[i] = e
    rc = getattr(_lib.load(), name)(table.ctypes.data, len(entries), *limit, norm, workspace, ws_bytes, None)
    return rc, _lib.load().dmoe_last_error().decode()


@pytest.mark.parametrize("name,limit", [("dmoe_grad_norm", ()), ("dmoe_clip_grads", (1.0,))])
def test_refused_descriptions(name, limit):
    ok = (0x10000, 16, _lib.FP32)
    assert _call(name, [ok, (0x20000, 8, _lib.FP8_E4M3)], *limit)[0] == _lib.ERR_DTYPE
    assert _call(name, [ok, (0x20000, -1, _lib.BF16)], *limit)[0] == _lib.ERR_SHAPE
    assert _call(name, [(0, 4, _lib.BF16)], *limit)[0] == _lib.ERR_ARG
    assert _call(name, [(0x20002, 4, _lib.FP32)], *limit)[0] == _lib.ERR_ARG
    assert _call(name, [(0x20001, 4, _lib.BF16)], *limit)[0] == _lib.ERR_ARG
    assert _call(name, [ok], *limit, norm=None)[0] == _lib.ERR_ARG
    assert _call(name, [ok], *limit, workspace=None)[0] == _lib.ERR_WORKSPACE
    assert _call(name, [ok], *limit, workspace=0x1004)[0] == _lib.ERR_WORKSPACE
    assert _call(name, [ok], *limit, ws_bytes=_lib.GRAD_WORKSPACE_BYTES - 1)[0] == _lib.ERR_WORKSPACE


def test_refused_clipping():
    a, b = (0x10000, 16, _lib.FP32), (0x1003c, 8, _lib.BF16)     # b begins in a's last element
    rc, said = _call("dmoe_clip_grads", [a, b], 1.0)
    assert rc == _lib.ERR_ARG and "share memory" in said
    assert _call("dmoe_clip_grads", [a, a], 1.0)[0] == _lib.ERR_ARG
    for limit in (-1.0, math.nan):
        assert _call("dmoe_clip_grads", [a], limit)[0] == _lib.ERR_ARG
        with pytest.raises(ValueError):
            grads.clip_by_global_norm_([torch.zeros(4)], limit)


def test_description_layout_and_host_tensors():
    assert grads._GRAD.itemsize == 24 == ctypes.sizeof(type("G", (ctypes.Structure,), {"_fields_": [
        ("data", ctypes.c_void_p), ("numel", ctypes.c_int64), ("dtype", ctypes.c_int)]}))
    assert float(grads.global_norm([])) == 0 and float(grads.clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0)) == 0
    with pytest.raises(RuntimeError):
        grads.global_norm([torch.ones(3)])


def test_what_counts_as_dense():
    x = torch.zeros(4, 6, 8)
    assert grads._dense(x) and grads._dense(x.transpose(0, 2)) and grads._dense(x.permute(1, 2, 0)) and grads._dense(x[:, :, :, None])
    assert grads._dense(x[1:2]) and grads._dense(x[0, 0, 0])
    assert not grads._dense(x[:, ::2]) and not grads._dense(x[:, :, 1:]) and not grads._dense(torch.zeros(1).expand(5))
