"""Global norm of the experts' gradients and clipping to a largest norm, computed by
the HIP kernels of libdmoe_hip.so on the current stream of the gradients' device; no
counterpart in the reference, which trains nothing.  Nothing here synchronises: the
norm comes back as a 0-dimensional fp32 tensor on the device.
"""
from __future__ import annotations

from typing import Iterable, List, Union

import numpy as np
import torch

from .. import _lib

_DTYPES = {torch.float32: _lib.FP32, torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
#: dmoe_grad of include/dmoe.h
_GRAD = np.dtype({"names": ["data", "numel", "dtype"], "formats": ["<u8", "<i8", "<i4"], "offsets": [0, 8, 16], "itemsize": 24})


def _dense(g: torch.Tensor) -> bool:
    """Whether the elements of ``g`` fill its memory without a hole, in whatever order."""
    expected = 1
    for stride, size in sorted((st, n) for n, st in zip(g.shape, g.stride()) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _table(grads: List[torch.Tensor]):
    """(device, host array of dmoe_grad) of the gradients."""
    device = grads[0].device
    if device.type != "cuda":
        raise RuntimeError("gradient norms need device tensors; disagmoe_amd has no CPU fallback")
    index = device.index
    if any(i != index for i in map(torch.Tensor.get_device, grads)):
        other = next(g.device for g in grads if g.device != device)
        if other.type != "cuda":
            raise RuntimeError("gradient norms need device tensors; disagmoe_amd has no CPU fallback")
        raise ValueError(f"gradients on {device} and {other}: one call handles one device")
    if not all(map(torch.Tensor.is_contiguous, grads)):
        for g in grads:
            if g.layout is not torch.strided:
                raise TypeError(f"gradients must be strided tensors, got {g.layout}")
            if g.numel() and not _dense(g):
                raise ValueError(f"a gradient of shape {tuple(g.shape)} with strides {g.stride()} does not fill its memory")
    try:
        kinds = [_DTYPES[g.dtype] for g in grads]
    except KeyError as e:
        raise TypeError(f"gradients must be fp32, bf16 or fp16, got {e.args[0]}") from None
    table = np.empty(len(grads), dtype=_GRAD)
    table["data"] = list(map(torch.Tensor.data_ptr, grads))
    table["numel"] = list(map(torch.Tensor.numel, grads))
    table["dtype"] = kinds
    return device, table


def _run(name: str, grads: List[torch.Tensor], *limit) -> torch.Tensor:
    if not grads:
        return torch.zeros(())
    device, table = _table(grads)
    with torch.cuda.device(device):
        norm = torch.empty((), dtype=torch.float32, device=device)
        # of this call alone: a graph that records it keeps the memory to itself
        workspace = torch.empty(_lib.GRAD_WORKSPACE_BYTES, dtype=torch.uint8, device=device)
        _lib.call(name, table.ctypes.data, len(table), *limit, norm.data_ptr(), workspace.data_ptr(),
                  _lib.GRAD_WORKSPACE_BYTES, torch.cuda.current_stream(device).cuda_stream)
    return norm


@torch.no_grad()
def global_norm(grads: Union[torch.Tensor, Iterable[torch.Tensor]]) -> torch.Tensor:
    """``sqrt(sum of g^2)`` over every element of all gradients (fp32, bf16, fp16, mixed;
    any sizes; dense, on one device), summed in 64 bits in a fixed order.  A 0-dimensional
    fp32 device tensor; an empty list has norm 0 (on the host)."""
    return _run("dmoe_grad_norm", [grads] if torch.is_tensor(grads) else list(grads))


@torch.no_grad()
def clip_by_global_norm_(grads: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float) -> torch.Tensor:
    """Scales all gradients in place by ``min(1, max_norm / (norm + 1e-6))`` and returns
    their :func:`global_norm` before that.  Gradients whose norm is below the limit are not
    written (to autograd they are modified in place all the same: the host does not wait for the
    norm).  A norm that is infinite or NaN is treated as torch.nn.utils.clip_grad_norm_ treats it:
    a factor of zero, or NaN.  No two gradients may share memory."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    grads = [grads] if torch.is_tensor(grads) else list(grads)
    norm = _run("dmoe_clip_grads", grads, max_norm)
    # written through their addresses, which autograd does not see: what saved one of them has to notice
    torch.autograd.graph.increment_version(grads)
    return norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float) -> torch.Tensor:
    """:func:`clip_by_global_norm_` on the ``.grad`` of the parameters that have one."""
    parameters = [parameters] if torch.is_tensor(parameters) else parameters
    return clip_by_global_norm_([p.grad for p in parameters if p.grad is not None], max_norm)
