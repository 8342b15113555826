"""The grouped products under autograd: :func:`gmm` and the gated block :func:`gmm_swiglu`
with the operands of ``backend`` and gradients of both ``a`` and ``b``.

Gradients are bf16 like the operands, each sum taken in fp32 and rounded once.  Rows past
``sum(batch_sizes)`` belong to no expert: they come out as zeros and their gradient is zero;
an expert without rows has a zero gradient.  ``workspace`` and ``arguments_ptr``
(``backend.get_arguments``) serve the forward and the backward launches, which follow each other
on the stream the forward ran on; a step that is captured into a graph has to bring them, as
``backend.gmm`` does.  The gradients themselves are not differentiable, and there is no
forward-mode derivative: both are refused.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import backend


def _prepare(a: torch.Tensor, batch_sizes: torch.Tensor, host_batch_sizes: Optional[torch.Tensor], workspace, arguments_ptr):
    """(sizes on the device, the trailing arguments of the forward and the backward launches, what those need alive): made
    once, because the engine runs the backward pass in a thread of its own where a statement costs several times what it
    costs here."""
    host = backend._host_sizes(batch_sizes, host_batch_sizes)
    state_args = backend._state_args(a.device, workspace, arguments_ptr, backend._stream(a.device), host)
    return backend._sizes_on_device(batch_sizes, a.device), state_args, (host, workspace, backend._STATE_BLOCKS.get(arguments_ptr))


def _check_capture(ctx) -> None:
    if ctx.alive[2] is None and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a backward pass recorded into a graph needs a state block of its own: pass the arguments_ptr of "
                           "get_arguments() (and a workspace) to the forward call")


def _check_aligned(a: torch.Tensor, b: torch.Tensor) -> None:
    if (a.data_ptr() | b.data_ptr()) & 15:
        raise ValueError("a and b must be 16-byte aligned")


def _has_tangent(x: torch.Tensor) -> bool:
    """Whether ``x`` carries a forward-mode derivative (which torch refuses of the functions below)."""
    return forward_ad.unpack_dual(x).tangent is not None


def _gradient(dc: torch.Tensor) -> torch.Tensor:
    """The gradient as the kernels read it, whatever view of other memory it arrived as."""
    dc = dc.contiguous()
    return dc.clone() if dc.data_ptr() & 15 else dc


def _once(backward):
    """``once_differentiable``, whose wrapper is left out where no gradient of the gradient can be asked for."""
    wrapped = once_differentiable(backward)

    def run(ctx, dc):
        return (wrapped if torch.is_grad_enabled() else backward)(ctx, dc)
    return run


class _Gmm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, sizes, trans_b, state_args, alive):
        ctx.save_for_backward(a, b, sizes)
        ctx.trans_b, ctx.state_args, ctx.alive = trans_b, state_args, alive
        return backend._gmm_zeroed(a, b, sizes, trans_b, state_args)

    @staticmethod
    @_once
    def backward(ctx, dc):
        _check_capture(ctx)
        a, b, sizes = ctx.saved_tensors
        return (*backend._gmm_backward(_gradient(dc), a, b, sizes, ctx.trans_b, ctx.needs_input_grad[0], ctx.needs_input_grad[1],
                                       ctx.state_args), None, None, None, None)


class _GmmSwiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, sizes, trans_b, state_args, alive):
        h, u = backend._swiglu_keep(a, b, sizes, trans_b, state_args)
        ctx.save_for_backward(a, b, sizes, u)
        ctx.trans_b, ctx.state_args, ctx.alive = trans_b, state_args, alive
        return h

    @staticmethod
    @_once
    def backward(ctx, dh):
        _check_capture(ctx)
        a, b, sizes, u = ctx.saved_tensors
        return (*backend._swiglu_backward(_gradient(dh), u, a, b, sizes, ctx.trans_b, ctx.needs_input_grad[0], ctx.needs_input_grad[1],
                                          ctx.state_args), None, None, None, None)


def gmm(a: torch.Tensor, b: torch.Tensor, batch_sizes: torch.Tensor, trans_b: bool = False,
        workspace: Optional[torch.Tensor] = None, arguments_ptr: Optional[int] = None,
        host_batch_sizes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Differentiable ``backend.gmm``: ``c[o_e:o_e+n_e] = a[o_e:o_e+n_e] @ b[e]`` (``b[e].T`` with
    ``trans_b``), bf16 in and out."""
    backend._check_product(a, b, batch_sizes, trans_b)
    _check_aligned(a, b)
    sizes, state_args, alive = _prepare(a, batch_sizes, host_batch_sizes, workspace, arguments_ptr)
    return _Gmm.apply(a, b, sizes, trans_b, state_args, alive)


def gmm_swiglu(a: torch.Tensor, b: torch.Tensor, batch_sizes: torch.Tensor, trans_b: bool = False,
               workspace: Optional[torch.Tensor] = None, arguments_ptr: Optional[int] = None,
               host_batch_sizes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Differentiable ``backend.gmm_swiglu``: ``silu(u[:, :I]) * u[:, I:]`` for ``u = gmm(a, b)``,
    ``b [E, K, 2I]`` (``[E, 2I, K]`` with ``trans_b``).  Keeps ``u`` in fp32 (8 bytes per element of
    the result) for the backward pass; without a gradient to come it is ``backend.gmm_swiglu``."""
    backend._check_block(a, b, batch_sizes, trans_b)
    _check_aligned(a, b)
    if not (torch.is_grad_enabled() and (a.requires_grad or b.requires_grad) or _has_tangent(a) or _has_tangent(b)):
        sizes, host = backend._sizes_on_device(batch_sizes, a.device), backend._host_sizes(batch_sizes, host_batch_sizes)
        return backend._zero_rows_behind(backend.gmm_swiglu(a, b, sizes, trans_b=trans_b, workspace=workspace,
                                                            arguments_ptr=arguments_ptr, host_batch_sizes=host), sizes)
    sizes, state_args, alive = _prepare(a, batch_sizes, host_batch_sizes, workspace, arguments_ptr)
    return _GmmSwiglu.apply(a, b, sizes, trans_b, state_args, alive)
