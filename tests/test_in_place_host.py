"""Tensors that a call writes through their addresses count as modified in place, as torch's own operators leave them."""
import contextlib

import pytest
import torch

from disagmoe_amd import _lib
from disagmoe_amd.ops import grads


@pytest.fixture
def no_device(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: type("Stream", (), {"cuda_stream": 0}))
    monkeypatch.setattr(_lib, "call", lambda name, *args: None)
    monkeypatch.setattr(grads, "_table", lambda tensors: (torch.device("cpu"), grads.np.empty(len(tensors), dtype=grads._GRAD)))


def _versions(tensors):
    return [t._version for t in tensors]


def test_clipping_modifies_its_gradients(no_device):
    g = [torch.ones(4), torch.ones(2, 3, dtype=torch.bfloat16), torch.ones(0)]
    before = _versions(g)
    grads.global_norm(g)
    assert _versions(g) == before
    grads.clip_by_global_norm_(g, 1.0)
    assert all(now > was for now, was in zip(_versions(g), before))
    one = torch.ones(3)
    grads.clip_by_global_norm_(one, 1.0)
    assert one._version > 0
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    grads.clip_grad_norm_([p], 1.0)
    assert p.grad._version > 0
    with torch.inference_mode():                      # such a tensor has no version
        grads.clip_by_global_norm_(torch.ones(3), 1.0)


def test_a_clipped_gradient_is_not_used_as_if_it_were_not(no_device):
    """Gradients of gradients, and whatever saved the gradient, notice that it was scaled since."""
    x = torch.ones(4, requires_grad=True)
    (g,) = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    later = g ** 2                                    # saves g
    grads.clip_by_global_norm_([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        later.sum().backward()
