"""Expert modules without a device: names, and what the forms without a gradient say about it."""
import warnings

import pytest
import torch

from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.models import experts


def test_names():
    from disagmoe_amd import models
    assert {"MoEExperts", "MoEExpertsSerial", "MoEExpertsFP8", "MoEExpertsW4"} <= set(models.__all__)
    assert models.MoEExpertsW4 is experts.MoEExpertsW4


@pytest.fixture
def layer(monkeypatch):
    monkeypatch.setattr(experts._GemmState, "_gemm_state", lambda self: {})
    monkeypatch.setattr(experts._GemmState, "__del__", lambda self: None)
    monkeypatch.setattr(gg, "gmm_swiglu", lambda a, b, n, **kw: torch.zeros(a.shape[0], b.shape[2] // 2))
    monkeypatch.setattr(gg, "gmm_swiglu_rows", lambda x, r, b, n, **kw: torch.zeros(r.numel(), b.shape[2] // 2))
    monkeypatch.setattr(gg, "gmm", lambda a, b, n, **kw: torch.zeros(a.shape[0], b.shape[2]))
    m = experts.MoEExperts.__new__(experts.MoEExperts)
    torch.nn.Module.__init__(m)
    m.w13_weight = torch.nn.Parameter(torch.zeros(2, 8, 32), requires_grad=False)
    m.w2_weight = torch.nn.Parameter(torch.zeros(2, 16, 8), requires_grad=False)
    m.enable_cache, m.gmm = False, gg.gmm
    return m


def test_forms_without_a_gradient_say_so(layer):
    x, n, rows = torch.zeros(4, 8), torch.tensor([1, 3]), torch.arange(4, dtype=torch.int32)
    forms = (lambda v: layer.forward(4, v, n), lambda v: layer.forward_rows(v, rows, n))

    def both(v, expect):
        for form in forms:
            with warnings.catch_warnings(record=True) as said:
                warnings.simplefilter("always")
                assert not form(v).requires_grad
            assert [str(w.message).count("forward_train") for w in said] == ([1] if expect else [])
            assert all(w.filename == __file__ for w in said)

    both(x, False)
    both(x.clone().requires_grad_(), True)
    layer.w2_weight.requires_grad_()
    both(x, True)
    with torch.no_grad():
        both(x, False)
    with torch.inference_mode():
        both(x, False)
    layer.w2_weight.requires_grad_(False)
    layer.w13_weight.requires_grad_()
    both(x, True)


@pytest.mark.parametrize("kind", ["MoEExpertsW4", "MoEExpertsFP8"])
def test_quantised_experts_say_so_too(monkeypatch, kind):
    """Frozen experts of few bits in the middle of something that is trained: the rows' gradient ends there."""
    monkeypatch.setattr(experts._GemmState, "_gemm_state", lambda self: {})
    monkeypatch.setattr(experts._GemmState, "__del__", lambda self: None)
    for name in ("gmm_w4", "gmm_w4_swiglu"):
        monkeypatch.setattr(gg, name, lambda a, w, n, **kw: a.detach())
    monkeypatch.setattr(gg, "quantize_rows", lambda x: (x.detach(), torch.ones(4)))
    for name in ("gmm_fp8", "gmm_fp8_swiglu"):
        monkeypatch.setattr(gg, name, lambda a, s, b, t, n, **kw: a)
    m = getattr(experts, kind).__new__(getattr(experts, kind))
    torch.nn.Module.__init__(m)
    m.hidden_size = m.intermediate_size = 8
    m._group13 = m._group2 = 32
    for w in ("w13", "w2"):
        for t in ("codes", "scales", "zeros", "q", "scale"):
            m.register_buffer(f"{w}_{t}", torch.zeros(1))
    x, n = torch.zeros(4, 8), torch.tensor([1, 3])
    for v, expect in ((x, 0), (x.clone().requires_grad_(), 1)):
        with warnings.catch_warnings(record=True) as said:
            warnings.simplefilter("always")
            m.forward(4, v, n)
        assert len(said) == expect and all(w.filename == __file__ and kind in str(w.message) for w in said)
