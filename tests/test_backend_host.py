"""What the wrappers of the grouped products do on the host around a call into the library, with the device left out."""
import contextlib
import threading
import weakref

import pytest
import torch
from torch.autograd import forward_ad

from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.grouped_gemm import ops
from disagmoe_amd.ops import memory


def test_threads_that_first_launch_on_one_stream_share_its_pair(monkeypatch):
    both = threading.Barrier(2, timeout=10)

    def block(device):
        with contextlib.suppress(threading.BrokenBarrierError):
            both.wait()                       # both threads have found nothing
        return torch.zeros(8, dtype=torch.uint8)

    monkeypatch.setattr(gg, "_DEFAULTS", {})
    monkeypatch.setattr(gg, "_new_state_block", block)
    monkeypatch.setattr(gg, "workspace_bytes", lambda: 8)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    pairs = []
    threads = [threading.Thread(target=lambda: pairs.append(gg._default_pair(torch.device("cpu"), 0))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(pairs) == 2 and pairs[0] is pairs[1] is gg._default_pair(torch.device("cpu"), 0)


class _OnDevice(torch.Tensor):
    """A host tensor that says it is on the device: the wrappers then go as far as the call."""
    is_cuda = True


def _fake_device(monkeypatch, called):
    """Replaces what needs a device; ``called(name, args)`` stands for the library."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(gg, "_stream", lambda device: 0)
    monkeypatch.setattr(gg, "_default_pair", lambda device, stream: (torch.zeros(8, dtype=torch.uint8),) * 2)
    monkeypatch.setattr(gg._lib, "call", lambda name, *args: called(name, args))


def _on_device(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=torch.float32).to(dtype).as_subclass(_OnDevice)


SIZES = [3, 0, 5]


def _products():
    a, b, h = _on_device(8, 32), _on_device(3, 32, 64), _on_device(8, 64)
    q, bq = _on_device(8, 32, dtype=torch.float8_e4m3fn), _on_device(3, 64, 32, dtype=torch.float8_e4m3fn)
    sa, sb = _on_device(8, dtype=torch.float32), _on_device(3, 64, dtype=torch.float32)
    u, dh = _on_device(8, 64, dtype=torch.float32), _on_device(8, 32)
    rows = _on_device(8, dtype=torch.int32)
    return {
        "gmm": lambda n: gg.gmm(a, b, n),
        "gmm_swiglu": lambda n: gg.gmm_swiglu(a, b, n),
        "gmm_swiglu_rows": lambda n: gg.gmm_swiglu_rows(a, rows, b, n),
        "gmm_swiglu_keep": lambda n: gg.gmm_swiglu_keep(a, b, n),
        "gmm_swiglu_backward": lambda n: gg.gmm_swiglu_backward(dh, u, a, b, n),
        "gmm_wgrad": lambda n: gg.gmm_wgrad(a, h, n),
        "gmm_fp8": lambda n: gg.gmm_fp8(q, sa, bq, sb, n),
        "gmm_fp8_swiglu": lambda n: gg.gmm_fp8_swiglu(q, sa, bq, sb, n),
    }


@pytest.mark.parametrize("name", list(_products()))
@pytest.mark.parametrize("kind", ["int32", "strided", "int64"])
def test_host_sizes_live_until_the_call_has_read_them(monkeypatch, name, kind):
    """Sizes that have to be converted are a tensor of the wrapper's own: the library reads it, so it is there until then."""
    sizes = {"int32": lambda: torch.tensor(SIZES, dtype=torch.int32), "int64": lambda: torch.tensor(SIZES),
             "strided": lambda: torch.tensor(SIZES).repeat_interleave(2)[::2]}[kind]()
    refs, reads = [], []
    convert = gg._host_sizes

    def host_sizes(*args):
        host = convert(*args)
        refs.append((weakref.ref(host), host.data_ptr()))
        return host

    def called(name, args):
        ref, address = refs[-1]
        assert args[-2] == address
        reads.append(ref() is not None and ref().tolist() == SIZES)

    monkeypatch.setattr(gg, "_host_sizes", host_sizes)
    _fake_device(monkeypatch, called)
    _products()[name](sizes)
    assert reads == [True]


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(monkeypatch, which, grad):
    """The products have no forward-mode derivative: an operand with a tangent is refused, not taken without it."""
    _fake_device(monkeypatch, lambda name, args: None)
    monkeypatch.setattr(gg, "_check_operands", lambda a, b, dtype: a.device)
    operands = [torch.zeros(8, 32, dtype=torch.bfloat16), torch.zeros(3, 32, 64, dtype=torch.bfloat16)]
    n = torch.tensor(SIZES)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        assert ops.gmm_swiglu(*operands, n).shape == (8, 32)          # nothing has a tangent
        operands[which] = forward_ad.make_dual(operands[which], torch.ones_like(operands[which]))
        for product in (ops.gmm, ops.gmm_swiglu):
            with pytest.raises(NotImplementedError):
                product(*operands, n)


def _written():
    """The calls that write into a tensor of the caller's, by the tensor."""
    a, b = _on_device(8, 32), _on_device(3, 32, 64)
    q, bq = _on_device(8, 32, dtype=torch.float8_e4m3fn), _on_device(3, 64, 32, dtype=torch.float8_e4m3fn)
    sa, sb = _on_device(8, dtype=torch.float32), _on_device(3, 64, dtype=torch.float32)
    rows, ptrs, n = _on_device(8, dtype=torch.int32), _on_device(8, dtype=torch.int64), torch.tensor(SIZES)
    w = gg.pack_w4(torch.zeros(3, 64, 32, dtype=torch.uint8), torch.ones(3, 64, 1), None, 32)
    return {
        "gmm": (64, lambda c: gg.gmm(a, b, n, c=c)),
        "gmm_swiglu": (32, lambda c: gg.gmm_swiglu(a, b, n, c=c)),
        "gmm_swiglu_rows": (32, lambda c: gg.gmm_swiglu_rows(a, rows, b, n, c=c)),
        "gmm_fp8": (64, lambda c: gg.gmm_fp8(q, sa, bq, sb, n, c=c)),
        "gmm_fp8_swiglu": (32, lambda c: gg.gmm_fp8_swiglu(q, sa, bq, sb, n, c=c)),
        "gmm_w4": (64, lambda c: gg.gmm_w4(a, w, n, c=c)),
        "gmm_w4_swiglu": (32, lambda c: gg.gmm_w4_swiglu(a, w, n, c=c)),
        "zero_rows_behind": (64, lambda c: gg.zero_rows_behind(c, n)),
        "gather_row_ptrs": (64, lambda c: memory.gather_row_ptrs(ptrs, 64, torch.bfloat16, out=c)),
    }


@pytest.mark.parametrize("name", list(_written()))
def test_a_result_in_the_callers_tensor_modifies_it(monkeypatch, name):
    """What autograd has saved of that tensor is not used as if it still held the old values."""
    _fake_device(monkeypatch, lambda name, args: None)
    monkeypatch.setattr(gg, "_check_w4", lambda w: w.codes.shape[0])
    monkeypatch.setattr(memory, "_stream", lambda device: 0)
    columns, call = _written()[name]
    c = _on_device(8, columns)
    x = torch.ones(8, columns, dtype=torch.bfloat16, requires_grad=True)
    y = x * c                                          # saves c
    assert call(c) is c
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():                       # a tensor without a version, and one with
        call(_on_device(8, columns))
        call(c)
