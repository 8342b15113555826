"""What the wrappers of the grouped products do on the host around a call into the library, with the device left out."""
import contextlib
import threading
import weakref

import pytest
import torch
from torch.autograd import forward_ad

from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.grouped_gemm import ops


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
    monkeypatch.setattr(gg, "zero_rows_behind", lambda c, sizes: c)
    operands = [torch.zeros(8, 32, dtype=torch.bfloat16), torch.zeros(3, 32, 64, dtype=torch.bfloat16)]
    n = torch.tensor(SIZES)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        assert ops.gmm_swiglu(*operands, n).shape == (8, 32)          # nothing has a tangent
        operands[which] = forward_ad.make_dual(operands[which], torch.ones_like(operands[which]))
        for product in (ops.gmm, ops.gmm_swiglu):
            with pytest.raises(NotImplementedError):
                product(*operands, n)
