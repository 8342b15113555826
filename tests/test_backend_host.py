"""What the wrappers of the grouped products do on the host around a call into the library, with the device left out."""
import contextlib
import threading

import pytest
import torch

from disagmoe_amd.grouped_gemm import backend as gg


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
