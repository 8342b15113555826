"""Two host threads that launch on one stream, as autograd's own thread does beside the caller's: they share that stream's
workspace, and every launch still finds its own partial sums there."""
import threading

import pytest
import torch

from disagmoe_amd.grouped_gemm import backend as gg
from helpers import announce, dev

pytestmark = pytest.mark.gpu


def _rand(shape, seed):
    g = torch.Generator(device=dev()).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=dev()).to(torch.bfloat16)


def test_cut_weight_gradients_beside_cut_products():
    """A weight gradient of few tiles leaves the pieces of its contractions in the workspace in one launch and adds them up
    in the next; another thread's launches leave sums there too."""
    sizes = torch.tensor([4096, 4096], dtype=torch.int64, device=dev())
    a, dc = _rand((8192, 512), 1), _rand((8192, 1024), 2)
    few = torch.tensor([64, 64], dtype=torch.int64, device=dev())
    x, w = _rand((128, 8192), 3), _rand((2, 8192, 512), 4)
    assert gg.launch_plan(128, 2, 8192, 512, workspace_bytes=gg.workspace_bytes(), batch_sizes=[64, 64])["cut_tiles"] > 0
    announce(what="weight gradients and products of two threads on one stream")
    want_db, want_c = gg.gmm_wgrad(a, dc, sizes), gg.gmm(x, w, few)
    torch.cuda.synchronize()
    wrong, failed = [], []
    stream = torch.cuda.current_stream()

    def many(what, call, want):
        try:
            with torch.cuda.stream(stream):
                differ = torch.zeros((), dtype=torch.int64, device=dev())
                for _ in range(200):
                    differ += (call() != want).any()
                if int(differ):
                    wrong.append((what, int(differ)))
        except Exception as e:   # a failure in a thread is the test's
            failed.append(e)

    threads = [threading.Thread(target=many, args=("db", lambda: gg.gmm_wgrad(a, dc, sizes), want_db)),
               threading.Thread(target=many, args=("c", lambda: gg.gmm(x, w, few), want_c))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and not wrong, (failed, wrong)
