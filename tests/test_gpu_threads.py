"""Two host threads that launch on one stream, as autograd's own thread does beside the caller's: they share that stream's
workspace, and every launch still finds its own partial sums there."""
import threading

import pytest
import torch

from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.models import MoEExperts
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


def test_training_steps_of_two_threads():
    """Two layers, each trained by a thread of its own on the same stream: forward passes of one beside backward passes of the
    other, all of them on the workspace that the stream's layers share."""
    announce(what="training steps of two threads on one stream")
    sizes = torch.tensor([2048, 0, 2048], dtype=torch.int64, device=dev())
    layers = [MoEExperts(256, 1024, 3, init_std=0.05, device=dev()).requires_grad_() for _ in range(2)]
    inputs = [(_rand((4096, 256), i), _rand((4096, 256), i + 7)) for i in range(2)]

    def step(i):
        x = inputs[i][0].clone().requires_grad_()
        y = layers[i].forward_train(4096, x, sizes)
        return (y.detach(), *torch.autograd.grad(y, [x, layers[i].w13_weight, layers[i].w2_weight], inputs[i][1]))

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    wrong, failed = [], []
    stream = torch.cuda.current_stream()

    def many(i):
        try:
            with torch.cuda.stream(stream):
                differ = torch.zeros((), dtype=torch.int64, device=dev())
                for _ in range(60):
                    for got, expected in zip(step(i), want[i]):
                        differ += (got != expected).any()
                if int(differ):
                    wrong.append((i, int(differ)))
        except Exception as e:   # a failure in a thread is the test's
            failed.append(e)

    threads = [threading.Thread(target=many, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and not wrong, (failed, wrong)
