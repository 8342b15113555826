"""Global gradient norm and clipping against 64-bit arithmetic.

Tolerances: the norm is one rounding to fp32 of a 64-bit sum (2^-24 relative, and as much for the square root's own sum);
a scaled gradient is g * coef with coef and product rounded to fp32 (2^-24 each) and one rounding to the gradient's type
(half a step of it, eps / 2 relative; below the type's normal range half of its smallest step)."""
import math

import pytest
import torch

from disagmoe_amd.ops import grads
from helpers import announce, dev

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def _check_scaled(before, after, coef):
    for b, a in zip(before, after):
        fi = torch.finfo(b.dtype)
        want = b.double() * coef
        allowed = want.abs() * (fi.eps / 2 + 3 * 2.0 ** -24) + fi.smallest_normal * fi.eps / 2
        assert bool(((a.double() - want).abs() <= allowed).all()), (b.dtype, b.numel())


def _make(sizes, kinds, seed, std=0.1):
    """Views of one flat bucket for each type, one behind the other: any element alignment."""
    g = torch.Generator(device=dev()).manual_seed(seed)
    out, flat, at = [], {}, {}
    for t in kinds:
        n = sum(s for i, s in enumerate(sizes) if kinds[i % len(kinds)] == t)
        flat[t], at[t] = (torch.randn(n + 1, generator=g, device=dev()) * std).to(t), 1
    for i, s in enumerate(sizes):
        t = kinds[i % len(kinds)]
        out.append(flat[t][at[t]:at[t] + s])
        at[t] += s
    return out, flat


@pytest.mark.parametrize("kinds", [[t] for t in TYPES] + [TYPES], ids=lambda k: "-".join(str(t).split(".")[1] for t in k))
@pytest.mark.parametrize("sizes", [[1], [0, 7, 0], [8], [9, 15, 16, 17, 1, 3], [32768, 32767, 32769, 5], [65536 * 3 + 1, 2, 131072],
                                   list(range(1, 400)), [5_000_003, 1]])
def test_norm_and_clip(sizes, kinds):
    announce(test="clip", sizes=str(sizes[:6]), n=len(sizes), kinds=str(kinds))
    ts, flat = _make(sizes, kinds, seed=len(sizes) + sizes[0])
    guard = {t: b[:1].clone() for t, b in flat.items()}
    want = _norm64(ts)
    n = grads.global_norm(ts)
    assert n.shape == () and n.dtype == torch.float32 and n.is_cuda
    assert abs(float(n) - want) <= want * 2.0 ** -23
    assert torch.equal(n, grads.global_norm(ts))                  # the same bits again
    before = [t.clone() for t in ts]
    # below the limit: nothing is written
    assert torch.equal(grads.clip_by_global_norm_(ts, want * 2 + 1), n)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    limit = want / 3
    assert torch.equal(grads.clip_by_global_norm_(ts, limit), n)
    _check_scaled(before, ts, limit / (want + 1e-6))
    assert all(torch.equal(b[:1], guard[t]) for t, b in flat.items())       # the element in front of the first view


@pytest.mark.parametrize("dtype,value", [(torch.float32, 1e30), (torch.float32, 1e-30), (torch.bfloat16, 1e30), (torch.float16, 6e4),
                                         (torch.float16, 6e-8)])
def test_squares_stay_in_range(dtype, value):
    announce(test="clip_range", dtype=str(dtype), value=value)
    t = torch.full((1000,), value, dtype=dtype, device=dev())
    want = _norm64([t])
    assert abs(float(grads.global_norm([t])) - want) <= want * 2.0 ** -23


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_not_finite(bad):
    announce(test="clip_not_finite", bad=bad)
    ts = [torch.ones(100, dtype=torch.bfloat16, device=dev()), torch.ones(50, device=dev())]
    ts[1][7] = bad
    n = grads.clip_by_global_norm_(ts, 1.0)
    if math.isnan(bad):
        assert math.isnan(float(n)) and all(bool(t.isnan().all()) for t in ts)
    else:
        assert float(n) == math.inf and bool((ts[0] == 0).all()) and bool(ts[1][7].isnan()) and int((ts[1] == 0).sum()) == 49
    z = [torch.zeros(10, device=dev())]
    assert float(grads.clip_by_global_norm_(z, 0.0)) == 0 and bool((z[0] == 0).all())
    one = [torch.ones(4, device=dev())]
    grads.clip_by_global_norm_(one, 0.0)
    assert bool((one[0] == 0).all())
    grads.clip_by_global_norm_([torch.ones(4, device=dev())], math.inf)


def test_against_torch_and_parameters():
    announce(test="clip_against_torch")
    g = torch.Generator().manual_seed(5)
    mine = [torch.nn.Parameter(torch.zeros(s, device=dev())) for s in ((3, 5), (17,), (8, 128, 33), (1,))]
    theirs = [torch.nn.Parameter(torch.zeros_like(p)) for p in mine]
    for a, b in zip(mine[:-1], theirs[:-1]):                    # the last one has no gradient
        a.grad = torch.randn(a.shape, generator=g).to(dev())
        b.grad = a.grad.clone()
    mine[2].grad = mine[2].grad.transpose(0, 2).contiguous().transpose(0, 2)     # dense in another order
    n, m = grads.clip_grad_norm_(mine, 1.5), torch.nn.utils.clip_grad_norm_(theirs, 1.5)
    assert abs(float(n) - float(m)) <= float(m) * 1e-5
    for a, b in zip(mine[:-1], theirs[:-1]):
        assert torch.allclose(a.grad, b.grad, rtol=1e-5, atol=0)
    assert mine[-1].grad is None
    p = mine[0]
    assert torch.equal(grads.clip_grad_norm_(p, 1e9), grads.global_norm(p.grad))


def test_refusals():
    announce(test="clip_refusals")
    x = torch.ones(8, 8, device=dev())
    with pytest.raises(ValueError):
        grads.global_norm([x[:, ::2]])
    with pytest.raises(ValueError):
        grads.clip_by_global_norm_([x, torch.zeros(1, device=dev()).expand(4)], 1.0)
    with pytest.raises(TypeError):
        grads.global_norm([x.double()])
    with pytest.raises(RuntimeError):
        grads.global_norm([x, x.cpu()])
    with pytest.raises(RuntimeError, match="share memory"):
        grads.clip_by_global_norm_([x, x[2]], 1.0)
    assert bool((x == 1).all())
    assert abs(float(grads.global_norm([x, x])) - math.sqrt(128)) < 1e-5       # reading twice is fine


def test_graph_replays_and_streams():
    announce(test="clip_graph")
    a = [torch.zeros(70001, dtype=torch.bfloat16, device=dev()), torch.zeros(301, device=dev())]
    b = [torch.zeros(50003, device=dev())]
    graphs = []
    for ts in (a, b):                       # two graphs on the same device: each with a workspace of its own
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            grads.clip_by_global_norm_(ts, 1.0)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            n = grads.clip_by_global_norm_(ts, 1.0)
        graphs.append((g, n, ts))
    s = torch.cuda.Stream()
    for rep in range(4):
        gen = torch.Generator().manual_seed(rep)
        want = []
        for g, n, ts in graphs:
            for t in ts:
                t.copy_(torch.randn(t.shape, generator=gen))
            eager = [t.clone() for t in ts]
            want.append((grads.clip_by_global_norm_(eager, 1.0), eager))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for (g, n, ts), (m, eager) in zip(graphs, want):
            assert torch.equal(n, m) and all(torch.equal(x, y) for x, y in zip(ts, eager))


def test_a_tensor_past_32_bits():
    announce(test="clip_large")
    n = (1 << 31) + 4099                                  # bf16: more than 4 GiB
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device=dev())
    g[n - 1] = 40000.0
    want = (0.25 * (n - 1) + float(g[n - 1]) ** 2) ** 0.5
    assert abs(float(grads.global_norm(g)) - want) <= 2.0 ** -23 * want
    last = float(g[n - 1])
    grads.clip_by_global_norm_(g, want / 4)
    assert bool((g[:n - 1] == 0.125).all()) and abs(float(g[n - 1]) - last / 4) <= 2.0 ** -8 * last
    del g
    torch.cuda.empty_cache()
