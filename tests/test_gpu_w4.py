"""4-bit products against the definition in 64 bits.

Tolerances, element by element.  A bf16 result is off by half a step, 2^-8 of its value (``HALF``).  The one kernel keeps the
weights as they are; it adds (16 + q) x over a group of G in fp32 (at most 31 |x| a term, n terms off by at most n 2^-24 of
their magnitudes, counted twice for a matrix core that adds several terms at a time: ``ACC``), takes (16 + z) times the
group's sum of x off, and adds the groups: ACC (G + 8) 47 sum s |x|, and ACC (K / G + 16) times the sum of the groups'
magnitudes.  The form for many rows rounds each weight to fp16 (2^-11 of it at most), after scaling a column by a power of
two below its largest scale and a row by one below its largest value, so that what is tiny beside those loses what lies
below 2^-24 of them: 2^-11 |w| |x| + 2^-24 (16 max s |x| + |w| max |x|) under the sum, and K products added in fp32."""
import pytest
import torch

from disagmoe_amd import _lib
from disagmoe_amd.expert_layer import expert_layer_forward
from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.models.experts import MoEExpertsW4
from helpers import announce, dev, ragged_sizes
from test_w4_host import unpack

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8
ACC = 2 * 2.0 ** -24


def _rand(shape, seed, std=1.0):
    g = torch.Generator(device=dev()).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev()) * std).to(torch.bfloat16)


def _weight(E, N, K, group, zeros, seed):
    g = torch.Generator(device=dev()).manual_seed(seed)
    groups = -(-K // group)
    q = torch.randint(0, 16, (E, N, K), generator=g, device=dev(), dtype=torch.uint8)
    s = (torch.rand(E, N, groups, generator=g, device=dev()) * 0.02 + 0.005).to(torch.bfloat16)
    z = torch.randint(0, 16, (E, N, groups), generator=g, device=dev(), dtype=torch.uint8) if zeros else None
    zs = torch.full_like(s, 8).double() if z is None else z.double()
    spread = lambda v: v.double().repeat_interleave(group, 2)[:, :, :K]
    return gg.pack_w4(q, s, z, group), (q.double() - spread(zs)) * spread(s), spread(s)


def _spans(sizes):
    o = 0
    for e, n in enumerate(sizes.tolist()):
        yield e, slice(o, o + n)
        o += n


def _check(got, x, w, s, sizes, group, swiglu, wide):
    for e, at in _spans(sizes):
        a = x[at].double()
        want = a @ w[e].t()
        mag = a.abs() @ w[e].abs().t()
        off = ACC * (group + 8) * 47 * (a.abs() @ s[e].t()) + ACC * (a.shape[1] / group + 16) * mag
        if wide:
            off = (2.0 ** -11 + ACC * (a.shape[1] + 4)) * mag
            off = off + 2.0 ** -24 * (a.abs().sum(1, keepdim=True) * 16 * s[e].max(1).values + a.abs().max(1, keepdim=True).values * w[e].abs().sum(1))
        if swiglu:
            I = w.shape[1] // 2
            g, p = want[:, :I], want[:, I:]
            sig = torch.sigmoid(g)
            # (second-order terms: 5 % of the first-order ones)
            off = 1.05 * ((p * sig * (1 + g * (1 - sig))).abs() * off[:, :I] + (g * sig).abs() * off[:, I:] + off[:, :I] * off[:, I:]) + 1e-6 * (g * p).abs()
            want = g * sig * p
        err = (got[at].double() - want).abs()
        bad = ~(err <= off + HALF * (want.abs() + off) + 1e-37)
        assert not bool(bad.any()), (e, int(bad.sum()), float(err[bad][0]), float(off[bad][0]), float(want[bad][0]))
        if not swiglu and want.numel():
            # every element's rounding is at most HALF of it, and so is the 2-norm's; the sums add a tenth at most here
            assert float(err.norm()) <= 1.1 * HALF * float(want.norm()) + 1e-30


SIZES = [[1], [0, 2, 0, 1], [15, 16, 17], [5, 0, 33, 64, 0, 65, 1], [3] * 40, [190, 2, 70]]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N", [(8, 16), (40, 48), (128, 272), (264, 128), (1408, 80), (2184, 144)])
def test_small_sizes(K, N, group, zeros):
    for sizes in SIZES:
        announce(test="w4", sizes=str(sizes[:8]), K=K, N=N, group=group, zeros=zeros)
        sizes = torch.tensor(sizes)
        E, R = len(sizes), int(sizes.sum())
        w, ref, s = _weight(E, N, K, group, zeros, seed=K + N)
        x = _rand((R, K), R)
        c = gg.gmm_w4(x, w, sizes)
        assert c.shape == (R, N) and c.dtype == torch.bfloat16
        _check(c, x, ref, s, sizes, group, False, False)
        assert torch.equal(c, gg.gmm_w4(x, w, sizes.to(dev()), host_batch_sizes=sizes))
        h = gg.gmm_w4_swiglu(x, w, sizes.to(dev()))
        assert h.shape == (R, N // 2)
        _check(h, x, ref, s, sizes, group, True, False)


@pytest.mark.parametrize("rows_e", [1, 20, 50, 100])
@pytest.mark.parametrize("swiglu", [False, True])
def test_sizes_alone_on_the_device(rows_e, swiglu):
    announce(test="w4_device_sizes", rows_e=rows_e, swiglu=swiglu)
    # every row tile height, planned from rows / E alone, skewed and with empty experts
    E, K, N, group = 8, 520, 208, 64
    sizes = ragged_sizes(E, E * rows_e, seed=rows_e, empty_every=4)
    w, ref, s = _weight(E, N, K, group, True, seed=rows_e)
    x = _rand((E * rows_e, K), rows_e)
    call = gg.gmm_w4_swiglu if swiglu else gg.gmm_w4
    out = call(x, w, sizes.to(dev()))
    _check(out, x, ref, s, sizes, group, swiglu, False)
    # sizes on the host that say something else cost speed and nothing else (where they plan for few experts with many rows,
    # the library says that it takes the form through bf16 weights: the roundings are that form's)
    for wrong in ([0] * E, [E * rows_e] + [0] * (E - 1), [1] * E):
        wrong, need = torch.tensor(wrong), _lib.c_size_t(0)
        _lib.call("dmoe_gmm_w4_wide_bytes", E * rows_e, E, K, N, group, wrong.data_ptr(), _lib.ctypes.byref(need))
        other = call(x, w, sizes.to(dev()), host_batch_sizes=wrong)
        _check(other, x, ref, s, sizes, group, swiglu, need.value > 0)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("group,zeros,K", [(32, True, 416), (64, False, 416), (128, False, 416), (128, True, 392), (32, False, 1000)])
def test_many_rows(swiglu, group, zeros, K):
    announce(test="w4_many_rows", swiglu=swiglu, group=group, zeros=zeros, K=K)
    sizes = torch.tensor([1400, 0, 1, 1513])
    E, N, R = 4, 304, 2914
    w, ref, s = _weight(E, N, K, group, zeros, seed=3)
    x = _rand((R, K), 4)
    call = gg.gmm_w4_swiglu if swiglu else gg.gmm_w4
    for bs in (sizes, sizes.to(dev())):
        need = _lib.c_size_t(0)
        _lib.call("dmoe_gmm_w4_wide_bytes", R, E, K, N, group, None, _lib.ctypes.byref(need))
        assert need.value > 0                                    # the form for many rows
        _check(call(x, w, bs), x, ref, s, sizes, group, swiglu, True)
    size, ptr = gg.get_arguments(E, dev())
    own = call(x, w, sizes, workspace=torch.empty(size, dtype=torch.uint8, device=dev()), arguments_ptr=ptr)
    assert torch.equal(own, call(x, w, sizes))
    gg.release_arguments(ptr)
    # without room for 16-bit weights the one kernel takes any number of rows
    c = torch.empty(R, N // 2 if swiglu else N, dtype=torch.bfloat16, device=dev())
    _lib.call("dmoe_gmm_w4_swiglu" if swiglu else "dmoe_gmm_w4", x.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
              None if w.zeros is None else w.zeros.data_ptr(), group, c.data_ptr(), sizes.to(dev()).data_ptr(), R, E, K, c.shape[1], None, 0,
              None, None, 0, None, torch.cuda.current_stream().cuda_stream)
    _check(c, x, ref, s, sizes, group, swiglu, False)


@pytest.mark.parametrize("rows", [40, 1100])
def test_range_of_values(rows):
    announce(test="w4_range", rows=rows)
    # rows and columns of any size, values far apart in one row and one column, zeros, and what is not finite stays in its row
    K, N, group = 256, 64, 64
    sizes = torch.tensor([rows])
    x = _rand((rows, K), 1)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, ::2] *= 1e-6
    x[4, 5] = 1e4
    q = torch.randint(0, 16, (1, N, K), device=dev(), dtype=torch.uint8)
    s = torch.full((1, N, K // group), 0.01, device=dev())
    s[0, 0], s[0, 1], s[0, 2, 1:], s[0, 3] = 1e6, 1e-25, 1e-7, 0
    s = s.to(torch.bfloat16)
    w = gg.pack_w4(q, s, None, group)
    sd = s.double().repeat_interleave(group, 2)
    out = gg.gmm_w4(x, w, sizes)
    _check(out, x, (q.double() - 8) * sd, sd, sizes, group, False, rows > 512)
    assert bool((out[2] == 0).all()) and bool((out[:, 3] == 0).all())
    x[7, 3], x[8, 9] = float("inf"), float("nan")
    again = gg.gmm_w4(x, w, sizes)
    keep = [r for r in range(rows) if r not in (7, 8)]
    assert torch.equal(again[keep], out[keep]) and not bool(again[8].isfinite().any()) and not bool(again[7, 4:].isfinite().any())


def test_rows_keep_apart_and_rows_behind():
    announce(test="w4_apart")
    sizes = torch.tensor([3, 0, 20, 7])
    E, K, N, R = 4, 264, 64, 30
    w, ref, s = _weight(E, N, K, 32, True, seed=5)
    x = _rand((R + 9, K), 6)
    clean = gg.gmm_w4(x, w, sizes)[:R].clone()
    x[1], x[10], x[R:] = float("nan"), float("inf"), float("nan")
    c = torch.full((R + 20, N), 7.0, dtype=torch.bfloat16, device=dev())
    out = gg.gmm_w4(x, w, sizes, c=c)
    assert out.data_ptr() == c.data_ptr() and bool((c[R:] == 7).all())
    keep = [r for r in range(R) if r not in (1, 10)]
    assert torch.equal(c[keep], clean[keep]) and not bool(c[[1, 10]].isfinite().any())
    c.fill_(7)
    gg.gmm_w4_swiglu(x, w, torch.zeros(E, dtype=torch.int64), c=c[:, :N // 2].contiguous())
    assert bool((gg.gmm_w4(x, w, torch.zeros(E, dtype=torch.int64).to(dev()), c=c) == 7).all())
    assert gg.gmm_w4(x[:0], w, torch.zeros(E, dtype=torch.int64)).shape == (0, N)
    # sizes that overrun the rows are clamped
    guard = torch.full((R + 4, N), 5.0, dtype=torch.bfloat16, device=dev())
    gg.gmm_w4(x[:R].contiguous(), w, torch.tensor([3, 0, 20, 700]), c=guard)
    assert torch.equal(guard[23:R], clean[23:]) and bool((guard[R:] == 5).all())


@pytest.mark.parametrize("rows", [40, 600])
def test_scales_whose_product_leaves_the_range(rows):
    announce(test="w4_scales_range", rows=rows)
    # rows and columns whose scales multiplied lie outside fp32 while every result is zero or of ordinary size
    K, N, group = 256, 48, 128
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device=dev())
    x[:, 7] = 2.0 ** 110
    x[1::2, 7] = 2.0 ** -100
    x[:, 200] = 1.0
    q = torch.full((1, N, K), 8, device=dev(), dtype=torch.uint8)
    q[0, :, 200] = 9
    s = torch.ones(1, N, K // group, device=dev(), dtype=torch.bfloat16)
    s[0, :, 0] = 2.0 ** 40                                # of weights that are zero
    s[0, 16:, 0] = 2.0 ** -60
    s[0, 32:, 1] = 0
    out = gg.gmm_w4(x, gg.pack_w4(q, s, None, group), torch.tensor([rows]))
    assert bool((out[:, 32:] == 0).all())
    # (many rows: a 1 beside 2^110 in its row, or a scale of 1 beside 2^40 in its column, is below what fp16 has left)
    near = out[1::2, 16:32] if rows > 512 else out[:, :32]
    assert bool((near == 1).all()) and bool(out.isfinite().all())


def test_offsets_past_32_bits():
    announce(test="w4_offsets")
    # codes of 5 GiB, 16-bit weights of 20 GiB: the last expert's rows, few and many
    E, N, K, group = 80, 16384, 8192, 128
    codes, groups = gg._w4_shapes(E, K, N, group)
    w = gg.W4Weight(torch.zeros(codes, dtype=torch.uint8, device=dev()), torch.zeros(groups, dtype=torch.bfloat16, device=dev()), None, K, N, group)
    one, ref, s = _weight(1, N, K, group, False, 3)
    w.codes[E - 1], w.scales[E - 1] = one.codes[0], one.scales[0]
    for rows in (5, 100, 600):
        sizes = torch.zeros(E, dtype=torch.int64)
        sizes[E - 1] = rows
        x = _rand((rows, K), rows)
        got = gg.gmm_w4(x, w, sizes)
        assert torch.equal(got, gg.gmm_w4(x, one, torch.tensor([rows])))
        _check(got[:8, -64:], x[:8], ref[:, -64:], s[:, -64:], torch.tensor([min(rows, 8)]), group, False, rows > 512)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("zeros", [False, True])
def test_quantisation_of_tiny_weights(zeros):
    announce(test="w4_tiny", zeros=zeros)
    # down to the smallest numbers of bf16: a weight is off by half a step of its group and what the rounded scale cuts off
    # (2^-8 of 7.5 steps); a scale below 2^-126 counts as zero, and its weights, of up to 7 or 15 steps, with it
    K, N, group = 128, 48, 32
    w = _rand((1, K, N), 1) * (2.0 ** -torch.arange(100, 148, device=dev()).double()).to(torch.float32)
    w = w.to(torch.bfloat16)
    got = gg.dequantize_w4(gg.quantize_weight_w4(w, group=group, zeros=zeros))[0].t().double()
    v = w[0].double().view(K // group, group, N)
    top = v.abs().amax(1) / 7 if not zeros else (v.amax(1).clamp(min=0) - v.amin(1).clamp(max=0)) / 15
    allowed = torch.where(top * (1 + 2.0 ** -7) < 2.0 ** -126, 15 * 2.0 ** -126, top * (0.5 + 15 * 2.0 ** -8) + 2.0 ** -126)
    bad = (got.view_as(v) - v).abs() > allowed.unsqueeze(1)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows_e,N", [(5, 528), (5, 1040), (5, 4112), (5, 4128), (20, 528), (20, 2064), (20, 2080), (45, 528), (45, 1040), (45, 1056)])
def test_forms_for_more_and_less_work(rows_e, N, group, zeros):
    announce(test="w4_forms", rows_e=rows_e, N=N, group=group, zeros=zeros)
    # columns x row tiles on either side of every threshold between the forms; halves of N that are and are not whole tiles
    E, K = 40, 272
    sizes = ragged_sizes(E, E * rows_e, seed=N) if rows_e != 45 else torch.full((E,), rows_e, dtype=torch.int64)
    w, ref, s = _weight(E, N, K, group, zeros, seed=N + rows_e)
    x = _rand((int(sizes.sum()), K), N)
    _check(gg.gmm_w4(x, w, sizes), x, ref, s, sizes, group, False, False)
    _check(gg.gmm_w4_swiglu(x, w, sizes), x, ref, s, sizes, group, True, False)


def test_many_experts():
    announce(test="w4_many_experts")
    E, K, N = 300, 64, 32
    sizes = ragged_sizes(E, 500, seed=9)
    w, ref, s = _weight(E, N, K, 32, False, seed=8)
    x = _rand((500, K), 9)
    _check(gg.gmm_w4(x, w, sizes.to(dev())), x, ref, s, sizes, 32, False, False)


def test_sums_that_nearly_cancel():
    announce(test="w4_cancel")
    # every code is the zero point: the weights are zero whatever the rows
    E, K, N = 1, 512, 32
    q = torch.full((E, N, K), 8, dtype=torch.uint8, device=dev())
    s = torch.ones(E, N, K // 128, dtype=torch.bfloat16, device=dev())
    x = _rand((5, K), 2) + 3
    out = gg.gmm_w4(x, gg.pack_w4(q, s, None, 128), torch.tensor([5]))
    assert bool((out.double().abs() <= ACC * 136 * 47 * x.double().abs().sum(1, keepdim=True)).all())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N", [(128, 48), (72, 24), (328, 136)])
def test_quantisation(K, N, group, zeros):
    announce(test="w4_quant", K=K, N=N, group=group, zeros=zeros)
    E = 2
    w = _rand((E, K, N), K, 0.02)
    w[0, :, 3] = 0                                               # a column of zeros
    w[1, :, 5] = w[1, :, 5].abs() + 0.01                         # one without a negative weight
    w[0, 7, 7] = 4.0                                             # one with an outlier
    p = gg.quantize_weight_w4(w, group, zeros)
    q, s, z = unpack(p)
    assert int(q.max()) <= 15 and bool((s.double() >= 0).all())
    spread = lambda v: v.double().repeat_interleave(group, 2)[:, :, :K]
    step = spread(s)
    value = (q.double() - (8.0 if z is None else spread(z))) * step
    wt = w.cpu().double().transpose(1, 2)
    # off by half a step; at the ends by what rounding the step to bf16 moves them (7 or 15 steps by HALF each, with zero
    # points half a step more, by which the zero point is off its place)
    off = (0.5 + (15 * HALF + 0.5 if zeros else 7 * HALF)) * step + 1e-6
    assert bool(((value - wt).abs() <= off).all()), float(((value - wt).abs() / step.clamp(min=1e-9)).max())
    assert bool((value[0, 3] == 0).all())
    assert torch.equal(gg.dequantize_w4(p).cpu(), value.to(torch.bfloat16))
    again = gg.pack_w4(q, s, z, group)
    assert torch.equal(again.codes, p.codes.cpu()) and torch.equal(again.scales, p.scales.cpu())


@pytest.mark.parametrize("T", [1, 40, 700])
@pytest.mark.parametrize("zeros", [False, True])
def test_layer(T, zeros):
    announce(test="w4_layer", T=T, zeros=zeros)
    # quantise, then the whole step: route -> permute -> 4-bit experts -> combine
    E, d, I, k = 8, 256, 328, 2
    w13, w2 = _rand((E, d, 2 * I), 1, 0.05), _rand((E, I, d), 2, 0.05)
    layer = MoEExpertsW4(w13, w2, group=64, zeros=zeros)
    assert sorted(n for n, _ in layer.named_buffers()) == sorted(
        [f"{w}_{t}" for w in ("w13", "w2") for t in ("codes", "scales") + (("zeros",) if zeros else ())])
    g = torch.Generator().manual_seed(T)
    x = _rand((T, d), 3)
    ids = torch.argsort(torch.rand(T, E, generator=g), dim=1)[:, :k].to(torch.int32).to(dev())
    gates = torch.softmax(torch.randn(T, k, generator=g), 1).to(dev())
    stages = {}
    out = expert_layer_forward(layer, x, ids, gates, stages=stages)
    b13 = gg.dequantize_w4(gg.quantize_weight_w4(w13, 64, zeros)).double()
    b2 = gg.dequantize_w4(gg.quantize_weight_w4(w2, 64, zeros)).double()
    xd, want = x.double(), torch.zeros(T, d, dtype=torch.float64, device=dev())
    for j in range(k):
        for t in range(T):
            e = int(ids[t, j])
            u = b13[e] @ xd[t]
            want[t] += float(gates[t, j]) * (b2[e] @ (torch.nn.functional.silu(u[:I]) * u[I:]))
    # roundings: the reference's weights, the intermediate, the rows and the sum: four of them, of the terms of sums of I
    # and d elements that are as good as independent: a tenth of the largest value at most is never reached
    assert float((out.double() - want).abs().max()) <= 4 * HALF * float(want.abs().max())
    sizes = stages["batch_sizes"]
    again = layer.forward(T * k, stages["permuted"], sizes, host_batch_sizes=sizes.cpu())
    assert torch.equal(again, stages["expert_out"]) or T > 100
    ready = MoEExpertsW4(gg.quantize_weight_w4(w13, 64, zeros), gg.quantize_weight_w4(w2, 64, zeros))
    assert torch.equal(ready.forward(T * k, stages["permuted"], sizes), stages["expert_out"])


@pytest.mark.parametrize("T", [6, 400, 1200])
def test_graph_replays_and_streams(T):
    announce(test="w4_graph", T=T)
    E, d, I = 4, 256, 136
    layer = MoEExpertsW4(_rand((E, d, 2 * I), 1, 0.05), _rand((E, I, d), 2, 0.05), group=32, zeros=True)
    x = torch.zeros(T * 2, d, dtype=torch.bfloat16, device=dev())
    sizes = torch.zeros(E, dtype=torch.int64, device=dev())
    sizes[0] = T * 2
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.forward(T * 2, x, sizes)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.forward(T * 2, x, sizes)
    for rep in range(4):
        x.copy_(_rand((T * 2, d), rep))
        sizes.copy_(ragged_sizes(E, T * 2, seed=rep, empty_every=rep + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            want = layer.forward(T * 2, x, sizes)
        side.synchronize()
        assert torch.equal(got, want), rep


def test_refusals():
    announce(test="w4_refusals")
    w, _, _ = _weight(2, 32, 64, 32, True, 1)
    x, n = _rand((4, 64), 1), torch.tensor([2, 2])
    for bad in (x.float(), x[:, :56], x.t().contiguous().t(), x.cpu()):
        with pytest.raises(AssertionError):
            gg.gmm_w4(bad, w, n)
    for bad in (w._replace(K=72), w._replace(N=40), w._replace(group=64), w._replace(scales=w.scales.float()), w._replace(zeros=w.scales),
                w._replace(codes=w.codes[:1])):
        with pytest.raises(AssertionError):
            gg.gmm_w4(x, bad, n)
    with pytest.raises(ValueError):
        gg.gmm_w4(x, w._replace(group=16), n)
    with pytest.raises(AssertionError):
        gg.gmm_w4(x, w, torch.tensor([4]))
    w8, _, _ = _weight(2, 24, 64, 32, True, 1)
    with pytest.raises(AssertionError):
        gg.gmm_w4_swiglu(x, w8, n)
    with pytest.raises(AssertionError):
        gg.quantize_weight_w4(_rand((2, 64, 32), 1).float())
    with pytest.raises(RuntimeError, match="multiple of 8"):
        gg.quantize_weight_w4(_rand((1, 12, 16), 1))
