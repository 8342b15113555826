"""4-bit weights of unusual values: scales below zero, few columns under long contractions, what is not finite, and values
that are smaller than the normal numbers.  Tolerances: those of the 4-bit products' tests."""
import pytest
import torch

from disagmoe_amd.expert_layer import expert_layer_forward
from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.models.experts import MoEExpertsW4
from helpers import announce, dev
from test_gpu_w4 import ACC, HALF, _check, _rand, _weight
from test_w4_host import unpack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("rows", [1, 30, 60, 1100])
@pytest.mark.parametrize("group,zeros", [(32, True), (128, False)])
def test_negative_scales(rows, swiglu, group, zeros):
    announce(test="w4_negative_scales", rows=rows, swiglu=swiglu, group=group, zeros=zeros)
    E, N, K = 1, 144, 520
    g = torch.Generator(device=dev()).manual_seed(rows)
    q = torch.randint(0, 16, (E, N, K), generator=g, device=dev(), dtype=torch.uint8)
    s = ((torch.rand(E, N, -(-K // group), generator=g, device=dev()) - 0.5) * 0.05).to(torch.bfloat16)
    z = torch.randint(0, 16, s.shape, generator=g, device=dev(), dtype=torch.uint8) if zeros else None
    spread = lambda v: v.double().repeat_interleave(group, 2)[:, :, :K]
    ref = (q.double() - (8.0 if z is None else spread(z))) * spread(s)
    w, x, sizes = gg.pack_w4(q, s, z, group), _rand((rows, K), rows), torch.tensor([rows])
    out = (gg.gmm_w4_swiglu if swiglu else gg.gmm_w4)(x, w, sizes)
    _check(out, x, ref, spread(s).abs(), sizes, group, swiglu, rows > 512)
    assert torch.equal(gg.dequantize_w4(w), ref.to(torch.bfloat16))


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("N", [16, 48, 208, 272])
@pytest.mark.parametrize("K,group", [(16392, 32), (12288, 128)])
def test_few_columns_and_long_contractions(N, K, group, swiglu):
    announce(test="w4_few_columns", N=N, K=K, group=group, swiglu=swiglu)
    sizes = torch.tensor([900, 0, 1203])
    w, ref, s = _weight(3, N, K, group, True, seed=N)
    x = _rand((2103, K), K)
    call = gg.gmm_w4_swiglu if swiglu else gg.gmm_w4
    _check(call(x, w, sizes), x, ref, s, sizes, group, swiglu, True)
    few = torch.tensor([5, 0, 9])
    _check(call(x[:14], w, few), x[:14], ref, s, few, group, swiglu, False)


@pytest.mark.parametrize("zeros", [False, True])
def test_plans_of_a_layer_agree(zeros):
    """700 tokens planned from the sizes on the host and from the device's alone: other forms, whose results differ by their
    roundings.  Either form is off by at most ``_off`` before it rounds its result: the intermediate h by the slope of the
    gated activation times that and half a step, the result by what h is off times the weights, ``_off`` and half a step."""
    announce(test="w4_layer_plans", zeros=zeros)
    E, d, I, T, k = 8, 256, 328, 700, 2
    w13, w2 = _rand((E, d, 2 * I), 1, 0.05), _rand((E, I, d), 2, 0.05)
    layer = MoEExpertsW4(w13, w2, group=64, zeros=zeros)
    x = _rand((T, d), 3)
    ids = torch.zeros(T, k, dtype=torch.int32, device=dev())
    ids[:, 1] = 3
    stages = {}
    expert_layer_forward(layer, x, ids, torch.full((T, k), 0.5, device=dev()), stages=stages)
    sizes, rows = stages["batch_sizes"], stages["permuted"]
    host = sizes.cpu()
    assert host.tolist() == [T, 0, 0, T] + [0] * 4              # 700 rows a busy expert, 175 an expert
    again = layer.forward(T * k, rows, sizes, host_batch_sizes=host)
    unpacked = []
    for w in (w13, w2):
        q, scales, z = unpack(gg.quantize_weight_w4(w, 64, zeros))
        spread = lambda v: v.double().repeat_interleave(64, 2)[:, :, :q.shape[2]]
        unpacked.append((((q.double() - (8 if z is None else spread(z))) * spread(scales)).to(dev()), spread(scales).to(dev())))
    (b13, s13), (b2, s2) = unpacked
    for e, at in ((0, slice(0, T)), (3, slice(T, 2 * T))):
        a = rows[at].double()
        u, off = a @ b13[e].t(), _off(a, b13[e], s13[e])
        g, p = u[:, :I], u[:, I:]
        sig = torch.sigmoid(g)
        h = g * sig * p
        off = 1.05 * ((p * sig * (1 + g * (1 - sig))).abs() * off[:, :I] + (g * sig).abs() * off[:, I:] + off[:, :I] * off[:, I:]) + 1e-6 * h.abs()
        off = off + HALF * (h.abs() + off)
        result = off @ b2[e].abs().t() + _off(h.abs() + off, b2[e], s2[e])
        result = result + HALF * ((h @ b2[e].t()).abs() + result)
        assert bool(((again[at].double() - stages["expert_out"][at].double()).abs() <= 2 * result).all())


def _off(a, w, s):
    """What either form is off by before its result is rounded: the larger of the two that ``_check`` counts."""
    mag = a.abs() @ w.abs().t()
    one = ACC * (64 + 8) * 47 * (a.abs() @ s.t()) + ACC * (a.shape[1] / 64 + 16) * mag
    many = (2.0 ** -11 + ACC * (a.shape[1] + 4)) * mag
    many = many + 2.0 ** -24 * (a.abs().sum(1, keepdim=True) * 16 * s.max(1).values + a.abs().max(1, keepdim=True).values * w.abs().sum(1))
    return torch.maximum(one, many)


@pytest.mark.parametrize("rows", [3, 30, 60, 700])
def test_rows_and_scales_below_the_normal_numbers(rows):
    """bf16 has numbers down to 2^-133: rows that hold no larger one, and columns whose scales are no larger, count."""
    announce(test="w4_subnormal", rows=rows)
    K, N, group = 256, 48, 128
    g = torch.Generator(device=dev()).manual_seed(rows)
    x = (torch.randint(-100, 101, (rows, K), generator=g, device=dev()).double() * 2.0 ** -133).to(torch.bfloat16)
    q = torch.randint(0, 16, (1, N, K), generator=g, device=dev(), dtype=torch.uint8)
    spread = lambda v: v.double().repeat_interleave(group, 2)[:, :, :K]
    s = (torch.rand(1, N, K // group, generator=g, device=dev()).double() * 2.0 ** 120).to(torch.bfloat16)
    out = gg.gmm_w4(x, gg.pack_w4(q, s, None, group), torch.tensor([rows]))
    _check(out, x, (q.double() - 8) * spread(s), spread(s), torch.tensor([rows]), group, False, rows > 512)
    x = (torch.randn(rows, K, generator=g, device=dev()).double() * 2.0 ** 110).to(torch.bfloat16)
    s = (torch.randint(1, 128, s.shape, generator=g, device=dev()).double() * 2.0 ** -133).to(torch.bfloat16)
    out = gg.gmm_w4(x, gg.pack_w4(q, s, None, group), torch.tensor([rows]))
    _check(out, x, (q.double() - 8) * spread(s), spread(s), torch.tensor([rows]), group, False, rows > 512)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantisation_of_what_is_not_finite(group, zeros):
    """A group with an infinity or NaN has NaN weights, and no other group has; ones that finite weights of the largest
    magnitudes fill are finite."""
    announce(test="w4_not_finite", group=group, zeros=zeros)
    K, N = 264, 32
    w = _rand((1, K, N), group)
    top = 2.0 ** 127      # (not the largest bf16: seven steps, rounded up by 2^-8 of them, would lie past it)
    w[0, :, 4], w[0, 1, 4], w[0, 2, 4] = 0, top, -top
    clean = gg.dequantize_w4(gg.quantize_weight_w4(w, group, zeros))
    assert bool(clean.isfinite().all())
    # within half a step (a whole one with zero points, off by half a step too) and what the step's rounding moves its ends by
    step = 2 * top / 15 if zeros else top / 7
    assert bool(((clean[0, 4, 1:3].double() - torch.tensor([top, -top], device=dev())).abs() <= (1.5 + 15 * HALF) * step).all())
    bad = [(0, 3, float("nan")), (130, 7, float("inf")), (263, 9, float("-inf")), (40, 31, float("nan"))]
    for k, n, v in bad:
        w[0, k, n] = v
    q = gg.quantize_weight_w4(w, group, zeros)
    got, want = gg.dequantize_w4(q), clean.clone()
    for k, n, _ in bad:
        want[0, n, k // group * group:(k // group + 1) * group] = float("nan")
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    for rows in (3, 700):
        out = gg.gmm_w4(_rand((rows, K), rows), q, torch.tensor([rows]))
        assert torch.equal(out.isnan().all(0), want[0].isnan().any(1)) and torch.equal(out.isnan().any(0), want[0].isnan().any(1))


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
def test_one_round_of_workgroups_and_more(group, zeros, swiglu):
    """64-row tiles on either side of where one round of workgroups ends: 32 and 36 workgroups of 128 columns to an XCD."""
    K = 200
    for E, N in ((8, 4096), (9, 3584)):
        announce(test="w4_rounds", E=E, N=N, group=group, zeros=zeros, swiglu=swiglu)
        sizes = torch.tensor([64, 33, 0, 64, 1, 50] + [64] * (E - 6))
        sizes[2] = 64 * E - int(sizes.sum())
        w, ref, s = _weight(E, N, K, group, zeros, seed=N)
        x = _rand((64 * E, K), E)
        _check((gg.gmm_w4_swiglu if swiglu else gg.gmm_w4)(x, w, sizes), x, ref, s, sizes, group, swiglu, False)
        even = torch.full((E,), 64)
        _check((gg.gmm_w4_swiglu if swiglu else gg.gmm_w4)(x, w, even), x, ref, s, even, group, swiglu, False)
