"""The gated block and the grouped product under autograd, against the formulas in 64 bits.

Tolerances, element by element.  A bf16 result is off by half a step, 2^-8 of its value (``HALF``), and by its sum: n
products added in fp32 in any order are off by at most n 2^-24 times the sum of their magnitudes (``ACC`` counts twice that,
for a matrix core that adds more than two terms at a time).  What a later product reads rounded carries its own error into
the sum, weighted with the magnitudes it meets."""
import pytest
import torch

from disagmoe_amd.grouped_gemm import backend as gg
from disagmoe_amd.grouped_gemm import ops
from disagmoe_amd.models.experts import MoEExperts
from disagmoe_amd.ops import grads
from helpers import announce, dev, ragged_sizes

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8
ACC = 2 * 2.0 ** -24
TINY = 2.0 ** -126


def _rand(shape, seed, std=1.0):
    g = torch.Generator(device=dev()).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev()) * std).to(torch.bfloat16)


def _spans(sizes):
    o = 0
    for e, n in enumerate(sizes.tolist()):
        yield e, slice(o, o + n), n
        o += n


def _close(got, want, off, what=""):
    """|got - want| <= off + half a step of want; got is finite wherever want is."""
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    err = (got.double() - want).abs()
    allowed = off + HALF * (want.abs() + off) + 1e-37
    bad = ~(err <= allowed)
    assert not bool(bad.any()), (what, int(bad.sum()), float(err[bad][0]), float(allowed[bad][0]))


def _check_wgrad(db, a, dc, sizes):
    for e, at, n in _spans(sizes):
        x, d = a[at].double(), dc[at].double()
        _close(db[e], x.t() @ d, ACC * (n + 4) * (x.abs().t() @ d.abs()), f"expert {e} of {n} rows")


def _check_block(u, h, da, db, a, b, dh, sizes):
    """u and h against the operands, da and db against the kept u (b in the [E, K, 2I] layout)."""
    I = h.shape[1]
    for e, at, n in _spans(sizes):
        x, w, d = a[at].double(), b[e].double(), dh[at].double()
        want_u = x @ w
        off_u = ACC * (x.shape[1] + 4) * (x.abs() @ w.abs())
        assert u.dtype == torch.float32 and bool(((u[at].double() - want_u).abs() <= off_u + 2.0 ** -24 * want_u.abs()).all())
        g, p = want_u[:, :I], want_u[:, I:]
        s = torch.sigmoid(g)
        slope = (p * s * (1 + g * (1 - s))).abs()
        # (second-order terms: 1 % of the first-order ones)
        off_h = 1.01 * (slope * off_u[:, :I] + (g * s).abs() * off_u[:, I:])
        _close(h[at], g * s * p, off_h + 1e-6 * (g * s * p).abs() + 2e-4 * HALF * p.abs(), "h")
        g, p = u[at].double()[:, :I], u[at].double()[:, I:]
        s = torch.sigmoid(g)
        du = torch.cat([d * p * s * (1 + g * (1 - s)), d * g * s], 1)
        size = torch.cat([(d * p * s) * (1 + g.abs()), d * g * s], 1).abs()
        off_du = HALF * du.abs() + 1e-6 * size               # rounded once; 8 fp32 operations and two functions of 1 - 2 ulp
        # Below 2^-126, where the normal numbers of fp32 and bf16 end, a value may count as zero: s itself (off by less than
        # TINY, which its factors in du carry on: |d p| (1 + |g|) in the gate's half, |d g| in the other) and du.
        off_du = off_du + TINY * (1 + torch.cat([(d * p).abs() * (1 + g.abs()), (d * g).abs()], 1))
        if da is not None:
            _close(da[at], du @ w.t(), off_du @ w.abs().t() + ACC * (2 * I + 4) * (du.abs() @ w.abs().t()), "da")
        if db is not None:
            _close(db[e], x.t() @ du, x.abs().t() @ off_du + ACC * (n + 4) * (x.abs().t() @ du.abs()), f"db of {n} rows")


SIZES = [
    [1], [0], [31], [32], [33], [64, 0, 65], [0, 0, 96, 1, 0, 127, 128, 129, 0], [2, 1, 3, 1, 1, 2], [300, 700], [1000, 24, 513, 160],
]


@pytest.mark.parametrize("K,N", [(8, 8), (64, 264), (256, 256), (520, 40), (128, 768)])
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_wgrad(sizes, K, N):
    announce(test="wgrad", sizes=sizes, K=K, N=N)
    sizes = torch.tensor(sizes)
    R = int(sizes.sum())
    a, dc = _rand((R, K), R + 1), _rand((R, N), R + 2)
    db = gg.gmm_wgrad(a, dc, sizes)
    assert db.shape == (len(sizes), K, N)
    _check_wgrad(db, a, dc, sizes)
    assert torch.equal(db, gg.gmm_wgrad(a, dc, sizes.to(dev()), host_batch_sizes=sizes))
    assert bool((db[sizes.to(dev()) == 0] == 0).all())


def test_wgrad_keeps_experts_apart():
    announce(test="wgrad_apart")
    # what is not finite stays in its expert; rows behind the last expert's (not finite here) reach nobody
    sizes = torch.tensor([40, 3, 29, 0, 70])
    R, K, N = 142, 264, 72
    a, dc = _rand((R + 10, K), 1), _rand((R + 10, N), 2)
    a[41], dc[42] = float("inf"), float("nan")
    a[R:], dc[R:] = float("nan"), float("inf")
    db = gg.gmm_wgrad(a, dc, sizes)
    assert not bool(db[1].isfinite().any())
    clean_a, clean_d = a.clone(), dc.clone()
    for t in (clean_a, clean_d):
        t[40:43] = 0
        t[R:] = 0
    db[1] = 0
    _check_wgrad(db, clean_a, clean_d, sizes)
    # sizes that overrun the operands are clamped
    over = gg.gmm_wgrad(a[:R].contiguous(), dc[:R].contiguous(), torch.tensor([40, 3, 29, 0, 700]))
    assert torch.equal(over[4], db[4]) and torch.equal(over[0], db[0])


def test_wgrad_many_experts_and_long_contraction():
    announce(test="wgrad_many_experts")
    sizes = ragged_sizes(200, 1500, seed=3)
    a, dc = _rand((1500, 40), 5), _rand((1500, 24), 6)
    _check_wgrad(gg.gmm_wgrad(a, dc, sizes), a, dc, sizes)
    sizes = torch.tensor([20000, 1])
    a, dc = _rand((20001, 264), 7), _rand((20001, 512), 8)
    _check_wgrad(gg.gmm_wgrad(a, dc, sizes), a, dc, sizes)


@pytest.mark.parametrize("sizes", [[1024], [3001], [1700, 0, 900], [4000, 37], [0, 20000, 1, 0]], ids=str)
@pytest.mark.parametrize("K,N", [(8, 264), (264, 512)])
def test_wgrad_of_few_tiles(sizes, K, N):
    announce(test="wgrad_few_tiles", sizes=sizes, K=K, N=N)
    # contractions that are cut in pieces: pieces of any length, experts without rows, the same bits every time, and a state
    # block that every launch leaves clean
    sizes = torch.tensor(sizes)
    R = int(sizes.sum())
    a, dc = _rand((R, K), R + 1), _rand((R, N), R + 2)
    size, ptr = gg.get_arguments(len(sizes), dev())
    own = dict(arguments_ptr=ptr, workspace=torch.empty(size, dtype=torch.uint8, device=dev()).fill_(255))
    db = gg.gmm_wgrad(a, dc, sizes, **own)
    _check_wgrad(db, a, dc, sizes)
    for _ in range(3):
        assert torch.equal(db, gg.gmm_wgrad(a, dc, sizes, **own))
    _check_wgrad(gg.gmm_wgrad(a, dc, sizes, arguments_ptr=ptr), a, dc, sizes)      # no workspace: nothing is cut
    small = own["workspace"][:3 * 256 * 256 * 4]
    _check_wgrad(gg.gmm_wgrad(a, dc, sizes, arguments_ptr=ptr, workspace=small), a, dc, sizes)
    assert not bool(gg._STATE_BLOCKS[ptr].any())
    gg.release_arguments(ptr)


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("E,R,K,I", [(1, 1, 8, 8), (3, 50, 64, 40), (4, 300, 256, 128), (6, 900, 264, 328), (5, 1500, 512, 136),
                                     (64, 500, 128, 96), (2, 700, 1024, 256)])
def test_gated_block(E, R, K, I, trans_b):
    announce(test="gated_block", E=E, R=R, K=K, I=I, trans_b=trans_b)
    sizes = ragged_sizes(E, R, seed=E + R) if E > 1 else torch.tensor([R])
    a, b, dh = _rand((R, K), 1), _rand((E, K, 2 * I), 2, 1.0 / K ** 0.5), _rand((R, I), 3)
    bl = b.transpose(1, 2).contiguous() if trans_b else b
    h, u = gg.gmm_swiglu_keep(a, bl, sizes, trans_b=trans_b)
    da, db = gg.gmm_swiglu_backward(dh, u, a, bl, sizes, trans_b=trans_b)
    _check_block(u, h, da, db.transpose(1, 2) if trans_b else db, a, b, dh, sizes)
    # the same through autograd, and each gradient alone
    x, w = a.clone().requires_grad_(), bl.clone().requires_grad_()
    y = ops.gmm_swiglu(x, w, sizes.to(dev()), trans_b=trans_b)
    assert torch.equal(y, h)
    gx, gw = torch.autograd.grad(y, (x, w), dh, retain_graph=True)
    assert torch.equal(gx, da) and torch.equal(gw, db)
    assert torch.equal(torch.autograd.grad(y, x, dh, retain_graph=True)[0], da)
    assert torch.equal(torch.autograd.grad(y, w, dh)[0], db)
    with torch.no_grad():
        fused = ops.gmm_swiglu(x, w, sizes, trans_b=trans_b)
    assert torch.equal(fused, y) and not fused.requires_grad     # the same sums, kept or not


@pytest.fixture
def default_tile():
    yield
    gg.set_tile_variant(0)


@pytest.mark.parametrize("variant", [0, 5, 6, 7])
@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("sizes,K,I", [([5], 8, 8), ([300, 0, 17], 24, 4), ([70, 1, 256, 257], 40, 300), ([600, 520], 4104, 132),
                                       ([33], 8200, 4100), ([2000, 0, 1500], 1000, 516), ([900, 700], 56, 2052), ([3] * 40, 1000, 72),
                                       ([1600, 4000], 40, 2052), ([3000, 40], 4104, 1500), ([5000], 8, 1800)], ids=str)
def test_contractions_that_end_inside_a_stage(sizes, K, I, trans_b, variant, default_tile):
    announce(test="block_tail", sizes=sizes, K=K, I=I, trans_b=trans_b, variant=variant)
    # K and 2I of any multiple of 8, long ones of few tiles among them (cut into pieces).  The rows, weights and gradients
    # stand in front of NaN: a k past the end that got into a product would show, as a zero times it would.
    if I % 8:
        I += 4
    E, R, sizes = len(sizes), sum(sizes), torch.tensor(sizes)
    gg.set_tile_variant(variant)                          # (5, 6, 7: tiles of 64, 128 and 256 rows)

    def guarded(*shape, seed, std=1.0):
        n = 1
        for s in shape:
            n *= s
        buf = torch.full((n + 4096,), float("nan"), device=dev(), dtype=torch.bfloat16)
        buf[:n] = _rand((n,), seed, std)
        return buf[:n].view(shape)
    a, dh = guarded(R, K, seed=1), guarded(R, I, seed=3)
    w = (2 * I, K) if trans_b else (K, 2 * I)
    b = guarded(E, *w, seed=2, std=K ** -0.5)
    h, u = gg.gmm_swiglu_keep(a, b, sizes, trans_b=trans_b)
    da, db = gg.gmm_swiglu_backward(dh, u, a, b, sizes, trans_b=trans_b)
    _check_block(u, h, da, db.transpose(1, 2) if trans_b else db, a, b.transpose(1, 2) if trans_b else b, dh, sizes)


def test_offsets_past_32_bits():
    announce(test="ffn_offsets")
    # sums of 4.5 GB, then weight gradients of 5.4 GB: what lies at the far end
    K, I, sizes = 64, 16384, torch.tensor([33000, 1000])
    a, b, dh = _rand((34000, K), 1), _rand((2, K, 2 * I), 2, 0.125), _rand((34000, I), 3)
    h, u = gg.gmm_swiglu_keep(a, b, sizes)
    da, db = gg.gmm_swiglu_backward(dh, u, a, b, sizes)
    _check_block(u[33000:], h[33000:], da[33000:], db[1:], a[33000:], b[1:], dh[33000:], torch.tensor([1000]))
    del u, h, da, db, dh
    E, K, N = 40, 8192, 8192
    sizes = torch.zeros(E, dtype=torch.int64)
    sizes[0], sizes[E - 1] = 30, 40
    a, dc = _rand((70, K), 4), _rand((70, N), 5)
    db = gg.gmm_wgrad(a, dc, sizes)
    for e, at in ((0, slice(0, 30)), (E - 1, slice(30, 70))):
        x, d = a[at].double(), dc[at].double()
        _close(db[e], x.t() @ d, ACC * 44 * (x.abs().t() @ d.abs()))
    assert not bool(db[1:E - 1].any())
    del db
    torch.cuda.empty_cache()


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("variant", range(1, 9))
def test_gated_block_on_every_tile(variant, trans_b, default_tile):
    announce(test="gated_block_tiles", variant=variant, trans_b=trans_b)
    # tiles full of rows and tiles with a few, columns that end inside one, more than one k-stage
    E, K, I = 4, 160, 328
    sizes = torch.tensor([600, 0, 17, 303])
    R = 920
    gg.set_tile_variant(variant)
    a, b, dh = _rand((R, K), 1), _rand((E, K, 2 * I), 2, 1.0 / K ** 0.5), _rand((R, I), 3)
    bl = b.transpose(1, 2).contiguous() if trans_b else b
    h, u = gg.gmm_swiglu_keep(a, bl, sizes, trans_b=trans_b)
    da, db = gg.gmm_swiglu_backward(dh, u, a, bl, sizes, trans_b=trans_b)
    _check_block(u, h, da, db.transpose(1, 2) if trans_b else db, a, b, dh, sizes)
    if not (variant == 8 and not trans_b):                       # (that hook's own kernel keeps nothing: other sums)
        assert torch.equal(h, gg.gmm_swiglu(a, bl, sizes, trans_b=trans_b))


def test_gated_block_that_fills_the_chip():
    announce(test="gated_block_large")
    E, K, I, R = 3, 96, 4104, 2300
    sizes = torch.tensor([1000, 5, 1295])
    a, b, dh = _rand((R, K), 1), _rand((E, K, 2 * I), 2, 1.0 / K ** 0.5), _rand((R, I), 3)
    for host in (None, sizes):
        h, u = gg.gmm_swiglu_keep(a, b, sizes.to(dev()), host_batch_sizes=host)
        da, db = gg.gmm_swiglu_backward(dh, u, a, b, sizes.to(dev()), host_batch_sizes=host)
        _check_block(u, h, da, db, a, b, dh, sizes)
        assert torch.equal(h, gg.gmm_swiglu(a, b, sizes.to(dev()), host_batch_sizes=host))


def test_gated_block_where_the_gate_saturates():
    announce(test="gated_block_saturated")
    # gates from -200 to 200: exp(-g) leaves the range of fp32, the sigmoid is 0 or 1 to the last bit
    R, K, I = 64, 64, 64
    a = torch.zeros(R, K, dtype=torch.bfloat16, device=dev())
    a[torch.arange(R), torch.arange(K)] = 1
    b = torch.zeros(1, K, 2 * I, dtype=torch.bfloat16, device=dev())
    b[0, :, :I] = torch.linspace(-200, 200, K, device=dev()).to(torch.bfloat16)[:, None]
    b[0, :, I:] = 1.5
    dh, sizes = _rand((R, I), 9), torch.tensor([R])
    h, u = gg.gmm_swiglu_keep(a, b, sizes)
    da, db = gg.gmm_swiglu_backward(dh, u, a, b, sizes)
    assert bool(h.isfinite().all()) and bool(da.isfinite().all()) and bool(db.isfinite().all())
    _check_block(u, h, da, db, a, b, dh, sizes)


def test_gradient_against_differences():
    announce(test="gated_block_differences")
    E, R, K, I = 3, 96, 64, 48
    sizes = torch.tensor([50, 0, 46])
    a, b, dh = _rand((R, K), 1), _rand((E, K, 2 * I), 2, 0.125), _rand((R, I), 3)
    x, w = a.clone().requires_grad_(), b.clone().requires_grad_()
    da, db = torch.autograd.grad(ops.gmm_swiglu(x, w, sizes), (x, w), dh)

    def f(x, w):
        total = 0.0
        for e, at, n in _spans(sizes):
            u = x[at] @ w[e]
            total = total + (torch.nn.functional.silu(u[:, :I]) * u[:, I:] * dh[at].double()).sum()
        return float(total)

    va, vb = _rand((R, K), 4).double(), _rand((E, K, 2 * I), 5, 0.125).double()
    t = 1e-4
    for g, dx, dw in ((da, va, 0 * vb), (db, 0 * va, vb)):
        v = dx if g is da else dw
        slope = (f(a.double() + t * dx, b.double() + t * dw) - f(a.double() - t * dx, b.double() - t * dw)) / (2 * t)
        # every gradient element is off by at most 2 roundings (du, itself) of the terms in its sum; as independent errors of
        # the n elements they add like sqrt(n), 6 of their deviations are allowed, and as much for the terms' spread
        off = 6 * 4 * HALF * float((g.double() * v).square().sum().sqrt()) + 6 * 4 * HALF * float(v.square().sum().sqrt() * g.double().square().mean().sqrt())
        assert abs(slope - float((g.double() * v).sum())) <= off, (slope, float((g.double() * v).sum()), off)


def test_rows_behind_the_last_expert():
    announce(test="rows_behind")
    sizes = torch.tensor([17, 0, 40])
    R, K, I = 90, 128, 64
    a, b, dh = _rand((R, K), 1), _rand((3, K, 2 * I), 2, 0.1), _rand((R, I), 3)
    a[57:], dh[57:] = float("nan"), float("inf")
    for bs, host in ((sizes, None), (sizes.to(dev()), None), (sizes.to(dev()), sizes)):
        x, w = a.clone().requires_grad_(), b.clone().requires_grad_()
        y = ops.gmm_swiglu(x, w, bs, host_batch_sizes=host)
        assert bool((y[57:] == 0).all())
        gx, gw = torch.autograd.grad(y, (x, w), dh)
        assert bool((gx[57:] == 0).all()) and bool(gx.isfinite().all()) and bool(gw.isfinite().all()) and bool((gw[1] == 0).all())
        z = ops.gmm(x, w, bs, host_batch_sizes=host)
        assert bool((z[57:] == 0).all())
        gx, gw = torch.autograd.grad(z, (x, w), torch.cat([dh, dh], 1))
        assert bool((gx[57:] == 0).all()) and bool(gx.isfinite().all()) and bool(gw.isfinite().all())
    # no rows at all, and rows that all lie behind
    for n in (0, 5):
        x = torch.full((n, K), float("nan"), dtype=torch.bfloat16, device=dev(), requires_grad=True)
        w = b.clone().requires_grad_()
        y = ops.gmm(ops.gmm_swiglu(x, w, torch.zeros(3, dtype=torch.int64)), w.detach()[:, :I].contiguous(), torch.zeros(3, dtype=torch.int64))
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == (n, 2 * I) and bool((y == 0).all()) and bool((gx == 0).all()) and bool((gw == 0).all())


@pytest.mark.parametrize("trans_b", [False, True])
def test_product(trans_b):
    announce(test="product_grad", trans_b=trans_b)
    sizes = ragged_sizes(5, 700, seed=2)
    a, b, dc = _rand((700, 264), 1), _rand((5, 264, 136), 2, 0.06), _rand((700, 136), 3)
    x = a.clone().requires_grad_()
    w = (b.transpose(1, 2).contiguous() if trans_b else b.clone()).requires_grad_()
    c = ops.gmm(x, w, sizes, trans_b=trans_b)
    assert torch.equal(c, gg.gmm(a, w.detach(), sizes, trans_b=trans_b))
    # a gradient that arrives in another order of memory
    gx, gw = torch.autograd.grad(c, (x, w), dc.t().contiguous().t())
    gw = gw.transpose(1, 2) if trans_b else gw
    _check_wgrad(gw, a, dc, sizes)
    for e, at, n in _spans(sizes):
        d, m = dc[at].double(), b[e].double()
        _close(gx[at], d @ m.t(), ACC * 140 * (d.abs() @ m.abs().t()), "da")
    # every row of the gradient alike, from one number
    gx, gw2 = torch.autograd.grad(ops.gmm(x, w, sizes, trans_b=trans_b).sum(), (x, w))
    one = torch.ones_like(dc)
    _check_wgrad(gw2.transpose(1, 2) if trans_b else gw2, a, one, sizes)


def test_training_step_of_a_layer():
    announce(test="layer_step")
    # forward_train -> backward -> clip -> update, against the same step in 64 bits on the layer's own roundings
    E, d, I, R = 4, 128, 192, 260
    layer = MoEExperts(d, I, E, init_std=0.1, device=dev()).requires_grad_()
    sizes = torch.tensor([100, 0, 31, 129])
    x, dy = _rand((R, d), 1).requires_grad_(), _rand((R, d), 2)
    y = layer.forward_train(R, x, sizes.to(dev()), host_batch_sizes=sizes)
    with torch.no_grad():
        plain = layer.forward(R, x, sizes)
    assert float((y - plain).abs().max()) <= 4 * HALF * float(plain.abs().max())
    y.backward(dy)
    h, u = gg.gmm_swiglu_keep(x.detach(), layer.w13_weight.detach(), sizes)
    dh = gg.gmm(dy, layer.w2_weight.detach(), sizes, trans_b=True)
    _check_wgrad(layer.w2_weight.grad, h, dy, sizes)
    _check_block(u, h, x.grad, layer.w13_weight.grad, x.detach(), layer.w13_weight.detach(), dh, sizes)
    before = [p.grad.clone() for p in layer.parameters()]
    norm = grads.clip_grad_norm_(layer.parameters(), 0.25)
    want = sum(float(g.double().square().sum()) for g in before) ** 0.5
    assert abs(float(norm) - want) <= 2.0 ** -22 * want
    after = sum(float(p.grad.double().square().sum()) for p in layer.parameters()) ** 0.5
    assert abs(after - 0.25) <= 0.25 * HALF
    old = [p.detach().clone() for p in layer.parameters()]
    torch.optim.SGD(layer.parameters(), lr=0.5).step()
    assert all(not torch.equal(p, o) for p, o in zip(layer.parameters(), old))
    # the layer's forward pass takes the updated weights
    assert not torch.equal(layer.forward(R, x.detach(), sizes), plain)


def test_step_in_a_graph_beside_eager_steps():
    announce(test="step_graph")
    E, K, I, R = 4, 256, 136, 400
    b0 = _rand((E, K, 2 * I), 2, 0.06)
    b2 = _rand((E, I, K), 4, 0.06)
    x = torch.zeros(R, K, dtype=torch.bfloat16, device=dev(), requires_grad=True)
    w = b0.clone().requires_grad_()
    w2 = b2.clone().requires_grad_()
    dy = torch.zeros(R, K, dtype=torch.bfloat16, device=dev())
    sizes = torch.zeros(E, dtype=torch.int64, device=dev())
    size, ptr = gg.get_arguments(E, dev())
    own = dict(workspace=torch.empty(size, dtype=torch.uint8, device=dev()), arguments_ptr=ptr)

    def step(**state):
        y = ops.gmm(ops.gmm_swiglu(x, w, sizes, **state), w2, sizes, **state)
        g = torch.autograd.grad(y, (x, w, w2), dy)
        return (y.detach(), *g, grads.clip_by_global_norm_(g[1:], 1.0))

    with pytest.raises(RuntimeError, match="state"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()                                        # a recorded launch needs a state block of its own
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(**own)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step(**own)
    for rep in range(4):
        with torch.no_grad():
            x.copy_(_rand((R, K), 10 + rep))
            dy.copy_(_rand((R, K), 20 + rep))
            sizes.copy_(ragged_sizes(E, R - 7 * rep, seed=rep, empty_every=rep))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), rep
    gg.release_arguments(ptr)


def test_backward_after_the_layer_is_gone():
    announce(test="layer_gone")
    # the state block and the sizes that a backward pass needs live as long as its graph
    sizes = torch.tensor([40, 24])
    x, dy = _rand((64, 128), 1), _rand((64, 128), 2)
    layer = MoEExperts(128, 64, 2, init_std=0.1, device=dev()).requires_grad_()
    want_x = x.clone().requires_grad_()
    layer.forward_train(64, want_x, sizes).backward(dy)
    got_x = x.clone().requires_grad_()
    y = layer.forward_train(64, got_x, sizes.clone(), host_batch_sizes=sizes.clone())
    ptr = layer.arguments_ptr
    del layer
    assert ptr not in gg._STATE_BLOCKS
    y.backward(dy)
    assert torch.equal(want_x.grad, got_x.grad)


def test_a_layer_without_rows():
    announce(test="no_rows")
    layer = MoEExperts(64, 48, 3, device=dev()).requires_grad_()
    sizes = torch.zeros(3, dtype=torch.int64)
    for rows in (0, 700):                                 # none at all, and a padded batch that belongs to nobody
        x = torch.full((rows, 64), float("nan"), dtype=torch.bfloat16, device=dev(), requires_grad=True)
        y = layer.forward_train(rows, x, sizes)
        assert y.shape == (rows, 64) and not bool(y.any())
        for g in torch.autograd.grad(y, (x, *layer.parameters()), torch.ones_like(y)):
            assert not bool(g.any())
        assert float(grads.global_norm(torch.autograd.grad(layer.forward_train(rows, x, sizes).sum(), list(layer.parameters())))) == 0


def test_gradients_that_arrive_unaligned():
    announce(test="unaligned_gradient")
    # a gradient may be a view of other memory at any element; the operands may not
    sizes, K, N = torch.tensor([3, 0, 5]), 64, 48
    a, b = _rand((8, K), 1).requires_grad_(), _rand((3, K, N), 2, 0.1).requires_grad_()
    for call, cols in ((ops.gmm, N), (ops.gmm_swiglu, N // 2)):
        c = call(a, b, sizes)
        d = _rand((8 * cols + 1,), 3)
        view, copy = d[1:].view(8, cols), d[1:].clone().view(8, cols)
        assert view.data_ptr() % 16 != 0
        for x, y in zip(torch.autograd.grad(c, (a, b), view, retain_graph=True), torch.autograd.grad(c, (a, b), copy)):
            assert torch.equal(x, y)
        with pytest.raises(ValueError, match="aligned"):
            call(_rand((8 * K + 1,), 1)[1:].view(8, K), b, sizes)


def test_another_stream():
    announce(test="step_stream")
    sizes = torch.tensor([90, 30])
    a, b, dh = _rand((120, 128), 1), _rand((2, 128, 256), 2, 0.1), _rand((120, 128), 3)
    x, w = a.clone().requires_grad_(), b.clone().requires_grad_()
    want = torch.autograd.grad(ops.gmm_swiglu(x, w, sizes), (x, w), dh)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = torch.autograd.grad(ops.gmm_swiglu(x, w, sizes), (x, w), dh)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refusals():
    announce(test="grad_refusals")
    a, b = _rand((16, 64), 1).requires_grad_(), _rand((2, 64, 32), 2)
    n = torch.tensor([8, 8])
    with pytest.raises(AssertionError):
        ops.gmm(a.float(), b.float(), n)
    with pytest.raises(AssertionError):
        ops.gmm_swiglu(a, b, torch.tensor([16]))
    with pytest.raises(AssertionError):
        gg.gmm_wgrad(a.detach(), a.detach()[:8], n)
    y = ops.gmm_swiglu(a, b, n)
    g = torch.autograd.grad(y.sum(), a, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()                                 # the gradients themselves are not differentiable
