"""The 4-bit products of many rows and the memory they write 16-bit weights to: none, some, all of what they ask for.

Results in the form for many rows and in the one kernel differ by their roundings; ``_check`` of the 4-bit products' tests
has the tolerances of both, and both have to hold for the experts that each form serves."""
import pytest
import torch

from disagmoe_amd import _lib
from disagmoe_amd.grouped_gemm import backend as gg
from helpers import announce, dev
from test_gpu_w4 import _check, _rand, _spans, _weight

pytestmark = pytest.mark.gpu


def _call(swiglu, x, w, c, sizes, host, wide, nbytes):
    E = w.codes.shape[0]
    size, ptr = gg.get_arguments(E, dev())
    ws = torch.empty(size, dtype=torch.uint8, device=dev())
    _lib.call("dmoe_gmm_w4_swiglu" if swiglu else "dmoe_gmm_w4", x.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
              None if w.zeros is None else w.zeros.data_ptr(), w.group, c.data_ptr(), sizes.data_ptr(), x.shape[0], E, w.K, c.shape[1],
              wide.data_ptr(), nbytes, ptr, ws.data_ptr(), size, None if host is None else host.data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    gg.release_arguments(ptr)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("K,zeros", [(264, True), (384, False)])
def test_room_for_some_experts(swiglu, K, zeros):
    """The first experts with rows go through the room there is, the others through the one kernel; rows behind the last
    expert and behind the result stay as they are, whatever lies in the scratch memory and behind it."""
    sizes, N, group = torch.tensor([0, 1400, 3, 0, 2200, 1, 1800, 0]), 144, 64
    E, used = len(sizes), int(sizes.sum())
    R = used + 37
    w, ref, s = _weight(E, N, K, group, zeros, seed=K)
    x = _rand((R, K), 5)
    x[used:] = float("nan")
    n_out = N // 2 if swiglu else N
    busy = [e for e in range(E) if sizes[e] > 0]
    for host in (None, sizes, torch.tensor([0] * 7 + [R])):       # the last one disagrees with the device
        for room in range(0, E + 1):
            announce(test="w4_room", swiglu=swiglu, K=K, room=room, host=None if host is None else host.tolist())
            need = _lib.c_size_t(0)
            _lib.call("dmoe_gmm_w4_wide_bytes_of", R, max(room, 1), K, N, _lib.ctypes.byref(need))
            nbytes = need.value - (256 if room == 0 else 0)       # room for none: a little short of one
            wide = torch.full((need.value + 256,), 0xff, dtype=torch.uint8, device=dev())   # NaN in every format
            c = torch.full((R + 5, n_out), 7.0, dtype=torch.bfloat16, device=dev())
            _call(swiglu, x, w, c, sizes.to(dev()), host, wide, nbytes)
            first = int(sizes[:busy[room]].sum()) if room < len(busy) else used
            through = torch.where(torch.arange(E) < (busy[room] if room < len(busy) else E), sizes, 0)
            _check(c[:first], x, ref, s, through, group, swiglu, True)
            rest = torch.where(through > 0, 0, sizes)
            _check(c[first:used], x[first:used], ref, s, rest, group, swiglu, False)
            assert bool((c[used:] == 7).all()) and bool((wide[nbytes:] == 0xff).all())


@pytest.mark.parametrize("swiglu", [False, True])
def test_memory_for_the_experts_that_have_rows(swiglu):
    """One busy expert of many: the call takes memory for one, and for the others not a byte each."""
    E, N, K, rows = 48, 2048, 1024, 700
    w, ref, s = _weight(E, N, K, 128, False, seed=2)
    sizes = torch.zeros(E, dtype=torch.int64)
    sizes[37] = rows
    x = _rand((rows, K), 3)
    call = gg.gmm_w4_swiglu if swiglu else gg.gmm_w4
    call(x, w, sizes)                                             # (the stream's own pair exists from here on)
    announce(test="w4_memory", swiglu=swiglu)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = call(x, w, sizes)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 3 * N * K * 2
    _check(got, x, ref, s, sizes, 128, swiglu, True)
    one = w._replace(codes=w.codes[37:38].clone(), scales=w.scales[37:38].clone())
    assert torch.equal(got, call(x, one, torch.tensor([rows])))


@pytest.mark.parametrize("swiglu", [False, True])
def test_no_memory_left(monkeypatch, swiglu):
    sizes, N, K, group = torch.tensor([600, 0, 800]), 96, 200, 32
    w, ref, s = _weight(3, N, K, group, True, seed=9)
    x = _rand((1400, K), 9)
    call = gg.gmm_w4_swiglu if swiglu else gg.gmm_w4
    empty, asked = torch.empty, []

    def no_room(shape, **kwargs):
        if kwargs.get("dtype") is torch.uint8:
            asked.append(shape)
            raise torch.OutOfMemoryError("no room")
        return empty(shape, **kwargs)

    call(x, w, sizes)
    monkeypatch.setattr(gg.torch, "empty", no_room)
    for bs in (sizes, sizes.to(dev())):
        announce(test="w4_no_memory", swiglu=swiglu, device=str(bs.device))
        got = call(x, w, bs)
        assert len(asked) == 1 and asked.pop() > 2 * 2 * N * K
        _check(got, x, ref, s, sizes, group, swiglu, False)


@pytest.mark.parametrize("rows", [30, 1500])
def test_gated_form_leaves_rows_that_are_nobodys(rows):
    """As the plain product: rows behind sum(batch_sizes) stay, rows do not see each other, sizes that overrun are clamped."""
    announce(test="w4_gated_apart", rows=rows)
    sizes = torch.tensor([rows // 10, 0, rows - rows // 10 - 7, 7])
    E, K, N, group = 4, 264, 64, 32
    w, ref, s = _weight(E, N, K, group, True, seed=5)
    x = _rand((rows + 9, K), 6)
    clean = gg.gmm_w4_swiglu(x, w, sizes)[:rows].clone()
    _check(clean, x, ref, s, sizes, group, True, rows > 1000)
    x[1], x[10], x[rows:] = float("nan"), float("inf"), float("nan")
    c = torch.full((rows + 20, N // 2), 7.0, dtype=torch.bfloat16, device=dev())
    assert gg.gmm_w4_swiglu(x, w, sizes, c=c) is c and bool((c[rows:] == 7).all())
    keep = [r for r in range(rows) if r not in (1, 10)]
    assert torch.equal(c[keep], clean[keep]) and not bool(c[[1, 10]].isfinite().any())
    c.fill_(7)
    for nobody in (torch.zeros(E, dtype=torch.int64), torch.zeros(E, dtype=torch.int64, device=dev())):
        gg.gmm_w4_swiglu(x, w, nobody, c=c)
        assert bool((c == 7).all())
    assert gg.gmm_w4_swiglu(x[:0], w, torch.zeros(E, dtype=torch.int64)).shape == (0, N // 2)
    guard = torch.full((rows + 4, N // 2), 5.0, dtype=torch.bfloat16, device=dev())
    gg.gmm_w4_swiglu(x[:rows].contiguous(), w, sizes + torch.tensor([0, 0, 0, 700]), c=guard)
    assert torch.equal(guard[keep], clean[keep]) and bool((guard[rows:] == 5).all())
