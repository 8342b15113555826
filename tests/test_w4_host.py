"""4-bit weights: layout, and the refusals that answer without a device."""
import ctypes

import pytest
import torch

from disagmoe_amd import _lib
from disagmoe_amd.grouped_gemm import backend as gg


def test_host_side_argument_errors():
    lib = _lib.load()
    p = 0x100000   # never touched: every call is refused before a launch

    def call(a=p, codes=p, scales=p, zeros=None, group=128, c=p, bs=p, rows=16, E=4, K=64, N=64, wide=None, name="dmoe_gmm_w4"):
        return getattr(lib, name)(a, codes, scales, zeros, group, c, bs, rows, E, K, N, wide, 0, None, None, 0, None, None)

    for name in ("dmoe_gmm_w4", "dmoe_gmm_w4_swiglu"):
        for bad in (dict(K=60), dict(N=12), dict(N=0), dict(K=0), dict(E=0), dict(E=1025), dict(rows=-1), dict(rows=1 << 31), dict(N=1 << 20)):
            assert call(**bad, name=name) == _lib.ERR_SHAPE, bad
        for bad in (dict(group=16), dict(group=0), dict(a=None), dict(codes=None), dict(scales=None), dict(c=None), dict(bs=None),
                    dict(a=p + 8), dict(codes=p + 4), dict(zeros=p + 1), dict(c=p + 2), dict(scales=p + 8), dict(wide=p + 8)):
            assert call(**bad, name=name) == _lib.ERR_ARG, bad
        assert call(rows=0, name=name) == 0
    n = [ctypes.c_size_t() for _ in range(3)]
    assert lib.dmoe_w4_bytes(2, 136, 24, 32, *map(ctypes.byref, n)) == 0
    assert [v.value for v in n] == [2 * 2 * 2 * 1024, 2 * 2 * 2 * 16 * 4 * 2, 2 * 2 * 2 * 16 * 4]
    assert lib.dmoe_w4_bytes(2, 136, 24, 48, *map(ctypes.byref, n)) == _lib.ERR_ARG
    assert lib.dmoe_w4_quant(p, 2, 64, 64, 64, None, p, None, None) == _lib.ERR_ARG
    assert lib.dmoe_w4_dequant(p, p, None, 64, p + 8, None, 2, 64, 64, None) == _lib.ERR_ARG
    need = ctypes.c_size_t(1)
    assert lib.dmoe_gmm_w4_wide_bytes(8, 8, 64, 64, 128, None, ctypes.byref(need)) == 0 and need.value == 0
    up = lambda n: -(-n // 256) * 256                             # weights, their scales, rows, their scales
    wide = lambda rows: up(8 * 64 * 64 * 2) + up(8 * 64 * 4) + up(rows * 64 * 2) + up(rows * 4)
    assert lib.dmoe_gmm_w4_wide_bytes(1 << 20, 8, 64, 64, 128, None, ctypes.byref(need)) == 0 and need.value == wide(1 << 20)
    assert lib.dmoe_gmm_w4_wide_bytes(1 << 20, 8, 40, 64, 128, None, ctypes.byref(need)) == 0 and need.value == wide(1 << 20)  # K up to 32s
    sizes = (ctypes.c_int64 * 8)(*([0] * 7 + [4000]))             # one expert has all the rows
    assert lib.dmoe_gmm_w4_wide_bytes(4000, 8, 64, 64, 128, sizes, ctypes.byref(need)) == 0 and need.value == wide(4000)
    assert lib.dmoe_gmm_w4_wide_bytes(-1, 8, 64, 64, 128, None, ctypes.byref(need)) == _lib.ERR_ARG


def unpack(w):
    """(codes [E, N, K], scales [E, N, groups], zeros or None) of packed weights, word by word as the header describes."""
    E, nt, kt, _ = w.codes.shape
    q = torch.zeros(E, nt * 16, kt * 128, dtype=torch.uint8)
    b = w.codes.cpu().view(E, nt, kt, 4, 16, 4, 4).int()          # [.., g, r, j, byte]
    word = b[..., 0] | b[..., 1] << 8 | b[..., 2] << 16 | b[..., 3] << 24
    for g in range(4):
        for j in range(4):
            for i in range(8):
                nibble = i // 2 if i % 2 == 0 else 4 + i // 2
                k = 32 * j + 8 * g + i
                q.view(E, nt, 16, kt, 128)[..., k] = ((word[:, :, :, g, :, j] >> (4 * nibble)) & 15).transpose(2, 3).to(torch.uint8)
    def groups(v):
        return None if v is None else v.cpu().permute(0, 1, 3, 5, 2, 4).reshape(E, nt * 16, -1)[:, :w.N, :-(-w.K // w.group)]
    return q[:, :w.N, :w.K], groups(w.scales), groups(w.zeros)


@pytest.mark.parametrize("E,N,K,group", [(1, 8, 8, 128), (2, 24, 136, 32), (3, 48, 264, 64), (1, 16, 128, 128), (2, 40, 72, 32)])
@pytest.mark.parametrize("zeros", [False, True])
def test_pack(E, N, K, group, zeros):
    g = torch.Generator().manual_seed(K)
    codes = torch.randint(0, 16, (E, N, K), generator=g, dtype=torch.uint8)
    groups = -(-K // group)
    s = torch.rand(E, N, groups, generator=g).to(torch.bfloat16)
    z = torch.randint(0, 16, (E, N, groups), generator=g, dtype=torch.uint8) if zeros else None
    w = gg.pack_w4(codes, s, z, group)
    assert w.codes.shape == (E, -(-N // 16), -(-K // 128), 1024) and (w.K, w.N, w.group) == (K, N, group)
    q, s2, z2 = unpack(w)
    assert torch.equal(q, codes) and torch.equal(s2, s) and (z2 is None if z is None else torch.equal(z2, z))
    # what reaches past the weights is code 0 with scale 0
    assert int(w.codes.sum(dtype=torch.int64)) == _byte_sum(codes)
    assert float(w.scales.double().sum()) == float(s.double().sum())


def _byte_sum(codes):
    """The sum of the packed bytes: odd nibbles of a word are the high halves of their bytes."""
    i = torch.arange(codes.shape[2]) % 8
    nibble = torch.where(i % 2 == 0, i // 2, 4 + i // 2)
    return int((codes.long() * torch.where(nibble % 2 == 1, 16, 1)).sum())


def test_python_refusals():
    with pytest.raises(ValueError):
        gg.pack_w4(torch.zeros(1, 8, 8, dtype=torch.uint8), torch.zeros(1, 8, 1), None, 16)
    with pytest.raises(AssertionError):
        gg.pack_w4(torch.zeros(1, 8, 12, dtype=torch.uint8), torch.zeros(1, 8, 1), None, 32)
    with pytest.raises(RuntimeError):
        gg.quantize_weight_w4(torch.zeros(1, 8, 8, dtype=torch.bfloat16))
    w = gg.pack_w4(torch.zeros(1, 8, 8, dtype=torch.uint8), torch.zeros(1, 8, 1), None, 32)
    with pytest.raises(RuntimeError):
        gg.gmm_w4(torch.zeros(1, 8, dtype=torch.bfloat16), w, torch.tensor([1]))


def test_room_for_some_experts():
    lib, need, all_of_them = _lib.load(), ctypes.c_size_t(), ctypes.c_size_t()
    up = lambda n: -(-n // 256) * 256                             # weights, their scales, rows, their scales, sizes
    for experts in (1, 3, 8):
        assert lib.dmoe_gmm_w4_wide_bytes_of(5000, experts, 40, 24, ctypes.byref(need)) == 0
        assert need.value == up(experts * 24 * 64 * 2) + up(experts * 24 * 4) + up(5000 * 64 * 2) + up(5000 * 4) + up(experts * 8 + 8)
    assert lib.dmoe_gmm_w4_wide_bytes(5000, 8, 40, 24, 128, None, ctypes.byref(all_of_them)) == 0 and all_of_them.value <= need.value
    assert lib.dmoe_gmm_w4_wide_bytes_of(5000, 0, 40, 24, ctypes.byref(need)) == _lib.ERR_SHAPE
    assert lib.dmoe_gmm_w4_wide_bytes_of(5000, 2, 44, 24, ctypes.byref(need)) == _lib.ERR_SHAPE
    assert lib.dmoe_gmm_w4_wide_bytes_of(-1, 2, 40, 24, ctypes.byref(need)) == _lib.ERR_ARG
    assert lib.dmoe_gmm_w4_wide_bytes_of(1, 2, 40, 24, None) == _lib.ERR_ARG


def test_values_that_four_bits_do_not_hold():
    """A code above 15 would run into its neighbour."""
    codes, scales, zeros = torch.full((1, 8, 32), 15, dtype=torch.uint8), torch.ones(1, 8, 1), torch.full((1, 8, 1), 15, dtype=torch.uint8)
    gg.pack_w4(codes, scales, zeros, 32)
    for bad in (16, 255):
        c, z = codes.clone(), zeros.clone()
        c[0, 3, 5] = z[0, 2, 0] = bad
        with pytest.raises(ValueError, match="codes"):
            gg.pack_w4(c, scales, zeros, 32)
        with pytest.raises(ValueError, match="zeros"):
            gg.pack_w4(codes, scales, z, 32)
    with pytest.raises(ValueError, match="codes"):
        gg.pack_w4(codes.to(torch.int8) - 20, scales, None, 32)
    with pytest.raises(ValueError, match="codes"):
        gg.pack_w4(codes.float(), scales, None, 32)
    assert torch.equal(gg.pack_w4(codes.long(), scales, zeros.int(), 32).codes, gg.pack_w4(codes, scales, zeros, 32).codes)
    with pytest.raises(AssertionError):                          # one zero point for all groups is not taken for the first one's
        gg.pack_w4(torch.zeros(1, 8, 64, dtype=torch.uint8), torch.ones(1, 8, 2), torch.zeros(1, 8, 1, dtype=torch.uint8), 32)
