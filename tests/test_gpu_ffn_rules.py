"""Gated blocks on either side of where their tiles change, with the kernels that the library chooses by itself.  Tolerances:
those of the gated block's tests."""
import pytest
import torch

from disagmoe_amd.grouped_gemm import backend as gg
from helpers import announce, dev
from test_gpu_ffn_grad import _check_block, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("K,I", [(2040, 3832), (2296, 3832), (2296, 3816), (3832, 3832)])
def test_contractions_cut_in_two(K, I, trans_b):
    """Gradient of the rows on 64, 72 and 120 tiles of 256 rows, of 240 stages and one fewer, with the last stage half full."""
    announce(test="block_cut", K=K, I=I, trans_b=trans_b)
    sizes = torch.tensor([1000, 1000])
    a, dh = _rand((2000, K), 1), _rand((2000, I), 2)
    b = _rand((2, K, 2 * I), 3, K ** -0.5)
    given = b.transpose(1, 2).contiguous() if trans_b else b
    h, u = gg.gmm_swiglu_keep(a, given, sizes, trans_b=trans_b)
    da, db = gg.gmm_swiglu_backward(dh, u, a, given, sizes, trans_b=trans_b)
    _check_block(u, h, da, db.transpose(1, 2) if trans_b else db, a, b, dh, sizes)
    again, _ = gg.gmm_swiglu_backward(dh, u, a, given, sizes.to(dev()), trans_b=trans_b, need_db=False)
    _check_block(u, h, again, None, a, b, dh, sizes)
