"""Edges of the operators of a recurrent layer: calls that their documentation allows and that lie beside the ordinary ones."""
import numpy as np
import pytest
import torch

from test_gpu_layer_ops import F16, F32, _check, _linear_want, _rand

pytestmark = pytest.mark.gpu


# ---- slots -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,row", [(F32, 25), (F32, 25001), (F32, 750001), (F16, 51), (F16, 50001), (F16, 1500001), (torch.uint8, 101), (torch.uint8, 100001),
                                       (torch.uint8, 3000001), (F32, 24), (F32, 25000)])
def test_copy_slots_that_only_clears(pkg, dtype, row):
    """no slot is read: slots of 4-, 2-, 1- and 16-byte granules, of one column of a CTA and of many"""
    pool = torch.randint(1, 200, (9, row), device="cuda").to(dtype)
    for dst in ([4], [0, 8], [7, 1, 2, 6, 3]):
        p = pool.clone()
        pkg.copy_slots(p, [-1] * len(dst), np.asarray(dst, np.int32))
        want = pool.clone()
        want[dst] = 0
        assert torch.equal(p, want)


# ---- waits that give up ------------------------------------------------------------------------------------------

def test_a_wait_that_gave_up_is_told_once_and_refuses_nobody(pkg):
    """the status word is asked for; products that have nothing to do with it run, before and behind the question"""
    L = pkg.lib()
    pkg.check_operators()
    x, w = _rand(40, 64, dtype=F16), _rand(24, 64, dtype=F16, scale=0.1, seed=1)
    want, err = _linear_want(x, w, None, "none", None)
    assert L.fr_b200_op_wait_selftest(0, 1000, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    _check(pkg.linear(x, w), want, err)
    assert L.fr_b200_op_status(0) == -6 and b"gave up" in L.fr_b200_op_last_error()
    assert L.fr_b200_op_status(0) == 0
    _check(pkg.linear(x, w), want, err)
    assert L.fr_b200_op_wait_selftest(0, 1000, None) == 0
    torch.cuda.synchronize()
    with pytest.raises(pkg.FrB200Error):
        pkg.check_operators(0)
    pkg.check_operators(0)
