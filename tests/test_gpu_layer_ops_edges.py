"""Edges of the operators of a recurrent layer: calls that their documentation allows and that lie beside the ordinary ones."""
import numpy as np
import pytest
import torch

from test_gpu_layer_ops import F16, F32

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
