"""Edges of the operators of a recurrent layer that need no device: refusals, status codes, arguments."""
import pytest
import torch


def test_status_of_the_operators_without_a_device(pkg):
    L = pkg.lib()
    for limit in (0, 1000001):
        assert L.fr_b200_op_wait_selftest(0, limit, None) == -1
        assert b"limit" in L.fr_b200_op_last_error()
    assert L.fr_b200_op_status(1000) == -3                # no such device
    if not torch.cuda.is_available():
        assert L.fr_b200_op_status(0) == -3
        with pytest.raises(pkg.FrB200Error):
            pkg.check_operators()
