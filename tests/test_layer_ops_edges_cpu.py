"""Edges of the operators of a recurrent layer that need no device: refusals, status codes, arguments."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from test_layer_ops_cpu import BF16, F32, O, R, S, W, X, _conv, _linear, _refused, _ssm


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


# ---- what may not overlap ----------------------------------------------------------------------------------------
# conv: w [64, 4] and a bias of 64, out [20, 64] f16, a pool of 4 slots of 192; ssm: A [64, 16], D and dt_bias of 64, a pool of 4 of 1024 fp32

@pytest.mark.parametrize("kw", [dict(w=O), dict(w=O + 20 * 128 - 4), dict(w=O - 64 * 4 * 4 + 4), dict(bias=O + 64), dict(w=S), dict(bias=S + 4 * 384 - 4), dict(bias=S - 252)])
def test_conv_refuses_results_over_parameters(pkg, kw):
    _refused(pkg, "fr_b200_conv_seq", _conv(**kw), "parameter")


@pytest.mark.parametrize("seq", [True, False])
@pytest.mark.parametrize("kw", [dict(A=O), dict(A=S + 4), dict(D=O + 124), dict(D=S), dict(bias=O), dict(bias=S + 4 * 4096 - 4), dict(A=O - 64 * 16 * 4 + 4)])
def test_ssm_refuses_results_over_parameters(pkg, kw, seq):
    _refused(pkg, "fr_b200_ssm_seq" if seq else "fr_b200_ssm_step", _ssm(seq, **kw), "parameter")


def test_work_areas_overlap_nothing(pkg):
    L = pkg.lib()
    need = L.fr_b200_ssm_seq_workspace(2000, 1, 64, 16)
    far = 0x70000000
    assert need > 0
    a = dict(rows=2000, work=far, wb=need, D=W + 0x100000, bias=W + 0x200000)
    for at in (X, X + 0x1000000, X + 0x2000000, X + 0x3000000, W, W + 0x100000, W + 0x200000, S, O):
        _refused(pkg, "fr_b200_ssm_seq", _ssm(**{**a, "work": at}), "work area")
        _refused(pkg, "fr_b200_ssm_seq", _ssm(**{**a, "work": at - need + 4}), "work area")
    a = dict(rows=4000, K=1001, ldx=1001, ldw=1001, N=100, ldo=100, work_bytes=4100 * 126 * 16, bias=far, residual=R, ldr=100)
    for at in (X, W, O, R, far):
        _refused(pkg, "fr_b200_linear", _linear(**a, work=at), "work area")
    if not torch.cuda.is_available():     # (no device: past the checks)
        assert L.fr_b200_linear(*_linear(**a, work=far + 0x1000)) == -3
        assert L.fr_b200_ssm_seq(*_ssm(rows=2000, work=far, wb=need)) == -3


def test_a_parameter_between_rows_does_not_overlap(pkg):
    """rows far apart, with the parameters in what lies between them: taken as before"""
    if torch.cuda.is_available():
        pytest.skip("GPU present: the addresses are not memory")
    L = pkg.lib()
    assert L.fr_b200_conv_seq(*_conv(out=O, ldo=4096, w=O + 128, bias=O + 128 + 1024)) == -3
    _refused(pkg, "fr_b200_conv_seq", _conv(out=O, ldo=4096, w=O + 124), "parameter")
    _refused(pkg, "fr_b200_conv_seq", _conv(out=O, ldo=4096, bias=O + 8192 - 252), "parameter")
    assert L.fr_b200_linear(*_linear(out=O, ldo=512, bias=O + 64)) == -3
    _refused(pkg, "fr_b200_linear", _linear(out=O, ldo=512, bias=O + 60), "bias")
    assert L.fr_b200_linear(*_linear(dtype=BF16, out_dtype=F32, rows=1, x=O + 128)) == -3


# ---- lists of slots ----------------------------------------------------------------------------------------------

def test_model_copy_states_takes_whole_numbers_alone(pkg):
    """what is no 32-bit integer is refused, not cut down to one"""
    m = object.__new__(pkg.Model)
    m._h = None
    for src, dst in (([0.5], [1]), ([0], [1.9]), (np.array([2 ** 32]), [1]), ([0], np.array([2 ** 32 + 1])), ([-2 ** 40], [0]), (np.array([2 ** 63], np.uint64), [0]),
                     (["0"], ["1"]), ([True], [False]), ([[0]], [[1]]), (0, 1), ([0, 1], [1]), (np.array([2 ** 31]), [0])):
        with pytest.raises(ValueError):
            m.copy_states(src, dst)
    for src, dst in (([0], [1]), ((0, 2), np.array([1, 3], np.int64)), ([], []), (np.array([-1], np.int8), [5])):
        with pytest.raises(pkg.FrB200Error):       # taken: the library refuses the model that is not there
            m.copy_states(src, dst)


# ---- gradients ---------------------------------------------------------------------------------------------------

def test_tensors_that_require_a_gradient(pkg):
    """no gradient flows: said before anything else, instead of a result that has none.  Under no_grad and inference_mode they are taken (and
    refused here for their place, the CPU)."""
    x, p = torch.zeros(4, 8), torch.nn.Parameter(torch.zeros(8, 8))
    calls = [lambda: pkg.linear(p, x), lambda: pkg.linear(x, p), lambda: pkg.conv_step(p, x), lambda: pkg.conv_seq(x, p), lambda: pkg.ssm_step(x, x, p, x, x),
             lambda: pkg.ssm_seq(p, x, x, x, x), lambda: pkg.copy_slots(p, [0], [1])]
    for f in calls:
        with pytest.raises(ValueError, match="gradient"):
            f()
        for mode in (torch.no_grad, torch.inference_mode):
            with mode(), pytest.raises(ValueError, match="GPU"):
                f()


# ---- out of memory -----------------------------------------------------------------------------------------------

NOMEM = """
import resource
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import __graft_entry__ as entry
from test_layer_ops_cpu import _conv, _i32
pkg = entry.load_package()
L = pkg.lib()
assert L.fr_b200_conv_seq(*_conv(taps=9)) == -1
with open("/proc/self/statm") as f:
    held = int(f.read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (held + (1 << 30), resource.RLIM_INFINITY))
# the record of who writes which slot would take 16 GB
rc = L.fr_b200_conv_seq(*_conv(n_slots=2 ** 31 - 1, fro=_i32(0), to=_i32(1)))
print(rc, L.fr_b200_op_last_error().decode())
"""


def test_host_memory_that_runs_out_has_its_own_text(pkg):
    """no exception crosses the C interface, and the text is not that of the call before"""
    tests = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", NOMEM.format(root=os.path.dirname(tests), tests=tests)], capture_output=True, text=True, timeout=300)
    assert r.stdout == "-7 out of memory\n", (r.stdout, r.stderr[-500:])


def test_no_moves_ask_for_nothing(pkg):
    L = pkg.lib()
    assert L.fr_b200_slots_copy(None, 0, 0, 0, 0, None, None, 0, None) == 0
    assert L.fr_b200_slots_copy(S, 64, 64, 8, 0, None, None, 0, None) == 0
    _refused(pkg, "fr_b200_slots_copy", (S, 64, 64, 8, -1, None, None, 0, None), "moves")
