"""Operators of a recurrent layer over torch CUDA tensors: include/fr_b200.h's fr_b200_linear, fr_b200_conv_*, fr_b200_ssm_* and
fr_b200_slots_copy on the tensors' device and torch's current stream, through csrc/fr_b200_torch.so.

Tensors are [rows, width] with adjacent elements and any distance between rows, so that pieces of a wider projection go in as
they are; they are not copied or cast.  Results are new tensors unless `out` is given.  No gradient flows through them: a tensor that requires one is
refused outside torch.no_grad() and torch.inference_mode().
Sequences (`starts`) and slots are host lists, numpy int32 arrays or CPU integer tensors; a call that is captured into a CUDA
graph holds them by value.  ValueError: tensors that do not fit together; FrB200Error: what the library refuses.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

ACTIVATIONS = {"none": 0, "relu2": 1, "silu": 2, "sigmoid": 3, "gelu": 4, "softplus": 5}
EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "fr_b200_torch.so")
_ext = None


def _load():
    """csrc/fr_b200_torch.so, bound to the library that the package uses.  Raises if it was not built: there is no other path."""
    global _ext
    from . import LIB_PATH, FrB200Error, lib
    lib()
    if not os.path.exists(EXT_PATH):
        raise FrB200Error(-100, "fr_b200_torch.so is missing", "run `python -m faster_rwkv_b200.build` (or __graft_entry__.build()) first")
    import torch  # noqa: F401  (its libraries are what the extension is linked with)
    loader = importlib.machinery.ExtensionFileLoader("fr_b200_torch", EXT_PATH)
    ext = importlib.util.module_from_spec(importlib.util.spec_from_loader("fr_b200_torch", loader))
    loader.exec_module(ext)
    ext.bind(LIB_PATH)
    _ext = ext
    return ext


def _done(result, name):
    if result.__class__ is int:
        from . import FrB200Error, lib
        L = lib()
        raise FrB200Error(result, f"{name}: {L.fr_b200_strerror(result).decode()}", L.fr_b200_op_last_error().decode())
    return result


def _act(activation):
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {activation!r}") from None


def linear(x, w, bias=None, activation="none", residual=None, out=None, out_dtype=None):
    """residual + activation(x @ w.T + bias): x [rows, K], w [N, K] of one 16-bit type, bias [N] fp32; residual and the
    result [rows, N] in the type of x or out_dtype=torch.float32.  activation: none, relu2, silu, sigmoid, gelu, softplus.
    out may be the residual."""
    return _done((_ext or _load()).linear(x, w, bias, _act(activation), residual, out, out_dtype), "fr_b200_linear")


def check_operators(device=0):
    """Raises if a device-side wait of an operator gave up on `device` since the last check (NaN stands in the result of that call then).  It does
    not synchronise: torch.cuda.synchronize() comes before it."""
    from . import lib
    _done(lib().fr_b200_op_status(int(device)) or None, "fr_b200_op_status")


def conv_seq(x, w, bias=None, activation="silu", starts=None, state=None, from_slots=None, to_slots=None, out=None):
    """Causal convolution of each channel over the last taps rows of its sequence: x [rows, D], w [D, taps] (2 to 4) and bias
    [D] fp32, activation none or silu.  starts: first rows of the sequences and the end of the last (None: one sequence).
    state: pool [slots, taps - 1, D] of the last rows; sequence i begins from slot from_slots[i] (-1: from zero; a single
    number stands for all) and leaves its state in to_slots[i] (-1: nowhere); None: slot i.  Rows of no sequence stay as they
    are in `out`."""
    return _done((_ext or _load()).conv(x, w, bias, _act(activation), state, from_slots, to_slots, out, starts, True), "fr_b200_conv_seq")


def conv_step(x, w, bias=None, activation="silu", state=None, from_slots=None, to_slots=None, out=None):
    """conv_seq for one row of each stream: x [streams, D]."""
    return _done((_ext or _load()).conv(x, w, bias, _act(activation), state, from_slots, to_slots, out, None, False), "fr_b200_conv_step")


def ssm_seq(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=True, starts=None, state=None, from_slots=None, to_slots=None, out=None):
    """Selective state space scan over the rows of each sequence: for channel d, state n,
        delta = softplus(dt + dt_bias);  h = exp(delta * A) * h + delta * x * B;  y = (sum_n C * h + D * x) * silu(z).
    x, dt, z [rows, channels] and B, C [rows, groups * N] of one type; A [channels, N], D and dt_bias [channels] fp32.
    state: pool [slots, channels, N] fp32; starts, from_slots and to_slots as in conv_seq."""
    return _done((_ext or _load()).ssm(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, from_slots, to_slots, out, starts, True), "fr_b200_ssm_seq")


def ssm_step(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=True, state=None, from_slots=None, to_slots=None, out=None):
    """ssm_seq for one row of each stream."""
    return _done((_ext or _load()).ssm(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, from_slots, to_slots, out, None, False), "fr_b200_ssm_step")


def copy_slots(pool, src, dst):
    """pool[dst[i]] takes what pool[src[i]] holds before the call (src -1: zeros): states of streams forked, moved, reordered
    and cleared.  pool: [slots, ...] of any type with contiguous slots; every slot appears in dst once at most."""
    return _done((_ext or _load()).copy_slots(pool, src, dst), "fr_b200_slots_copy")
